// What the kernels of the 8-bit products share: the job, what becomes of a sum (finish), the loads of ragged rows.
#pragma once

#include "number_types.hpp"

namespace i8 {

using namespace num;

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

constexpr int BLOCK = 256;
constexpr int VEC = 8;                         // neighbouring outputs that a thread finishes at once

struct Job {
    const signed char *a, *b, *b2;             // b2: the second weights of the gated form
    i64 lda, ldb, ldb2;
    i64 m, k, n;
    const float *a_scale, *b_scale, *b2_scale, *bias;
    int dtype, act;
    void *out;
    i64 ldo;
    int *partial;                              // [slices][1 or 2][m][n] sums, for more than one slice of the inner dimension
    int slices, steps_per_slice, steps;
    int mt, nt;                                // tiles down and across
};

// 16 bytes of a row of which `left` are there (any number, also none or fewer); zero behind them
__device__ __forceinline__ v4i load_part(const signed char *p, i64 left) {
    if (left >= 16) return load_any<v4i>(p);
    v4i v = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 15; ++e)
        if (e < left) v[e / 4] |= (int)((u32)(unsigned char)p[e] << (8 * (e & 3)));
    return v;
}

// The same of a row of k: one load, of a long row's last 16 bytes at the latest, moved down where they begin before p.  (In single
// bytes, one behind the other, 3000 x 250 x 3000 took 27 us, 17-18 so, 12.3 with 256.)
__device__ __forceinline__ v4i load_end(const signed char *p, i64 left, i64 k) {
    if (k < 16) return load_part(p, left);
    const int here = (int)max((i64)0, min(left, (i64)16)), bits = (16 - here) * 8 & 63;
    v4i v = load_any<v4i>(p + min(left - 16, (i64)0));
    u64 lo = (u64)(u32)v.x | (u64)(u32)v.y << 32, hi = (u64)(u32)v.z | (u64)(u32)v.w << 32;
    if (here <= 8) lo = hi, hi = 0;
    lo = lo >> bits | hi << 1 << (63 - bits);
    hi >>= bits;
    if (here == 0) lo = hi = 0;
    return v4i{(int)lo, (int)(lo >> 32), (int)hi, (int)(hi >> 32)};
}

// x / (1 + e^-x), with e^-|x| so that nothing overflows, and a step of Newton's behind the reciprocal (one unit off as it comes)
// (for x > -80: v_exp_f32 has no results below 2^-126)
__device__ __forceinline__ float silu(float x) {
    const float t = __builtin_amdgcn_exp2f(fabsf(x) * -1.44269504f), y = 1.0f + t, r = __builtin_amdgcn_rcpf(y);
    return (x < 0.0f ? x * t : x) * fmaf(fmaf(-y, r, 1.0f), r, r);
}
// the same below, where the sum is one; 0 for products that have overflowed to -inf
__device__ __forceinline__ float silu_far(float x) { return fmaxf(x, -200.0f) * expf(x); }

// x Phi(x), with all digits below zero too, where 0.5 (1 + erf(x / sqrt 2)) cancels (4 % off at -5, 0 from -5.5 on):
// Phi(-u) = e^(-u^2 / 2) h(u), and h, which falls slowly from 1/2, is q P(q) with q = 1 / (1 + 0.27 u), P of degree 8 fitted to it over
// Chebyshev's nodes of q (2.4e-8 of h off for u up to 14.5, where the exponential has ended).  Some 7 + x^2 units of 2^-24 off, the second
// from the exponent's roundings.  Gated 1000 x 4096 x 11008 100 us, 1000 x 512 x 11008 31.5 (silu 98 and 28);
// 112 and 31.6 with erff, 111 and 36 with erfcf.
__device__ __forceinline__ float gelu(float x) {
    constexpr float P[] = {0.107720658f, 0.107542865f, 0.101810686f, 0.0720492899f, 0.107826404f,
                           -0.0692119151f, 0.169787183f, -0.126486361f, 0.0289612059f};
    const float q = __builtin_amdgcn_rcpf(fmaf(fabsf(x), 0.27f, 1.0f));
    float p = P[8];
#pragma unroll
    for (int i = 7; i >= 0; --i) p = fmaf(p, q, P[i]);
    const float tail = p * q * __builtin_amdgcn_exp2f(x * (x * -0.72134752f));
    const float near = fminf(fmaxf(x, -100.0f), 100.0f);           // the tail is 0 there, which infinities would make a NaN of
    return x < 0.0f ? near * tail : fmaf(-near, tail, x);
}

__device__ __forceinline__ void activate(float (&v)[VEC], int act) {
    if (act == VI_GELU) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = gelu(v[e]);
        return;
    }
    float least = v[0];
#pragma unroll
    for (int e = 1; e < VEC; ++e) least = fminf(least, v[e]);
    if (least > -80.0f) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = silu(v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = v[e] <= -80.0f ? silu_far(v[e]) : silu(v[e]);
    }
}

template <int DT>
__device__ __forceinline__ void store_floats(void *out, i64 at, const float (&v)[VEC], int count) {
    typedef typename type<DT>::t T;
    T *o = (T *)out + at;
    T r[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) r[e] = (T)v[e];
    if (count == VEC) {
        store_any(o, r);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (e < count) o[e] = r[e];
    }
}

// The sums of row `row`, columns col .. col + count - 1, as they go out: s of the first weights, t of the second.  Integers leave
// as they are (or as residues mod p); otherwise (s a_scale) b_scale in 32 bits, a sum of more than 24 bits rounded by the conversion,
// and one rounding to the type of the output.
template <bool GATED>
__device__ __forceinline__ void finish(const Job &J, i64 row, i64 col, int count, const int (&s)[VEC], const int (&t)[VEC]) {
    const i64 at = row * J.ldo + col;
    if (!GATED && J.dtype == VI_I32) {
        int *o = (int *)J.out + at;
        if (count == VEC) {
            store_any(o, s);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (e < count) o[e] = s[e];
        }
        return;
    }
    if (!GATED && J.dtype == VI_FIELD) {
        u64 *o = (u64 *)J.out + at;
        u64 r[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) r[e] = (u64)(i64)s[e] - (s[e] < 0 ? 0xFFFFFFFFull : 0);       // p - |s| below zero
        if (count == VEC) {
            store_any(o, r);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (e < count) o[e] = r[e];
        }
        return;
    }
    const float as = J.a_scale[row];
    float bs[VEC], v[VEC];
    auto scales = [&](const float *p) {
        if (count == VEC) {
            __builtin_memcpy(bs, p + col, sizeof(bs));
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) bs[e] = e < count ? p[col + e] : 0.0f;
        }
    };
    scales(J.b_scale);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = (float)s[e] * as * bs[e];
    if (GATED) {
        scales(J.b2_scale);
#pragma unroll
        for (int e = 0; e < VEC; ++e) bs[e] = (float)t[e] * as * bs[e];
        activate(v, J.act);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] *= bs[e];
    } else if (J.bias) {
        scales(J.bias);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] += bs[e];
    }
    if (J.dtype == VI_F32) store_floats<VI_F32>(J.out, at, v, count);
    if (J.dtype == VI_BF16) store_floats<VI_BF16>(J.out, at, v, count);
    if (J.dtype == VI_F16) store_floats<VI_F16>(J.out, at, v, count);
}

// the same of one output
template <bool GATED>
__device__ __forceinline__ void finish_one(const Job &J, i64 row, i64 col, int s, int t) {
    const i64 at = row * J.ldo + col;
    if (!GATED && J.dtype == VI_I32) {
        ((int *)J.out)[at] = s;
        return;
    }
    if (!GATED && J.dtype == VI_FIELD) {
        ((u64 *)J.out)[at] = (u64)(i64)s - (s < 0 ? 0xFFFFFFFFull : 0);
        return;
    }
    const float as = J.a_scale[row];
    float v = (float)s * as * J.b_scale[col];
    if (GATED) {
        if (J.act == VI_GELU) v = gelu(v);
        else v = v <= -80.0f ? silu_far(v) : silu(v);
        v *= (float)t * as * J.b2_scale[col];
    } else if (J.bias) {
        v += J.bias[col];
    }
    if (J.dtype == VI_F32) ((float *)J.out)[at] = v;
    if (J.dtype == VI_BF16) ((__bf16 *)J.out)[at] = (__bf16)v;
    if (J.dtype == VI_F16) ((_Float16 *)J.out)[at] = (_Float16)v;
}

}  // namespace i8
