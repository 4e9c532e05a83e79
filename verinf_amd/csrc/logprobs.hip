// Log probabilities of given tokens under rows of logits, the rows' entropies and their largest entries.
//
//     M = max_j x_j    d_j = (x_j - M) / T    Z = sum e^d_j    lp(j) = d_j - log Z    H = log Z - (sum e^d_j d_j) / Z
//
// One pass over the logits: a workgroup keeps its slice of a row in registers, 16-byte loads all requested before the first is
// looked at, and goes over them twice, for M and for the sums.  A row is cut into slices where there are few rows; a second launch joins
// the slices' (M, Z, sum, largest) and finishes.  All sums are in 32 bits, in the base of v_exp_f32: e^d = 2^((x - M) c), c = log2(e) / T.
//
// The largest entries.  Entries are ordered by a 64-bit key, above the value's bits as an ordered number (NaN above infinity, -0 as 0),
// below the complement of the index, so that keys differ and equal values go by the lowest index.  Each lane's largest value is known
// after the first pass; the top-th largest of a wavefront's 64 (found by bisection with ballots, no LDS) is a bound below which no entry
// of the result is, and few entries reach it: they are collected in LDS while the sums are taken, and each counts how many are above it.
// Where more of them reach the bound than LDS holds (equal values, a mask that leaves fewer than `top`), the bound is found exactly: a
// bisection over the keys, all entries counted in each step.  That takes the same time whatever the values are.
//
// -inf is no value: such entries take part neither in the sums nor in the first way, and a row or slice with fewer than `top` others
// goes the second.  NaN or +inf make Z NaN, and with it everything but the order.
#include "number_types.hpp"

namespace {

using namespace num;

constexpr int BLOCK = 256, WAVES = BLOCK / 64;
constexpr int MAX_TOP = 64;                    // a lane of a wavefront for each
constexpr int KEEP = 512;                      // collected entries
constexpr i64 MAX_V = (i64)1 << 24;

// a value as a number whose order is that of the values
__device__ __forceinline__ u32 ordered(float x) {
    if (!(x == x)) return 0xFFFFFFFFu;
    const u32 u = __float_as_uint(x + 0.0f);
    return u ^ ((u32)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ u64 key_of(float x, u32 index) { return (u64)ordered(x) << 32 | (u32)~index; }
__device__ __forceinline__ u32 index_of(u64 key) { return ~(u32)key; }
// the value behind a key
__device__ __forceinline__ float value_of(u64 key) {
    const u32 o = (u32)(key >> 32);
    if (o == 0xFFFFFFFFu) return __uint_as_float(0x7FC00000u);
    return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}

struct Shared {
    float most[WAVES], bound[WAVES], z[WAVES], w[WAVES];
    u32 count[2][WAVES];
    u32 kept;
    u64 keep[KEEP];
    u64 best[MAX_TOP];
};

struct Part {                                  // what a slice leaves, followed in memory by its `top` keys in falling order (0: none)
    float most, z, w, pad;
};

struct Args {
    const void *x;
    i64 v, ld;
    const i64 *tokens;
    float c, per_t;                            // log2(e) / T, 1 / T
    int top, slices;
    i64 per_slice;
    float *logprob, *entropy, *top_logprobs;
    i64 *top_tokens;
    Part *parts;                               // [row][slice]
    u64 *keys;                                 // [row][slice][top]
};

// the top-th largest of the lanes' 32-bit numbers
__device__ __forceinline__ u32 nth_of_lanes(u32 mine, int top) {
    u32 t = 0;
#pragma unroll 1
    for (int bit = 31; bit >= 0; --bit) {
        const u32 candidate = t | 1u << bit;
        if (__popcll(__ballot(mine >= candidate)) >= top) t = candidate;
    }
    return t;
}

// The top-th largest key, given how many of this thread's keys are at or above one; every thread has it.  Fewer than `top` keys: 0.
template <class Count>
__device__ u64 nth_key(Shared &sh, int top, Count count) {
    u64 t = 0;
#pragma unroll 1
    for (int bit = 63; bit >= 0; --bit) {
        const u64 candidate = t | 1ull << bit;
        u32 c = count(candidate);
#pragma unroll
        for (int d = 32; d; d >>= 1) c += __shfl_xor((int)c, d);
        if ((threadIdx.x & 63) == 0) sh.count[bit & 1][threadIdx.x / 64] = c;
        __syncthreads();
        c = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) c += sh.count[bit & 1][w];
        if (c >= (u32)top) t = candidate;
    }
    return t;
}

// the kept keys (at most KEEP) in falling order: the first `top` to sh.best, 0 behind the last
__device__ void rank_kept(Shared &sh, int top) {
    const u32 n = min(sh.kept, (u32)KEEP);
    if (threadIdx.x < top) sh.best[threadIdx.x] = 0;
    __syncthreads();
    for (u32 i = threadIdx.x; i < n; i += BLOCK) {
        const u64 mine = sh.keep[i];
        u32 above = 0;
        for (u32 j = 0; j < n; ++j) above += sh.keep[j] > mine;
        if (above < (u32)top) sh.best[above] = mine;
    }
    __syncthreads();
}

// (x - M) c; M = 0 where every entry is -inf
__device__ __forceinline__ float centre(float most) { return most == -INFINITY ? 0.0f : most; }

constexpr float LN2 = 0.69314718f;

template <int DT>
__device__ void finish(const Args &A, i64 row, float most, float z, float w, const u64 *best) {
    const float m = centre(most), logz = log2f(z) * LN2;
    // in nats from the start: (x - M) c would overflow for a mask of the type's lowest value, (x - M) / 1 does not
    auto lp_of = [&](float x) { return z != z ? z : x == -INFINITY ? x : (x - m) * A.per_t - logz; };
    if (threadIdx.x < A.top) {
        const u64 key = best[threadIdx.x];
        A.top_logprobs[row * A.top + threadIdx.x] = lp_of(value_of(key));
        A.top_tokens[row * A.top + threadIdx.x] = (i64)index_of(key);
    }
    if (threadIdx.x == BLOCK - 1) {
        const i64 t = A.tokens[row];
        const float x = t >= 0 && t < A.v ? (float)((const typename type<DT>::t *)A.x)[row * A.ld + t] : 0.0f;
        A.logprob[row] = t == -1 ? 0.0f : t < 0 || t >= A.v ? __uint_as_float(0x7FC00000u) : lp_of(x);
        A.entropy[row] = z == 0.0f ? 0.0f : logz - w / z * LN2;
    }
}

// A slice of a row (A.per_slice entries at most, R * 16 bytes a thread).
template <int DT, int R>
__global__ __launch_bounds__(BLOCK) void k_slice(Args A) {
    typedef typename type<DT>::t T;
    constexpr int PER = 16 / sizeof(T);
    __shared__ Shared sh;
    const i64 row = blockIdx.x / A.slices;
    const int slice = (int)(blockIdx.x % A.slices);
    const i64 first = slice * A.per_slice;
    const int n = (int)min(A.per_slice, A.v - first);
    const T *x = (const T *)A.x + row * A.ld + first;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;

    u32 raw[R][4];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int at = (r * BLOCK + threadIdx.x) * PER;
        if ((r + 1) * BLOCK * PER <= n) {      // the same for the workgroup, so that the loads stay together
            __builtin_memcpy(raw[r], x + at, 16);
        } else {
            T e[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i) e[i] = at + i < n ? x[at + i] : (T)-INFINITY;
            __builtin_memcpy(raw[r], e, 16);
        }
    }
    if (threadIdx.x == 0) sh.kept = 0;
    float most = -INFINITY;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < PER; ++e) most = fmaxf(most, element<DT>(raw[r], e));
    // the wavefront's bound: its top-th largest lane; none where fewer lanes have a value
    const u32 nth = A.top ? nth_of_lanes(ordered(most), A.top) : 0xFFFFFFFFu;
#pragma unroll
    for (int d = 32; d; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
    if (lane == 0) {
        sh.most[wave] = most;
        sh.bound[wave] = value_of((u64)nth << 32);
    }
    __syncthreads();
    float bound = sh.bound[0];
    most = sh.most[0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) {
        most = fmaxf(most, sh.most[i]);
        bound = fmaxf(bound, sh.bound[i]);
    }
    if (A.top == 0) bound = INFINITY;
    const float m = centre(most);
    float z = 0, w = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float biggest = -INFINITY;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const float v = element<DT>(raw[r], e), d = (v - m) * A.c, p = __builtin_amdgcn_exp2f(d);
            z += p;
            w += p * fmaxf(d, -1e30f);         // p = 0 where d is -inf
            biggest = fmaxf(biggest, v);
        }
        if (biggest >= bound && biggest > -INFINITY) {
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                const float v = element<DT>(raw[r], e);
                if (v >= bound && v > -INFINITY) {
                    const u32 i = atomicAdd(&sh.kept, 1u);
                    if (i < KEEP) sh.keep[i] = key_of(v, (u32)(first + (r * BLOCK + threadIdx.x) * PER + e));
                }
            }
        }
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        z += __shfl_xor(z, d);
        w += __shfl_xor(w, d);
    }
    if (lane == 0) {
        sh.z[wave] = z;
        sh.w[wave] = w;
    }
    __syncthreads();
    z = sh.z[0], w = sh.w[0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) {
        z += sh.z[i];
        w += sh.w[i];
    }
    if (A.top) {
        // too many at the bound, or fewer than there are to give, or a NaN that the comparisons above have passed over
        const u32 kept = sh.kept;
        if (kept > KEEP || kept < (u32)min(A.top, n) || z != z) {
            auto key_at = [&](int r, int e) -> u64 {
                const int at = (r * BLOCK + threadIdx.x) * PER + e;
                return at < n ? key_of(element<DT>(raw[r], e), (u32)(first + at)) : 0;
            };
            const u64 least = nth_key(sh, min(A.top, n), [&](u64 t) {
                u32 c = 0;
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int e = 0; e < PER; ++e) c += key_at(r, e) >= t;
                return c;
            });
            __syncthreads();
            if (threadIdx.x == 0) sh.kept = 0;
            __syncthreads();
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < PER; ++e)
                    if (key_at(r, e) >= least && key_at(r, e)) sh.keep[atomicAdd(&sh.kept, 1u)] = key_at(r, e);
            __syncthreads();
        }
        rank_kept(sh, A.top);
    }
    if (A.slices == 1) {
        finish<DT>(A, row, most, z, w, sh.best);
    } else {
        if (threadIdx.x == 0) A.parts[blockIdx.x] = {most, z, w, 0.0f};
        if (threadIdx.x < A.top) A.keys[(i64)blockIdx.x * A.top + threadIdx.x] = sh.best[threadIdx.x];
    }
}

// The slices of a row as one.
template <int DT>
__global__ __launch_bounds__(BLOCK) void k_join(Args A) {
    __shared__ Shared sh;
    const i64 row = blockIdx.x;
    const Part *parts = A.parts + row * A.slices;
    const u64 *keys = A.keys + row * A.slices * A.top;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = A.slices * A.top;
    float most = -INFINITY;
    for (int i = threadIdx.x; i < A.slices; i += BLOCK) most = fmaxf(most, parts[i].most);
#pragma unroll
    for (int d = 32; d; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
    u64 mine = 0;
    for (int i = threadIdx.x; i < n; i += BLOCK) mine = max(mine, keys[i]);
    const u32 nth = A.top ? nth_of_lanes((u32)(mine >> 32), A.top) : 0;
    if (threadIdx.x == 0) sh.kept = 0;
    if (lane == 0) {
        sh.most[wave] = most;
        sh.count[0][wave] = nth;
    }
    __syncthreads();
    most = sh.most[0];
    u32 bound = sh.count[0][0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) {
        most = fmaxf(most, sh.most[i]);
        bound = max(bound, sh.count[0][i]);
    }
    __syncthreads();
    const float m = centre(most);
    float z = 0, w = 0;
    for (int i = threadIdx.x; i < A.slices; i += BLOCK) {
        // sums relative to the slice's own largest entry: shift = (its - the row's) c, e^d d = e^d_own e^shift (d_own + shift)
        const float shift = fmaxf((centre(parts[i].most) - m) * A.c, -1e30f), p = __builtin_amdgcn_exp2f(shift), zi = parts[i].z;
        if (zi == 0.0f) continue;              // nothing but -inf
        z += p * zi;
        w += p == 0.0f ? 0.0f : p * (parts[i].w + zi * shift);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        z += __shfl_xor(z, d);
        w += __shfl_xor(w, d);
    }
    if (lane == 0) {
        sh.z[wave] = z;
        sh.w[wave] = w;
    }
    for (int i = threadIdx.x; i < n; i += BLOCK) {
        const u64 key = keys[i];
        if (key && (u32)(key >> 32) >= bound) {
            const u32 at = atomicAdd(&sh.kept, 1u);
            if (at < KEEP) sh.keep[at] = key;
        }
    }
    __syncthreads();
    z = sh.z[0], w = sh.w[0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) {
        z += sh.z[i];
        w += sh.w[i];
    }
    if (A.top) {
        if (sh.kept > KEEP) {
            const u64 least = nth_key(sh, A.top, [&](u64 t) {
                u32 c = 0;
                for (int i = threadIdx.x; i < n; i += BLOCK) c += keys[i] >= t;
                return c;
            });
            __syncthreads();
            if (threadIdx.x == 0) sh.kept = 0;
            __syncthreads();
            for (int i = threadIdx.x; i < n; i += BLOCK)
                if (keys[i] >= least && keys[i]) sh.keep[atomicAdd(&sh.kept, 1u)] = keys[i];
            __syncthreads();
        }
        rank_kept(sh, A.top);
    }
    finish<DT>(A, row, most, z, w, sh.best);
}

struct Plan {
    int r, slices;
    i64 per_slice;
    size_t ws_bytes;
};

// One slice a row where the rows fill the chip; else the shortest slices that four workgroups a CU take at once.
Plan make_plan(i64 m, i64 v, int dtype, int top) {
    const i64 unit = (i64)BLOCK * 16 / size_of(dtype);
    Plan L;
    for (L.r = 1; L.r < 16; L.r *= 2)
        if ((v + unit * L.r - 1) / (unit * L.r) * m <= 1024) break;
    L.per_slice = unit * L.r;
    L.slices = (int)((v + L.per_slice - 1) / L.per_slice);
    L.ws_bytes = L.slices > 1 ? (size_t)m * L.slices * (sizeof(Part) + 8 * top) + vi::WS_SLACK : 0;
    return L;
}

template <int DT>
void launch(const Plan &L, const Args &A, i64 m, hipStream_t s) {
    const dim3 grid((unsigned)(m * L.slices));
    if (L.r == 1) hipLaunchKernelGGL((k_slice<DT, 1>), grid, dim3(BLOCK), 0, s, A);
    if (L.r == 2) hipLaunchKernelGGL((k_slice<DT, 2>), grid, dim3(BLOCK), 0, s, A);
    if (L.r == 4) hipLaunchKernelGGL((k_slice<DT, 4>), grid, dim3(BLOCK), 0, s, A);
    if (L.r == 8) hipLaunchKernelGGL((k_slice<DT, 8>), grid, dim3(BLOCK), 0, s, A);
    if (L.r == 16) hipLaunchKernelGGL((k_slice<DT, 16>), grid, dim3(BLOCK), 0, s, A);
    if (L.slices > 1) hipLaunchKernelGGL(k_join<DT>, dim3((unsigned)m), dim3(BLOCK), 0, s, A);
}

}  // namespace

extern "C" size_t vi_token_logprobs_workspace_bytes(int dtype, int64_t m, int64_t v, int top) {
    if (!is_float(dtype) || m <= 0 || v <= 0 || v > MAX_V || top < 0 || top > MAX_TOP) return 0;
    return make_plan(m, v, dtype, top).ws_bytes;
}

extern "C" int vi_token_logprobs(int dtype, const void *logits, int64_t m, int64_t v, int64_t ld, const int64_t *tokens, float temperature,
                                 int top, float *logprob, float *entropy, float *top_logprobs, int64_t *top_tokens, void *ws,
                                 size_t ws_bytes, void *stream) {
    const char *who = "vi_token_logprobs";
    if (!is_float(dtype)) return vi::fail(VI_EINVAL, "%s: dtype %d is none of VI_F32, VI_BF16, VI_F16", who, dtype);
    if (m < 0 || v < 1 || v > MAX_V) return vi::fail(VI_EINVAL, "%s: %lld rows of %lld logits (1 to %lld)", who, (long long)m, (long long)v, (long long)MAX_V);
    if (ld < v) return vi::fail(VI_EINVAL, "%s: rows of %lld logits %lld apart", who, (long long)v, (long long)ld);
    if (top < 0 || top > MAX_TOP || top > v) return vi::fail(VI_EINVAL, "%s: the %d largest of %lld (%d at most)", who, top, (long long)v, MAX_TOP);
    if (!(temperature >= 1e-3f && temperature <= 1e3f)) return vi::fail(VI_EINVAL, "%s: temperature %g", who, (double)temperature);
    if (m == 0) return VI_OK;
    if (!logits || !tokens || !logprob || !entropy || (top && (!top_logprobs || !top_tokens))) return vi::fail(VI_EINVAL, "%s: null pointer", who);
    const Plan L = make_plan(m, v, dtype, top);
    if (m > 0x7FFFFFFF / L.slices) return vi::fail(VI_EINVAL, "%s: %lld rows of %lld logits", who, (long long)m, (long long)v);
    if (ws_bytes < L.ws_bytes || (L.ws_bytes && !ws)) return vi::fail(VI_ENOMEM, "%s: workspace %zu < %zu bytes", who, ws_bytes, L.ws_bytes);
    Args A = {};
    A.x = logits, A.v = v, A.ld = ld, A.tokens = tokens, A.c = 1.44269504f / temperature, A.per_t = 1.0f / temperature, A.top = top, A.slices = L.slices, A.per_slice = L.per_slice;
    A.logprob = logprob, A.entropy = entropy, A.top_logprobs = top_logprobs, A.top_tokens = top_tokens;
    A.parts = (Part *)vi::align16(ws);
    A.keys = (u64 *)(A.parts + m * L.slices);
    if (dtype == VI_F32) launch<VI_F32>(L, A, m, (hipStream_t)stream);
    if (dtype == VI_BF16) launch<VI_BF16>(L, A, m, (hipStream_t)stream);
    if (dtype == VI_F16) launch<VI_F16>(L, A, m, (hipStream_t)stream);
    VI_LAUNCH_CHECK(who);
    return VI_OK;
}
