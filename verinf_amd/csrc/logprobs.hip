// Log probabilities of given tokens under rows of logits, the rows' entropies and their largest entries.
//
//     M = max_j x_j    d_j = (x_j - M) / T    Z = sum e^d_j    lp(j) = d_j - log Z    H = log Z - (sum e^d_j d_j) / Z
//
// One pass over the logits: a workgroup keeps its slice of a row in registers, 16-byte loads all requested before the first is
// looked at, and goes over them twice, for M and for the sums.  A row is cut into slices where there are few rows; a second
// launch joins the slices' (M, Z, sum, largest) and finishes.  All sums are in 32 bits, in the base of v_exp_f32: e^d = 2^((x - M) c), c = log2(e) / T,
// c and the product rounded to 32 bits and the exponential by the hardware, about 1e-7 of a log probability in all (0.5e-7 with expf).
//
// The largest entries.  Entries are ordered by a 64-bit key, above the value's bits as an ordered number (NaN above infinity, -0 as 0),
// below the complement of the index, so that keys differ and equal values go by the lowest index.  Each thread's largest value is known
// after the first pass; the top-th largest of them (or a little less: bisection with ballots, ended once few enough reach it) is a
// bound below which no entry of the result is, and hardly more than `top` entries reach it: they are collected in LDS while the sums
// are taken, and each counts how many are above it.  Where more reach the bound than LDS holds (equal values), another is found by a
// bisection over the keys, all entries counted in each step, until few enough reach it: at the latest with the exact one.  (That branch alone
// has registers in scratch memory, 23 to 55 of them with 16 loads a thread.)
//
// 1000 x 32000 bfloat16, 5 largest: 21-23 us, 2.9 TB/s; 4096 rows 60 us, 4.3 TB/s.  A wave's 128 entries a lane are some 11 operations and an
// exponential each, 10 us of the CUs' time for 1000 rows, which comes behind the loads where all rows are there at once, and under them where
// there are more.  Sums taken as the loads arrive, relative to an entry of each thread, were no faster (23.5 us, 64).
//
// -inf is no value: such entries are not in the sums nor collected.  Where there are fewer than `top` others the lowest indexes of -inf
// fill up, which are among the first `top` entries (1000 x 50257 float16, 8 largest: 39 us with 5 entries allowed, 35 with 500).  NaN or +inf
// make Z NaN, and with it everything but the order.
#include <cfloat>

#include "number_types.hpp"

namespace {

using namespace num;

constexpr int BLOCK = 256, WIDE = 1024;         // threads
constexpr int MAX_TOP = 64;                    // a lane of a wavefront for each
constexpr int KEEP = 512, KEEP_VECTORS = 128;  // collected entries, and 16 bytes of them
constexpr i64 MAX_V = (i64)1 << 24;
constexpr int CUS = 256;                       // of a whole card; on a part of one the choice of slices costs time, nothing else
constexpr i64 MAX_ROWS = 1 << 23;              // of a launch, and slices of rows: it has less than 2^32 threads
constexpr int MAX_R = 16, MAX_WIDE_R = 8;      // 16-byte loads a thread

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

template <int B>
struct Shared {
    alignas(16) u32 largest[B];                // of each thread
    float z[B / 64], w[B / 64];
    u32 count[2][B / 64];
    u32 kept, vectors;
    u64 keep[KEEP];
    u64 best[MAX_TOP];
    u32 vector[KEEP_VECTORS][4], vector_at[KEEP_VECTORS];              // 16 bytes of entries one of which reaches the bound, and where they are
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

// The largest of all threads' numbers, and a number that at least `top` of them reach, and no more than SPARE others where that is
// possible.  `mine` is ordered(); a barrier inside.
// Of more than 256 threads, the larger of every B / 256 count as one.
constexpr int SPARE = 16;
template <int B>
__device__ __forceinline__ void look_at_all(Shared<B> &sh, u32 mine, int top, u32 *most, u32 *bound) {
    typedef u32 v4u __attribute__((ext_vector_type(4)));
    sh.largest[threadIdx.x] = mine;
    __syncthreads();
    v4u v = *(const v4u *)&sh.largest[(threadIdx.x & 63) * 4];
#pragma unroll
    for (int i = 1; i < B / 256; ++i) v = __builtin_elementwise_max(v, *(const v4u *)&sh.largest[i * 256 + (threadIdx.x & 63) * 4]);
    u32 m = max(max(v[0], v[1]), max(v[2], v[3]));
#pragma unroll
    for (int d = 32; d; d >>= 1) m = max(m, (u32)__shfl_xor((int)m, d));
    *most = m;
    u32 t = 0;
    if (top) {
#pragma unroll 1
        for (u32 bit = 1u << 31; bit; bit >>= 1) {
            const u32 at = t | bit;
            int c = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) c += __popcll(__ballot(v[i] >= at));
            if (c >= top) {
                t = at;
                if (c <= top + SPARE) break;
            }
        }
    }
    *bound = t;
}

// how many there are in the workgroup, of what each wavefront has counted; `turn` alternates
template <int B>
__device__ __forceinline__ u32 count_all(Shared<B> &sh, u32 of_wave, int turn) {
    if ((threadIdx.x & 63) == 0) sh.count[turn & 1][threadIdx.x / 64] = of_wave;
    __syncthreads();
    u32 c = 0;
#pragma unroll
    for (int w = 0; w < B / 64; ++w) c += sh.count[turn & 1][w];
    return c;
}

// A key that at least `top` of all entries' keys reach and at most KEEP.  above(t): how many of the wavefront's entries have an ordered
// value of t or more; equal(t, i): how many have t itself and an index of i or less.
template <int B, class Above, class Equal>
__device__ u64 bound_key(Shared<B> &sh, int top, Above above, Equal equal) {
    u32 t = 0;
    int turn = 0;
#pragma unroll 1
    for (u32 bit = 1u << 31; bit; bit >>= 1) {
        const u32 c = count_all(sh, above(t | bit), turn++);
        if (c >= (u32)top) {
            t |= bit;
            if (c <= KEEP) return (u64)t << 32;
        }
    }
    // t is the top-th largest value and more have it than are needed: those of the lowest indexes
    const u32 more = t == 0xFFFFFFFFu ? 0 : count_all(sh, above(t + 1), turn++);
    u32 index = 0xFFFFFFFFu;                   // the least so far that is enough
#pragma unroll 1
    for (u32 bit = 1u << 31; bit; bit >>= 1) {
        const u32 c = more + count_all(sh, equal(t, index ^ bit), turn++);
        if (c >= (u32)top) {
            index ^= bit;
            if (c <= KEEP) break;
        }
    }
    return (u64)t << 32 | (u32)~index;
}

// the kept keys (at most KEEP) in falling order: the first `top` to sh.best, 0 behind the last
template <int B>
__device__ void rank_kept(Shared<B> &sh, int top) {
    const u32 n = min(sh.kept, (u32)KEEP);
    if (threadIdx.x < top) sh.best[threadIdx.x] = 0;
    __syncthreads();
    for (u32 i = threadIdx.x; i < n; i += B) {
        const u64 mine = sh.keep[i];
        u32 above = 0;
#pragma unroll 8
        for (u32 j = 0; j < n; ++j) above += sh.keep[j] > mine;
        if (above < (u32)top) sh.best[above] = mine;
    }
    __syncthreads();
}

// (x - M) c; M = 0 where every entry is -inf
__device__ __forceinline__ float centre(float most) { return most == -INFINITY ? 0.0f : most; }

constexpr float LN2 = 0.69314718f;

// The logit of the row's token, which the last thread asks for early; what it does not find is left to finish.
struct Asked {
    i64 token;
    float x;
};
template <int DT>
__device__ __forceinline__ Asked ask(const Args &A, i64 row) {
    Asked a = {-1, 0.0f};
    if (threadIdx.x == 255) {
        a.token = A.tokens[row];
        if (a.token >= 0 && a.token < A.v) a.x = (float)((const typename type<DT>::t *)A.x)[row * A.ld + a.token];
    }
    return a;
}

__device__ void finish(const Args &A, i64 row, float most, float z, float w, const u64 *best, const Asked &asked) {
    const float m = centre(most), logz = log2f(z) * LN2;
    // in nats from the start: (x - M) c would overflow for a mask of the type's lowest value, (x - M) / 1 does not; and by halves, since x - M
    // may be twice what 32 bits hold
    auto lp_of = [&](float x) { return z != z ? z : x == -INFINITY ? x : (0.5f * x - 0.5f * m) * (2.0f * A.per_t) - logz; };
    if (threadIdx.x < A.top) {
        const u64 key = best[threadIdx.x];
        A.top_logprobs[row * A.top + threadIdx.x] = lp_of(value_of(key));
        A.top_tokens[row * A.top + threadIdx.x] = (i64)index_of(key);
    }
    if (threadIdx.x == 255) {
        const i64 t = asked.token;
        A.logprob[row] = t == -1 ? 0.0f : t < 0 || t >= A.v ? __uint_as_float(0x7FC00000u) : lp_of(asked.x);
        A.entropy[row] = z == 0.0f ? 0.0f : logz - w / z * LN2;
    }
}

// The largest of entries, from their bits: as signed numbers those of positive values are in order, and any is above those of negative
// values, which are in the opposite order as unsigned numbers.  Two entries an operation in 16-bit types.  A NaN may pass for the largest
// (the sums become NaN then) or be passed over.
template <int DT>
struct Largest;
template <>
struct Largest<VI_F32> {
    int up = (int)0x80000000;
    u32 down = 0xFFFFFFFFu;
    Largest() = default;
    // a value to be reached
    __device__ explicit Largest(float v) : up(__float_as_int(v)), down(__float_as_uint(v)) {}
    __device__ __forceinline__ void take(const u32 (&w)[4]) {
        up = max(max(up, max((int)w[0], (int)w[1])), max((int)w[2], (int)w[3]));
        down = min(min(down, min(w[0], w[1])), min(w[2], w[3]));
    }
    __device__ __forceinline__ float value() const { return __uint_as_float(up >= 0 ? (u32)up : down); }
    __device__ __forceinline__ bool reached(const u32 (&w)[4]) const {
        if (up >= 0) return max(max((int)w[0], (int)w[1]), max((int)w[2], (int)w[3])) >= up;
        return min(min(w[0], w[1]), min(w[2], w[3])) <= down;
    }
};
typedef short v2i16 __attribute__((ext_vector_type(2)));
typedef unsigned short v2u16 __attribute__((ext_vector_type(2)));
template <int DT>
struct Largest {
    v2i16 up = {-32768, -32768};
    v2u16 down = {65535, 65535};
    Largest() = default;
    __device__ explicit Largest(float v) {
        const unsigned short h = __builtin_bit_cast(unsigned short, (typename type<DT>::t)v);       // exact: it is an entry's, or infinite
        up = v2i16{(short)h, (short)h};
        down = v2u16{h, h};
    }
    static __device__ __forceinline__ v2i16 greatest(const u32 (&w)[4]) {
        return __builtin_elementwise_max(__builtin_elementwise_max(__builtin_bit_cast(v2i16, w[0]), __builtin_bit_cast(v2i16, w[1])),
                                         __builtin_elementwise_max(__builtin_bit_cast(v2i16, w[2]), __builtin_bit_cast(v2i16, w[3])));
    }
    static __device__ __forceinline__ v2u16 least(const u32 (&w)[4]) {
        return __builtin_elementwise_min(__builtin_elementwise_min(__builtin_bit_cast(v2u16, w[0]), __builtin_bit_cast(v2u16, w[1])),
                                         __builtin_elementwise_min(__builtin_bit_cast(v2u16, w[2]), __builtin_bit_cast(v2u16, w[3])));
    }
    __device__ __forceinline__ void take(const u32 (&w)[4]) {
        up = __builtin_elementwise_max(up, greatest(w));
        down = __builtin_elementwise_min(down, least(w));
    }
    __device__ __forceinline__ float value() const {
        const short u = up[0] > up[1] ? up[0] : up[1];
        const unsigned short d = down[0] < down[1] ? down[0] : down[1];
        const u32 w[4] = {u >= 0 ? (u32)(unsigned short)u : (u32)d, 0, 0, 0};
        return element<DT>(w, 0);
    }
    __device__ __forceinline__ bool reached(const u32 (&w)[4]) const {
        if (up[0] >= 0) {
            const v2i16 g = greatest(w);
            return g[0] >= up[0] || g[1] >= up[0];
        }
        const v2u16 l = least(w);
        return l[0] <= down[0] || l[1] <= down[0];
    }
};

// What is made of the entries next is made of them anew: the compiler would keep floats or keys of all of them, up to 256 registers.
template <int R>
__device__ __forceinline__ void again(u32 (&raw)[R][4]) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(raw[r][i]));
}

// A slice of a row (A.per_slice entries at most, R * 16 bytes a thread).
template <int DT, int R, int B>
__global__ __launch_bounds__(B, 4) void k_slice(Args A) {
    typedef typename type<DT>::t T;
    constexpr int PER = 16 / sizeof(T);
    __shared__ Shared<B> sh;
    const i64 row = blockIdx.x / A.slices;
    const int slice = (int)(blockIdx.x % A.slices);
    const i64 first = slice * A.per_slice;
    const int n = (int)min(A.per_slice, A.v - first);
    const T *x = (const T *)A.x + row * A.ld + first;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;

    // all loads, then the last few entries where they fill no vector; -inf behind them
    u32 raw[R][4];
    constexpr u32 NONE = DT == VI_F32 ? 0xFF800000u : DT == VI_BF16 ? 0xFF80FF80u : 0xFC00FC00u;
    const int vectors = n / PER, ragged = n % PER;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = r * B + (int)threadIdx.x;
        if ((r + 1) * B <= vectors || i < vectors) {               // the first test is the same for the workgroup
            __builtin_memcpy(raw[r], x + i * PER, 16);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) raw[r][e] = NONE;
        }
    }
    u32 rest[4] = {NONE, NONE, NONE, NONE};
    const bool mine = ragged && (int)threadIdx.x == vectors % B;       // this thread has them, as its vector vectors / B
    if (mine) {
        T e[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) e[i] = i < ragged ? x[vectors * PER + i] : (T)-INFINITY;
        __builtin_memcpy(rest, e, 16);
    }
    Asked asked;
    if (A.slices == 1) asked = ask<DT>(A, row);
    if (threadIdx.x == 0) sh.kept = sh.vectors = 0;

    Largest<DT> top;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (mine && r == vectors / B) {
#pragma unroll
            for (int e = 0; e < 4; ++e) raw[r][e] = rest[e];
        }
        top.take(raw[r]);
    }
    u32 all, reach;
    look_at_all(sh, ordered(top.value()), A.top, &all, &reach);
    const float most = value_of((u64)all << 32), m = centre(most);
    // -inf does not reach it, nor once it is a number of the type; where none are asked for only +inf does, which does no harm
    constexpr float LOWEST = DT == VI_F32 ? -FLT_MAX : DT == VI_BF16 ? -0x1.FEp127f : -65504.0f;
    const float bound = A.top ? value_of((u64)max(reach, ordered(LOWEST)) << 32) : INFINITY;
    const Largest<DT> least(bound == 0.0f ? -0.0f : bound);        // 0.0 reaches -0.0 as well, but not the other way round: bits are compared
    float z = 0, w = 0;
    again(raw);
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const float d = (element<DT>(raw[r], e) - m) * A.c, p = __builtin_amdgcn_exp2f(d);
            z += p;
            w = fmaf(p, fmaxf(d, -1e30f), w);  // p = 0 where d is -inf
        }
        asm volatile("" : "+v"(z), "+v"(w));   // here: the compiler would take all exponentials behind all branches, with their arguments in registers until then
        if (least.reached(raw[r])) {           // which of them is looked at later: few come here, and this is in every place
            const u32 i = atomicAdd(&sh.vectors, 1u);
            if (i < KEEP_VECTORS) {
#pragma unroll
                for (int e = 0; e < 4; ++e) sh.vector[i][e] = raw[r][e];
                sh.vector_at[i] = (u32)(r * B + threadIdx.x) * PER;
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
    for (int i = 1; i < (B / 64); ++i) {
        z += sh.z[i];
        w += sh.w[i];
    }
    if (A.top) {
        const int give = min(A.top, n);
        const u32 vectors_kept = sh.vectors;
        for (u32 i = threadIdx.x; i < min(vectors_kept, (u32)KEEP_VECTORS) * PER; i += B) {
            const float v = element<DT>(sh.vector[i / PER], i % PER);
            if (v >= bound) {
                const u32 at = atomicAdd(&sh.kept, 1u);
                if (at < KEEP) sh.keep[at] = key_of(v, (u32)first + sh.vector_at[i / PER] + i % PER);
            }
        }
        __syncthreads();
        const u32 kept = sh.kept;
        if (vectors_kept > KEEP_VECTORS || kept > KEEP || z != z) {
            // too many at the bound, or a NaN that the comparisons above have passed over
            auto count = [&](auto test) {
                u32 c = 0, index = (u32)first + threadIdx.x * PER;
                again(raw);
                asm volatile("" : "+v"(index));
#pragma unroll
                for (int r = 0; r < R; ++r) {
#pragma unroll
                    for (int e = 0; e < PER; ++e) c += __popcll(__ballot(test(element<DT>(raw[r], e), index + (u32)(r * B * PER + e))));
                    asm volatile("" : "+s"(c), "+v"(index));           // one vector after the other: registers
                }
                return c;
            };
            auto above = [&](u32 t) {
                if (t > ordered(INFINITY)) return count([](float v, u32) { return v != v; });
                const float least = value_of((u64)t << 32);            // a NaN for numbers below -inf's: all are above
                return count([=](float v, u32) { return !(v < least); });
            };
            auto equal = [&](u32 t, u32 i) { return count([=](float v, u32 index) { return ordered(v) == t && index <= i; }); };
            const u64 least = bound_key(sh, give, above, equal);
            __syncthreads();
            if (threadIdx.x == 0) sh.kept = 0;
            __syncthreads();
            again(raw);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                u32 at = (u32)(r * B + threadIdx.x) * PER;
                asm volatile("" : "+v"(at));
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    const u64 key = key_of(element<DT>(raw[r], e), (u32)first + at + e);
                    if (key >= least && at + e < (u32)n) sh.keep[atomicAdd(&sh.kept, 1u)] = key;
                }
            }
            __syncthreads();
        } else if (kept < (u32)give) {
            __syncthreads();
            if (threadIdx.x < give && (float)x[threadIdx.x] == -INFINITY)
                sh.keep[atomicAdd(&sh.kept, 1u)] = key_of(-INFINITY, (u32)(first + threadIdx.x));
            __syncthreads();
        }
        rank_kept(sh, A.top);
    }
    if (A.slices == 1) {
        finish(A, row, most, z, w, sh.best, asked);
    } else {
        if (threadIdx.x == 0) A.parts[blockIdx.x] = {most, z, w, 0.0f};
        if (threadIdx.x < A.top) A.keys[(i64)blockIdx.x * A.top + threadIdx.x] = sh.best[threadIdx.x];
    }
}

// The slices of a row as one.
template <int DT>
__global__ __launch_bounds__(BLOCK) void k_join(Args A) {
    __shared__ Shared<BLOCK> sh;
    const i64 row = blockIdx.x;
    const Part *parts = A.parts + row * A.slices;
    const u64 *keys = A.keys + row * A.slices * A.top;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = A.slices * A.top;
    const Asked asked = ask<DT>(A, row);
    float most = -INFINITY;
    for (int i = threadIdx.x; i < A.slices; i += BLOCK) most = fmaxf(most, parts[i].most);
#pragma unroll
    for (int d = 32; d; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
    u64 mine = 0;
    for (int i = threadIdx.x; i < n; i += BLOCK) mine = max(mine, keys[i]);
    if (threadIdx.x == 0) sh.kept = 0;
    if (lane == 0) sh.z[wave] = most;
    u32 bound, largest;
    look_at_all(sh, (u32)(mine >> 32), A.top, &largest, &bound);
    most = sh.z[0];
#pragma unroll
    for (int i = 1; i < (BLOCK / 64); ++i) most = fmaxf(most, sh.z[i]);
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
    for (int i = 1; i < (BLOCK / 64); ++i) {
        z += sh.z[i];
        w += sh.w[i];
    }
    if (A.top) {
        if (sh.kept > KEEP) {
            auto count = [&](auto test) {
                u32 c = 0;
                for (int i = 0; i < n; i += BLOCK) c += __popcll(__ballot(i + (int)threadIdx.x < n && test(keys[i + threadIdx.x])));
                return c;
            };
            const u64 least = bound_key(sh, A.top, [&](u32 t) { return count([=](u64 key) { return (u32)(key >> 32) >= t; }); },
                                        [&](u32 t, u32 i) { return count([=](u64 key) { return (u32)(key >> 32) == t && index_of(key) <= i; }); });
            __syncthreads();
            if (threadIdx.x == 0) sh.kept = 0;
            __syncthreads();
            for (int i = threadIdx.x; i < n; i += BLOCK)
                if (keys[i] >= least && keys[i]) sh.keep[atomicAdd(&sh.kept, 1u)] = keys[i];
            __syncthreads();
        }
        rank_kept(sh, A.top);
    }
    finish(A, row, most, z, w, sh.best, asked);
}

struct Plan {
    int r, slices;
    bool wide;
    i64 per_slice;
    size_t ws_bytes;
};

// One slice a row where the rows fill the chip; one in a workgroup of 1024 threads where that holds it and there is a CU for each row (one launch: 1 x
// 32000 float32 8.4 us, 10.1 in slices; 200 x 5000 7.2, 11.5; 1000 x 32000 bfloat16 34, 22 with 256 threads a row); else the shortest slices
// that four workgroups a CU take at once.
Plan make_plan(i64 m, i64 v, int dtype, int top) {
    const i64 unit = (i64)BLOCK * 16 / size_of(dtype), wide = unit * (WIDE / BLOCK);
    Plan L = {};
    L.wide = v > unit && v <= wide * MAX_WIDE_R && m <= CUS;
    for (L.r = 1; L.r < (L.wide ? MAX_WIDE_R : MAX_R); L.r *= 2) {
        const i64 slices = (v + (L.wide ? wide : unit) * L.r - 1) / ((L.wide ? wide : unit) * L.r);
        if (slices == 1 || (!L.wide && slices * m <= 1024)) break;
    }
    L.per_slice = (L.wide ? wide : unit) * L.r;
    L.slices = (int)((v + L.per_slice - 1) / L.per_slice);
    L.ws_bytes = L.slices > 1 ? (size_t)m * L.slices * (sizeof(Part) + 8 * top) + vi::WS_SLACK : 0;
    return L;
}

template <int DT>
void launch(const Plan &L, const Args &A, i64 m, hipStream_t s) {
    const dim3 grid((unsigned)(m * L.slices));
#define GO(R, B) hipLaunchKernelGGL((k_slice<DT, R, B>), grid, dim3(B), 0, s, A)
    if (L.wide && L.r == 1) GO(1, WIDE);
    if (L.wide && L.r == 2) GO(2, WIDE);
    if (L.wide && L.r == 4) GO(4, WIDE);
    if (L.wide && L.r == 8) GO(8, WIDE);
    if (!L.wide && L.r == 1) GO(1, BLOCK);
    if (!L.wide && L.r == 2) GO(2, BLOCK);
    if (!L.wide && L.r == 4) GO(4, BLOCK);
    if (!L.wide && L.r == 8) GO(8, BLOCK);
    if (!L.wide && L.r == 16) GO(16, BLOCK);
#undef GO
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
    if (m > (L.slices > 1 ? MAX_ROWS / L.slices : 0x7FFFFFFF)) return vi::fail(VI_EINVAL, "%s: %lld rows of %lld logits", who, (long long)m, (long long)v);
    if (ws_bytes < L.ws_bytes || (L.ws_bytes && !ws)) return vi::fail(VI_ENOMEM, "%s: workspace %zu < %zu bytes", who, ws_bytes, L.ws_bytes);
    for (i64 first = 0; first < m; first += MAX_ROWS) {
        const i64 rows = m - first < MAX_ROWS ? m - first : MAX_ROWS;
        Args A = {};
        A.x = (const char *)logits + first * ld * size_of(dtype), A.v = v, A.ld = ld, A.tokens = tokens + first;
        A.c = 1.44269504f / temperature, A.per_t = 1.0f / temperature, A.top = top, A.slices = L.slices, A.per_slice = L.per_slice;
        A.logprob = logprob + first, A.entropy = entropy + first;
        A.top_logprobs = top ? top_logprobs + first * top : nullptr, A.top_tokens = top ? top_tokens + first * top : nullptr;
        if (L.slices > 1) {
            A.parts = (Part *)vi::align16(ws);
            A.keys = (u64 *)(A.parts + m * L.slices);
        }
        if (dtype == VI_F32) launch<VI_F32>(L, A, rows, (hipStream_t)stream);
        if (dtype == VI_BF16) launch<VI_BF16>(L, A, rows, (hipStream_t)stream);
        if (dtype == VI_F16) launch<VI_F16>(L, A, rows, (hipStream_t)stream);
        VI_LAUNCH_CHECK(who);
    }
    return VI_OK;
}
