// Rows of floats to 8-bit integers with a scale each.
//
//     A = max |x_j|    s = A / 127    r = 127 / A (both rounded to 32 bits)    q_j = rint(x_j r), half to even
//
// The product x_j r is rounded to 32 bits before rint: one multiplication an element, and |q| <= 127 since |x_j| <= A.
// A row whose scale would be no normal number (A < 127 2^-126) is zero: its r would overflow.  A NaN or an infinity makes the
// row's scale NaN and its integers zero, so that it shows in every product with them.
//
// Memory bounds it: a row stays in registers between the two looks at it, so it is read once.  32000 x 4096 float32 132 us, 5.0 TB/s in and
// out, which a large copy reaches too (116 us over the same two inputs again and again, part of which stays in the last-level cache);
// 1000 x 11008 bfloat16 9.4 us, 3.5 TB/s (one round of workgroups); one row of 4096 2.1 us.
#include "number_types.hpp"

namespace {

using namespace num;

constexpr int BLOCK = 256;
constexpr int CHUNK = 8;                       // neighbouring entries of a thread: 16 or 32 bytes in, 8 out
constexpr i64 MAX_ROWS = 1 << 23;              // of a launch, which has less than 2^32 threads
constexpr int MAX_CHUNKS = 8;                  // of a thread, in registers between the two looks at them

// Eight entries as they come, in four words (16-bit types) or eight.
template <int DT> struct Entries { u32 w[DT == VI_F32 ? 8 : 4]; };

template <int DT>
__device__ __forceinline__ Entries<DT> load_entries(const typename type<DT>::t *x) {
    return load_any<Entries<DT>>(x);
}
// the first `n` of them, zeros behind
template <int DT>
__device__ __forceinline__ Entries<DT> load_entries(const typename type<DT>::t *x, i64 n) {
    typename type<DT>::t e[CHUNK];
#pragma unroll
    for (int i = 0; i < CHUNK; ++i) e[i] = i < n ? x[i] : (typename type<DT>::t)0.0f;
    Entries<DT> v;
    __builtin_memcpy(&v, e, sizeof(v));
    return v;
}

// The sizes of the entries as bit patterns, which are in the order of the sizes, infinity above every number and NaN above that: 16-bit
// types two at a time.
typedef unsigned short v2h __attribute__((ext_vector_type(2)));
template <int DT>
__device__ __forceinline__ void widen(u32 &top, const Entries<DT> &v) {
#pragma unroll
    for (int i = 0; i < (DT == VI_F32 ? 8 : 4); ++i) {
        if constexpr (DT == VI_F32) {
            top = max(top, v.w[i] & 0x7FFFFFFFu);
        } else {
            const v2h a = __builtin_bit_cast(v2h, top), b = __builtin_bit_cast(v2h, v.w[i] & 0x7FFF7FFFu);
            top = __builtin_bit_cast(u32, __builtin_elementwise_max(a, b));
        }
    }
}
// the largest as a float's bit pattern
template <int DT>
__device__ __forceinline__ u32 widest(u32 top) {
    if constexpr (DT == VI_F32) {
        return top;
    } else {
        const unsigned short h = (unsigned short)max(top >> 16, top & 0xFFFFu);
        return __float_as_uint((float)__builtin_bit_cast(typename type<DT>::t, h));
    }
}

// How a row is rounded.
struct Scale {
    float r;
    u32 mask;                                  // of the integers: none where the row has no scale
};
// top: the row's largest size; the row's first thread writes the scale
__device__ __forceinline__ Scale scale_of(u32 top, float *out, bool first) {
    const float most = __uint_as_float(top);
    const bool bad = top >= 0x7F800000u, none = !bad && most < 127.0f * 0x1p-126f;
    if (first) *out = bad ? __uint_as_float(0x7FC00000u) : none ? 0.0f : most / 127.0f;
    return {bad || none ? 0.0f : 127.0f / most, bad ? 0u : 0xFFFFFFFFu};
}

// x r rounded to 32 bits, then to an integer by an addition whose result has units of one: its low byte is the integer's
template <int DT>
__device__ __forceinline__ u64 round_entries(const Entries<DT> &v, const Scale &s) {
    u32 b[CHUNK];
#pragma unroll
    for (int i = 0; i < CHUNK; ++i) {
        float x;
        if constexpr (DT == VI_F32) x = __uint_as_float(v.w[i]);
        else x = element<DT>(v.w, i);
        b[i] = __float_as_uint(x * s.r + 12582912.0f);
    }
    u32 o[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const u32 lo = __builtin_amdgcn_perm(b[4 * h + 1], b[4 * h], 0x0C0C0400u), hi = __builtin_amdgcn_perm(b[4 * h + 3], b[4 * h + 2], 0x0C0C0400u);
        o[h] = __builtin_amdgcn_perm(hi, lo, 0x05040100u) & s.mask;
    }
    return (u64)o[1] << 32 | o[0];
}

__device__ __forceinline__ void store_bytes(signed char *q, u64 v, i64 n) {
    if (n >= CHUNK) {
        store_any(q, v);
    } else {
        for (int i = 0; i < n; ++i) q[i] = (signed char)(v >> (8 * i));
    }
}

// the largest of LANES neighbouring lanes
template <int LANES>
__device__ __forceinline__ u32 most_of(u32 v) {
#pragma unroll
    for (int d = LANES / 2; d; d >>= 1) v = max(v, (u32)__shfl_xor((int)v, d));
    return v;
}

// THREADS to a row, R chunks a thread: the row is read once, all loads requested before the first is looked at.
template <int DT, int THREADS, int R>
__global__ __launch_bounds__(BLOCK) void k_quantize(const typename type<DT>::t *x, i64 m, i64 k, i64 ldx, signed char *q, i64 ldq, float *scale) {
    __shared__ u32 seen[BLOCK / 64];
    const int t = threadIdx.x % THREADS;
    const i64 row = (i64)blockIdx.x * (BLOCK / THREADS) + threadIdx.x / THREADS;
    if (THREADS < BLOCK && row >= m) return;   // no barrier below
    x += row * ldx;
    q += row * ldq;
    Entries<DT> v[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const i64 at = (i64)(r * THREADS + t) * CHUNK;
        // the first test is the same for the workgroup, so that its loads stay together
        if ((i64)(r + 1) * THREADS * CHUNK <= k || at + CHUNK <= k) v[r] = load_entries<DT>(x + at);
        else v[r] = load_entries<DT>(x + at, k - at);
    }
    u32 top = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) widen<DT>(top, v[r]);
    top = most_of<(THREADS < 64 ? THREADS : 64)>(widest<DT>(top));
    if constexpr (THREADS == BLOCK) {
        if ((threadIdx.x & 63) == 0) seen[threadIdx.x / 64] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < BLOCK / 64; ++w) top = max(top, seen[w]);
    }
    const Scale s = scale_of(top, scale + row, t == 0);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const i64 at = (i64)(r * THREADS + t) * CHUNK;
        store_bytes(q + at, round_entries<DT>(v[r], s), k - at);
    }
}

// Longer rows, read twice: the second time from the L2.
template <int DT>
__global__ __launch_bounds__(BLOCK) void k_quantize_long(const typename type<DT>::t *x, i64 k, i64 ldx, signed char *q, i64 ldq, float *scale) {
    __shared__ u32 seen[BLOCK / 64];
    const i64 row = blockIdx.x, whole = k / CHUNK * CHUNK;
    x += row * ldx;
    q += row * ldq;
    u32 top = 0;
#pragma unroll 4
    for (i64 at = (i64)threadIdx.x * CHUNK; at < whole; at += BLOCK * CHUNK) widen<DT>(top, load_entries<DT>(x + at));
    if (threadIdx.x == 0) widen<DT>(top, load_entries<DT>(x + whole, k - whole));
    top = most_of<64>(widest<DT>(top));
    if ((threadIdx.x & 63) == 0) seen[threadIdx.x / 64] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < BLOCK / 64; ++w) top = max(top, seen[w]);
    const Scale s = scale_of(top, scale + row, threadIdx.x == 0);
#pragma unroll 4
    for (i64 at = (i64)threadIdx.x * CHUNK; at < whole; at += BLOCK * CHUNK) store_any(q + at, round_entries<DT>(load_entries<DT>(x + at), s));
    if (threadIdx.x == 0 && whole < k) store_bytes(q + whole, round_entries<DT>(load_entries<DT>(x + whole, k - whole), s), k - whole);
}

template <int DT>
void launch(const void *px, i64 m, i64 k, i64 ldx, int8_t *pq, i64 ldq, float *scale, hipStream_t s) {
    typedef typename type<DT>::t T;
    const T *x = (const T *)px;
    signed char *q = (signed char *)pq;
    // Fewer threads a row where rows are short and fill the chip with them: 32000 x 1024 bfloat16 17.0 us with a wavefront a row, 30000 x
    // 102 float16 5.4 us with 16 lanes, 11.8 with a wavefront.
    const int threads = m >= 1024 && k <= 16 * CHUNK * 2 ? 16 : m >= 2048 && k <= 64 * CHUNK * 4 ? 64 : BLOCK;
    const i64 chunks = (k + threads * CHUNK - 1) / (threads * CHUNK);
#define GO(T, R) hipLaunchKernelGGL((k_quantize<DT, T, R>), dim3((unsigned)((m + BLOCK / T - 1) / (BLOCK / T))), dim3(BLOCK), 0, s, x, m, k, ldx, q, ldq, scale)
    if (threads == 16) {
        if (chunks <= 1) GO(16, 1);
        else GO(16, 2);
    } else if (threads == 64) {
        if (chunks <= 1) GO(64, 1);
        else if (chunks <= 2) GO(64, 2);
        else GO(64, 4);
    } else if (chunks <= 1) GO(BLOCK, 1);
    else if (chunks <= 2) GO(BLOCK, 2);
    else if (chunks <= 4) GO(BLOCK, 4);
    else if (chunks <= 6) GO(BLOCK, 6);
    else if (chunks <= MAX_CHUNKS) GO(BLOCK, MAX_CHUNKS);
    else hipLaunchKernelGGL((k_quantize_long<DT>), dim3((unsigned)m), dim3(BLOCK), 0, s, x, k, ldx, q, ldq, scale);
#undef GO
}

}  // namespace

extern "C" int vi_quantize_rows(int dtype, const void *x, int64_t m, int64_t k, int64_t ldx, int8_t *q, int64_t ldq, float *scale,
                                void *stream) {
    if (!is_float(dtype)) return vi::fail(VI_EINVAL, "vi_quantize_rows: dtype %d is none of VI_F32, VI_BF16, VI_F16", dtype);
    if (m < 0 || k < 0 || m > 0x7FFFFFFF) return vi::fail(VI_EINVAL, "vi_quantize_rows: %lld rows of %lld", (long long)m, (long long)k);
    if (ldx < k || ldq < k) return vi::fail(VI_EINVAL, "vi_quantize_rows: rows of %lld, %lld and %lld apart", (long long)k, (long long)ldx, (long long)ldq);
    if (m == 0) return VI_OK;
    if (!scale || (k && (!x || !q))) return vi::fail(VI_EINVAL, "vi_quantize_rows: null pointer");
    hipStream_t s = (hipStream_t)stream;
    for (i64 first = 0; first < m; first += MAX_ROWS) {
        const void *from = (const char *)x + first * ldx * size_of(dtype);
        const i64 rows = m - first < MAX_ROWS ? m - first : MAX_ROWS;
        if (dtype == VI_F32) launch<VI_F32>(from, rows, k, ldx, q + first * ldq, ldq, scale + first, s);
        if (dtype == VI_BF16) launch<VI_BF16>(from, rows, k, ldx, q + first * ldq, ldq, scale + first, s);
        if (dtype == VI_F16) launch<VI_F16>(from, rows, k, ldx, q + first * ldq, ldq, scale + first, s);
        VI_LAUNCH_CHECK("quantize_rows");
    }
    return VI_OK;
}
