// Rotary positions, and new tokens' keys and values into a paged cache.
//
//     a = p f_i    (x, y) -> (x cos a - y sin a, x sin a + y cos a) A
//
// Angles are whole numbers of 2^-64 turns: p steps_i mod 2^64 is exact for any p, where p f_i rounded to 32 bits is p 2^-24 off (6e-3 at 10^5).
// Sine and cosine are their Taylor series over an eighth of a turn to either side, 1e-7 off in 32 bits (1e-16 in 64); a workgroup takes each
// of its tokens' once for all heads, through LDS.
//
// Sixteen lanes have a head, so that a row of a cache leaves in one piece and its largest entry is theirs.
//
// What bounds them: memory where there is much to turn (4096 tokens of 32 heads of 128 fp16: 13 us, 5.1 TB/s, as a large copy); elsewhere one load behind the other
// (sequence, page, position, step), then the angles, then the heads: a token of 32 heads 2.6 us, 64 tokens into 8 heads of a bf16 cache 3.6, of 8 bits 4.0.  4096 tokens into 8 heads: bf16 10.9 us,
// 9.8 with nothing turned, where its bytes take 6.5; 8 bits 13.5 us, 11.6 with nothing turned, where its bytes take 5, so that angles in 64 bits are 2 of it and the integers another 2.  Asking
// for the next head ahead changes nothing; 32 heads, four times the bytes, take 40 us.
#include <type_traits>

#include "cache.hpp"

namespace {

using namespace kv;

constexpr int BLOCK = 256, LANES = 16, GROUPS = BLOCK / LANES;          // sixteen lanes to a head of a token
constexpr int MOST_PAIRS = 128;                // of a head
constexpr i64 MAX_BLOCKS = 1 << 23;            // of a launch, which has less than 2^32 threads

struct Turn {
    const u64 *steps;
    int rotated, interleaved;
    double amplitude;
};

template <class T> struct CosSin { T c, s; };

// cos and sin of phase 2^-64 turns, times the amplitude
__device__ __forceinline__ CosSin<float> turned(u64 phase, float amplitude) {
    const u32 quarter = (u32)((phase + (1ull << 61)) >> 62);
    const int r = (int)((i64)(phase - ((u64)quarter << 62)) >> 32);      // within an eighth of a turn, in 2^-32
    const float x = (float)r * (float)(6.283185307179586 * 0x1p-32), q = x * x;
    float s = fmaf(q, 2.7557319e-6f, -1.9841270e-4f), c = fmaf(q, -2.7557319e-7f, 2.4801587e-5f);
    s = fmaf(q, s, 8.3333333e-3f), c = fmaf(q, c, -1.3888889e-3f);
    s = fmaf(q, s, -1.6666667e-1f), c = fmaf(q, c, 4.1666667e-2f);
    c = fmaf(q, c, -0.5f);
    s = fmaf(q * x, s, x), c = fmaf(q, c, 1.0f);
    const float u = quarter & 1 ? s : c, v = quarter & 1 ? c : s;
    return {((quarter + 1) & 2 ? -u : u) * amplitude, (quarter & 2 ? -v : v) * amplitude};
}
__device__ __forceinline__ CosSin<double> turned(u64 phase, double amplitude) {
    const u32 quarter = (u32)((phase + (1ull << 61)) >> 62);
    const double x = (double)(i64)(phase - ((u64)quarter << 62)) * (6.283185307179586 * 0x1p-64), q = x * x;
    constexpr double S[] = {2.8114572543455206e-15, -7.647163731819816e-13, 1.6059043836821613e-10, -2.505210838544172e-8,
                            2.7557319223985893e-6,  -1.984126984126984e-4,  8.333333333333333e-3,   -0.16666666666666666};
    constexpr double C[] = {4.779477332387385e-14, -1.1470745597729725e-11, 2.08767569878681e-9, -2.755731922398589e-7,
                            2.48015873015873e-5,   -1.388888888888889e-3,   4.1666666666666664e-2, -0.5};
    double s = S[0], c = C[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) s = fma(q, s, S[i]), c = fma(q, c, C[i]);
    s = fma(q * x, s, x), c = fma(q, c, 1.0);
    const double u = quarter & 1 ? s : c, v = quarter & 1 ? c : s;
    return {((quarter + 1) & 2 ? -u : u) * amplitude, (quarter & 2 ? -v : v) * amplitude};
}

// A lane's part of a head: R units of VEC pairs, of the rotated columns or of those behind them, 16 units of neighbouring lanes apart.
// Values lie as they come: x[i], x[i + rotated / 2] as [i], [VEC + i], or as neighbours.
template <int VEC, int R>
struct Part {
    float v[R][2 * VEC];
};

// fixed-size copies of neighbouring numbers, as floats
template <int DT, int N>
__device__ __forceinline__ void get(float *to, const typename type<DT>::t *from) {
    typename type<DT>::t e[N];
    __builtin_memcpy(e, from, sizeof(e));
#pragma unroll
    for (int i = 0; i < N; ++i) to[i] = (float)e[i];
}
template <int DT, int N>
__device__ __forceinline__ void put(typename type<DT>::t *to, const float *from) {
    typename type<DT>::t e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = (typename type<DT>::t)from[i];
    __builtin_memcpy(to, e, sizeof(e));
}

// calls at(r, first, second, together) for the lane's units: `first` and `second` are where its halves begin, `together` whether they are one run
template <int VEC, int R, class At>
__device__ __forceinline__ void each_unit(int dim, int rotated, bool interleaved, int lane, At at) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int u = r * LANES + lane;
        if (u * 2 * VEC >= dim) continue;
        const bool apart = !interleaved && u * 2 * VEC < rotated;
        at(r, apart ? u * VEC : u * 2 * VEC, apart ? rotated / 2 + u * VEC : u * 2 * VEC + VEC, !apart);
    }
}

template <int DT, int VEC, int R>
__device__ __forceinline__ void load_part(Part<VEC, R> &p, const typename type<DT>::t *x, int dim, int rotated, bool interleaved, int lane) {
    each_unit<VEC, R>(dim, rotated, interleaved, lane, [&](int r, int first, int second, bool together) {
        if (together) {
            get<DT, 2 * VEC>(p.v[r], x + first);
        } else {
            get<DT, VEC>(p.v[r], x + first);
            get<DT, VEC>(p.v[r] + VEC, x + second);
        }
    });
}

__device__ __forceinline__ float fused(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double fused(double a, double b, double c) { return fma(a, b, c); }

template <class T, int VEC, int R>
__device__ __forceinline__ void turn_part(Part<VEC, R> &p, const CosSin<T> *table, int rotated, bool interleaved, int lane) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int u = r * LANES + lane;
        if (u * 2 * VEC >= rotated) continue;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const CosSin<T> a = table[u * VEC + i];
            float &x0 = p.v[r][i], &y0 = p.v[r][VEC + i], &x1 = p.v[r][2 * i], &y1 = p.v[r][2 * i + 1];
            const T x = interleaved ? x1 : x0, y = interleaved ? y1 : y0;
            const float nx = (float)fused(x, a.c, -(y * a.s)), ny = (float)fused(x, a.s, y * a.c);
            if (interleaved) x1 = nx, y1 = ny;
            else x0 = nx, y0 = ny;
        }
    }
}

template <int DT, int VEC, int R>
__device__ __forceinline__ void store_part(const Part<VEC, R> &p, typename type<DT>::t *to, int dim, int rotated, bool interleaved, int lane) {
    each_unit<VEC, R>(dim, rotated, interleaved, lane, [&](int r, int first, int second, bool together) {
        if (together) {
            put<DT, 2 * VEC>(to + first, p.v[r]);
        } else {
            put<DT, VEC>(to + first, p.v[r]);
            put<DT, VEC>(to + second, p.v[r] + VEC);
        }
    });
}

// ---- heads of x ---------------------------------------------------------------------------------------------------
struct Rotate {
    const void *x;
    void *out;
    i64 n, x_token, x_head, out_token, out_head;
    const i64 *positions;
    int heads, dim, tokens, per_block;         // tokens of a workgroup, heads of a workgroup
    Turn turn;
};

template <int DT, int VEC, int R>
__global__ __launch_bounds__(BLOCK) void k_rotate(Rotate A) {
    typedef typename type<DT>::t T;
    __shared__ CosSin<float> table[GROUPS * MOST_PAIRS];
    const int lane = threadIdx.x % LANES, half = A.turn.rotated / 2;
    const i64 first = (i64)blockIdx.x * A.tokens;
    const int tokens = (int)min((i64)A.tokens, A.n - first), head0 = (int)blockIdx.y * A.per_block, heads = min(A.per_block, A.heads - head0);
    const int items = tokens * heads;
    int item = threadIdx.x / LANES;
    Part<VEC, R> p;
    auto load = [&](int i) {
        const T *x = (const T *)A.x + (first + i / heads) * A.x_token + (head0 + i % heads) * A.x_head;
        load_part<DT, VEC, R>(p, x, A.dim, A.turn.rotated, A.turn.interleaved, lane);
    };
    if (item < items) load(item);              // on its way while the angles are made
    for (int i = threadIdx.x; i < tokens * half; i += BLOCK)
        table[i] = turned((u64)A.positions[first + i / half] * A.turn.steps[i % half], (float)A.turn.amplitude);
    __syncthreads();
    while (item < items) {
        const int t = item / heads, h = item % heads;
        turn_part<float, VEC, R>(p, table + t * half, A.turn.rotated, A.turn.interleaved, lane);
        store_part<DT, VEC, R>(p, (T *)A.out + (first + t) * A.out_token + (head0 + h) * A.out_head, A.dim, A.turn.rotated, A.turn.interleaved, lane);
        item += GROUPS;
        if (item < items) load(item);
    }
}

// ---- keys and values into the cache -------------------------------------------------------------------------------
struct Append {
    Cache cache;
    Batch batch;
    const void *x[2];                          // keys, values
    i64 token[2], head[2], n;
    const i64 *positions;
    int tokens;                                // of a workgroup
    Turn turn;
};

__device__ __forceinline__ u32 most_of_lanes(u32 v) {
#pragma unroll
    for (int d = LANES / 2; d; d >>= 1) v = max(v, (u32)__shfl_xor((int)v, d));
    return v;
}

// DT: of the new keys and values, TO: of the cache's
template <int DT, int TO, int VEC, int R>
__global__ __launch_bounds__(BLOCK) void k_append(Append A) {
    typedef typename type<DT>::t T;
    typedef typename std::conditional<TO == VI_I8, double, float>::type Wide;           // which integer it is, is decided near borders
    struct Place {
        i64 page, position;
        int row, fine;
    };
    __shared__ CosSin<Wide> table[GROUPS * MOST_PAIRS];
    __shared__ Place places[GROUPS];
    const int lane = threadIdx.x % LANES, half = A.turn.rotated / 2, heads = (int)A.cache.heads, wave = threadIdx.x / 64;
    const i64 first = (i64)blockIdx.x * A.tokens;
    const int tokens = (int)min((i64)A.tokens, A.n - first), items = tokens * 2 * heads, dim = A.cache.dim;
    int item = threadIdx.x / LANES;
    Part<VEC, R> p;
    auto load = [&](int i) {
        const int t = i / (2 * heads), h = i % (2 * heads), values = h >= heads;
        const T *x = (const T *)A.x[values] + (first + t) * A.token[values] + (values ? h - heads : h) * A.head[values];
        load_part<DT, VEC, R>(p, x, dim, values ? 0 : A.turn.rotated, A.turn.interleaved, lane);
    };
    if (item < items) load(item);
    for (int t = wave; t < tokens; t += BLOCK / 64) {
        const i64 row = first + t;
        const int b = find_sequence(A.batch, row);
        if (threadIdx.x % 64 == 0) {
            Place place = {0, 0, 0, 0};
            if (b >= 0) {
                const i64 j = (i64)A.batch.lengths[b] - A.batch.starts[b + 1] + row;
                place.fine = find_entry(A.cache, A.batch, b, j, &place.page, &place.row);
                place.position = A.positions ? A.positions[row] : j;
            }
            places[t] = place;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < tokens * half; i += BLOCK) table[i] = turned((u64)places[i / half].position * A.turn.steps[i % half], (Wide)A.turn.amplitude);
    __syncthreads();
    while (item < items) {
        const int t = item / (2 * heads), h = item % (2 * heads), values = h >= heads, head = values ? h - heads : h, rotated = values ? 0 : A.turn.rotated;
        const Place place = places[t];
        if (!values) turn_part<Wide, VEC, R>(p, table + t * half, rotated, A.turn.interleaved, lane);
        const Half &to = A.cache.half[values];
        char *at = to.at + place.page * to.page + head * to.head + place.row * to.row;
        if constexpr (TO == VI_I8) {
            u32 top = 0;
            each_unit<VEC, R>(dim, rotated, A.turn.interleaved, lane, [&](int r, int, int, bool) {
#pragma unroll
                for (int i = 0; i < 2 * VEC; ++i) top = max(top, __float_as_uint(p.v[r][i]) & 0x7FFFFFFFu);
            });
            top = most_of_lanes(top);          // sizes as bit patterns: in their order, infinity above, NaN above that
            const float most = __uint_as_float(top);
            const bool bad = top >= 0x7F800000u, none = bad || most < 127.0f * 0x1p-126f;
            const float steps = none ? 0.0f : 127.0f / most;
            if (place.fine) {
                if (lane == 0) to.scales[place.page * to.scale_page + head * to.scale_head + place.row] = bad ? __uint_as_float(0x7FC00000u) : none ? 0.0f : most / 127.0f;
                each_unit<VEC, R>(dim, rotated, A.turn.interleaved, lane, [&](int r, int from, int second, bool) {
                    // rounded by an addition whose result has units of one: its low byte is the integer
                    signed char q[2 * VEC];
#pragma unroll
                    for (int i = 0; i < 2 * VEC; ++i) q[i] = none ? 0 : (signed char)__float_as_uint(p.v[r][i] * steps + 12582912.0f);
                    __builtin_memcpy(at + from, q, VEC);
                    __builtin_memcpy(at + second, q + VEC, VEC);
                });
            }
        } else {
            if (place.fine) store_part<TO, VEC, R>(p, (typename type<TO>::t *)at, dim, rotated, A.turn.interleaved, lane);
        }
        item += GROUPS;
        if (item < items) load(item);
    }
}

int check_turn(const char *who, const u64 *steps, i64 rotated, i64 dim, double amplitude) {
    if (rotated < 0 || rotated > dim || rotated & 1) return vi::fail(VI_EINVAL, "%s: %lld of %lld columns rotated", who, (long long)rotated, (long long)dim);
    if (rotated && !steps) return vi::fail(VI_EINVAL, "%s: null pointer", who);
    if (!(amplitude > 0 && amplitude < 1e6)) return vi::fail(VI_EINVAL, "%s: an amplitude of %g", who, amplitude);
    return VI_OK;
}

// four pairs to a lane where columns and rotated columns come in eights, else single ones
#define WITH_PARTS(GO)                                  \
    do {                                                \
        if (fours && dim <= 8 * LANES) GO(4, 1);        \
        else if (fours) GO(4, 2);                       \
        else GO(1, 8);                                  \
    } while (0)

template <int DT>
void launch_rotate(const Rotate &A, dim3 grid, hipStream_t s) {
    const int dim = A.dim;
    const bool fours = dim % 8 == 0 && A.turn.rotated % 8 == 0;
#define GO(VEC, R) hipLaunchKernelGGL((k_rotate<DT, VEC, R>), grid, dim3(BLOCK), 0, s, A)
    WITH_PARTS(GO);
#undef GO
}

template <int DT, int TO>
void launch_append(const Append &A, dim3 grid, hipStream_t s) {
    const int dim = A.cache.dim;
    const bool fours = A.turn.rotated % 8 == 0;
#define GO(VEC, R) hipLaunchKernelGGL((k_append<DT, TO, VEC, R>), grid, dim3(BLOCK), 0, s, A)
    WITH_PARTS(GO);
#undef GO
}

}  // namespace

extern "C" int vi_rotate_heads(int dtype, const void *x, int64_t n, int64_t heads, int64_t dim, int64_t x_token, int64_t x_head, const int64_t *positions,
                               const uint64_t *steps, int64_t rotated, int interleaved, double amplitude, void *out, int64_t out_token, int64_t out_head,
                               void *stream) {
    const char *who = "vi_rotate_heads";
    if (!is_float(dtype)) return vi::fail(VI_EINVAL, "%s: dtype %d is none of VI_F32, VI_BF16, VI_F16", who, dtype);
    if (n < 0 || n > 0x7FFFFFFF || heads < 0 || heads > 0xFFFF || dim < 2 || dim > 2 * MOST_PAIRS || dim & 1)
        return vi::fail(VI_EINVAL, "%s: %lld tokens of %lld heads of %lld", who, (long long)n, (long long)heads, (long long)dim);
    if (const int rc = check_turn(who, steps, rotated, dim, amplitude)) return rc;
    if ((n > 1 && out_token < dim) || (heads > 1 && out_head < dim) || x_token < 0 || x_head < 0) return vi::fail(VI_EINVAL, "%s: heads that overlap", who);
    if (n == 0 || heads == 0) return VI_OK;
    if (!x || !out || !positions) return vi::fail(VI_EINVAL, "%s: null pointer", who);
    Rotate A = {};
    A.n = n, A.x_token = x_token, A.x_head = x_head, A.out_token = out_token, A.out_head = out_head, A.heads = (int)heads, A.dim = (int)dim;
    A.turn = {steps, (int)rotated, interleaved != 0, amplitude};
    // a workgroup's sixteen groups of lanes each have a head at least; all heads of a token in one where there are tokens enough
    A.per_block = (int)(n >= 1024 || heads < GROUPS ? heads : GROUPS);
    A.tokens = (int)(heads >= GROUPS ? 1 : GROUPS / heads);
    const i64 step = MAX_BLOCKS / ((heads + A.per_block - 1) / A.per_block) * A.tokens;
    for (i64 first = 0; first < n; first += step) {
        A.n = n - first < step ? n - first : step;
        A.x = (const char *)x + first * x_token * size_of(dtype), A.out = (char *)out + first * out_token * size_of(dtype), A.positions = positions + first;
        const dim3 grid((unsigned)((A.n + A.tokens - 1) / A.tokens), (unsigned)((heads + A.per_block - 1) / A.per_block));
        if (dtype == VI_F32) launch_rotate<VI_F32>(A, grid, (hipStream_t)stream);
        if (dtype == VI_BF16) launch_rotate<VI_BF16>(A, grid, (hipStream_t)stream);
        if (dtype == VI_F16) launch_rotate<VI_F16>(A, grid, (hipStream_t)stream);
        VI_LAUNCH_CHECK(who);
    }
    return VI_OK;
}

extern "C" int vi_append_tokens(const vi_cache *cache, const vi_batch *batch, int dtype, const void *k, int64_t k_token, int64_t k_head, const void *v,
                                int64_t v_token, int64_t v_head, int64_t n, const int64_t *positions, const uint64_t *steps, int64_t rotated,
                                int interleaved, double amplitude, void *stream) {
    const char *who = "vi_append_tokens";
    Append A = {};
    if (const int rc = take(who, cache, batch, &A.cache, &A.batch)) return rc;
    if (!is_float(dtype)) return vi::fail(VI_EINVAL, "%s: dtype %d is none of VI_F32, VI_BF16, VI_F16", who, dtype);
    if (n < 0 || n > MAX_BLOCKS) return vi::fail(VI_EINVAL, "%s: %lld tokens", who, (long long)n);
    if (const int rc = check_turn(who, steps, steps ? rotated : 0, cache->dim, amplitude)) return rc;
    if (k_token < 0 || k_head < 0 || v_token < 0 || v_head < 0) return vi::fail(VI_EINVAL, "%s: tokens %lld apart", who, (long long)k_token);
    if (n == 0 || batch->sequences == 0 || cache->pages == 0) return VI_OK;
    if (!k || !v) return vi::fail(VI_EINVAL, "%s: null pointer", who);
    A.x[0] = k, A.x[1] = v, A.token[0] = k_token, A.token[1] = v_token, A.head[0] = k_head, A.head[1] = v_head, A.n = n, A.positions = positions;
    A.turn = {steps, steps ? (int)rotated : 0, interleaved != 0, amplitude};
    // a group of lanes has a head at least; where there are many tokens four to a workgroup, whose threads then have an angle each (4096 tokens into 8 heads
    // of 8 bits: 14 us; 18 with one, 16 with two, 19 with eight)
    A.tokens = (int)(2 * cache->heads >= GROUPS ? (n >= 2048 ? 4 : 1) : GROUPS / (2 * cache->heads));
    const dim3 grid((unsigned)((n + A.tokens - 1) / A.tokens));
    const hipStream_t s = (hipStream_t)stream;
#define FROM(DT)                                                            \
    do {                                                                    \
        if (cache->dtype == VI_BF16) launch_append<DT, VI_BF16>(A, grid, s);\
        if (cache->dtype == VI_F16) launch_append<DT, VI_F16>(A, grid, s);  \
        if (cache->dtype == VI_I8) launch_append<DT, VI_I8>(A, grid, s);    \
    } while (0)
    if (dtype == VI_F32) FROM(VI_F32);
    if (dtype == VI_BF16) FROM(VI_BF16);
    if (dtype == VI_F16) FROM(VI_F16);
#undef FROM
    VI_LAUNCH_CHECK(who);
    return VI_OK;
}
