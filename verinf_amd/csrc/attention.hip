// Attention of new tokens over a paged cache: a token's, a chunk of a prompt's, a tree of drafts'.
//
//     s_j = scale q k_j    o = sum_j e^(s_j - M) v_j / sum_j e^(s_j - M)    over the keys j that the token attends to
//
// One pass with the running largest score and sum.  The heads that share keys are rows of one product: a tile is 32 NB WM rows, row r token r / group,
// head r % group of one head of the cache, and every key of it is read once for all of them.
//
// A wavefront takes 32 keys at a time as S^T = K Q^T, so that a lane holds sixteen scores of one row (key 8 (r / 4) + 4 (lane / 32) + r % 4 in register r):
// largest entry and sum are in the lane, but for one exchange with the lane 32 on.  Those sixteen, rounded to 16 bits, are the second operand
// of O^T += V^T P^T as they are, if the keys of a step are counted in the order in which they lie there; LDS's transposing reads fetch V^T in any order of rows.
//
// Keys and values go straight into LDS (1 KiB a load and wavefront), ST stages of 32 KBS keys, in an order in which the sixteen lanes that are served at a time
// meet all banks: unit u (16 bytes) of a row lies at u ^ order(row).  WM wavefronts share a stage; WK such groups take every WK-th stage and are added at the end.  Where
// there are few tiles the keys are cut between workgroups too, and k_join adds what they leave.
//
// Roundings: P to the type of the queries (as V has), relative to a largest score that may be up to 2^8 behind; all sums in 32 bits.
#include <type_traits>

#include "cache.hpp"

namespace {

using namespace kv;

typedef u32 v4u __attribute__((ext_vector_type(4)));
typedef u32 v2u __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int MAX_NODES = 256;                 // of a tree
constexpr int MASK_WORDS = MAX_NODES / 32 + 1;
constexpr i64 MAX_BLOCKS = 1 << 22;            // of a launch, which has less than 2^32 threads
constexpr float LATE = 8.0f;                   // powers of two that scores may exceed what they are relative to

// DT: of queries and outputs; I8: the cache has 8-bit integers; DP: columns, at least the cache's
template <int DT_, bool I8_, int DP_, int NB_, int WM_, int WK_, int KBS_, int ST_, int OCC_>
struct Form {
    static constexpr int DT = DT_, DP = DP_, NB = NB_, WM = WM_, WK = WK_, KBS = KBS_, ST = ST_, OCC = OCC_;
    static constexpr bool I8 = I8_;
    static constexpr int WAVES = WM * WK, THREADS = 64 * WAVES, ROWS = 32 * NB * WM;
    static constexpr int KEYS = 32 * KBS, GROUPS = 2 * KBS;            // of a stage; sixteen keys are of one page
    static constexpr int ROW = DP * (I8 ? 1 : 2), UNITS = ROW / 16, PER_LOAD = 64 / UNITS, LOADS = 16 / PER_LOAD;        // bytes, units; rows of a load, loads of a group
    static constexpr int HALF = KEYS * ROW, SCALES = I8 ? 2 * KEYS * 4 : 0, STAGE = 2 * HALF + SCALES;
    static constexpr int MINE = 2 * GROUPS * LOADS / WM + (I8 ? KBS : 0);             // loads of a wavefront in a stage
    static constexpr int PITCH = 36;           // floats between rows of 32 on their way out
    static constexpr int OUT = WAVES * NB * 32 * PITCH * 4 + WAVES * NB * 32 * 8 + ROWS * 8;
    static constexpr int LDS = WK * ST * STAGE > OUT ? WK * ST * STAGE : OUT;
    static constexpr int MASKS = ROWS < MAX_NODES ? ROWS : MAX_NODES;
    static_assert(2 * GROUPS * LOADS % WM == 0, "loads of a stage");
};

struct Args {
    Cache cache;
    Batch batch;
    const void *q;
    void *out;
    i64 q_token, q_head, out_token, out_head, n;
    const int *parents;
    int heads, group, tiles, splits, clear;
    float c;                                   // scale log2(e)
    float *part;                               // [tile][head][split][ROWS][DP] sums
    float *most;                               // [tile][head][split][ROWS][2] what they are relative to, sums of the exponentials
};

template <int UNITS>
__device__ __forceinline__ int order(int row) {
    if (UNITS == 4) return row >> 2 & 3;
    if (UNITS == 8) return (row >> 1 & 1) << 2 | (row >> 2 & 3);
    return (row & 3) << 2 | (row >> 2 & 3);    // four rows behind each other are in four quarters of the banks, sixteen at sixteen places
}

// ---- loads into LDS -----------------------------------------------------------------------------------------------
// 64 lanes' 16 bytes at base + off to LDS from `at` on, each lane's at its own place; base and `at` are the wavefront's.  As an instruction of its own
// the compiler does not wait for it before the next read of LDS: the waits are arrive()'s.  Inside an asm block nothing inserts wait states: one between the
// write of M0 and the load, five between a vector instruction's write of a scalar register (readfirstlane) and a load that reads it.
__device__ __forceinline__ void fetch_to_lds(u32 at, u32 off, const char *base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(at), "v"(off), "s"(base) : "memory");
}
// the same of 4 bytes a lane, each at an address of its own
__device__ __forceinline__ void fetch_words_to_lds(u32 at, const float *from) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(at), "v"(from) : "memory");
}
// all but the wavefront's last `N` loads have arrived and its LDS accesses are done
template <int N>
__device__ __forceinline__ void arrive() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(N) : "memory");
}
__device__ __forceinline__ void meet_wave() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ void meet_group() { asm volatile("s_barrier" : : : "memory"); }

// Four rows of sixteen 16-bit numbers, row i from lanes 4 i .. 4 i + 3 of each sixteen (8 bytes a lane); lane i gets column i.
__device__ __forceinline__ v2u read_columns16(const char *from) {
    typedef short v4s __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s *)from));
}
// Eight rows of sixteen bytes, row i from lanes 2 i and 2 i + 1 of each sixteen; lane i gets column i.
__device__ __forceinline__ v2u read_columns8(const char *from) {
    typedef int v2i __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i *)from));
}

// two numbers as the 16-bit type, the first in the lower half
template <int DT>
__device__ __forceinline__ u32 pack(float a, float b) {
    typedef float v2f __attribute__((ext_vector_type(2)));
    typedef typename type<DT>::t v2t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(u32, __builtin_convertvector((v2f{a, b}), v2t));
}
// eight 8-bit integers as bfloat16: exact
__device__ __forceinline__ v4u widen(v2u w) {
    v4u r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const u32 s = w[i / 2] >> (16 * (i & 1));
        r[i] = pack<VI_BF16>((float)(signed char)s, (float)(signed char)(s >> 8));
    }
    return r;
}

template <int DT>
__device__ __forceinline__ v16f multiply(v4u a, v4u b, v16f c) {
    typedef typename type<DT>::t v8t __attribute__((ext_vector_type(8)));
    if constexpr (DT == VI_BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8t, a), __builtin_bit_cast(v8t, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8t, a), __builtin_bit_cast(v8t, b), c, 0, 0, 0);
}

// the larger of the lane's number and that of the lane 32 on
__device__ __forceinline__ float most_of_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ int same(int v) { return (int)__builtin_amdgcn_readfirstlane((u32)v); }

// ---- which rows ---------------------------------------------------------------------------------------------------
// Sequence b's tiles begin at starts[b] group / rows + b: apart by at least as many as it needs, and no sequence's start has to be known to count them.
struct Tile {
    int b, n, first;                           // sequence, its new tokens, the tile's first row in it
    i64 s0;
};
template <int ROWS>
__device__ __forceinline__ bool find_tile(const Args &A, int tile, Tile *t) {
    auto start = [&](int b) { return max((i64)0, min((i64)A.batch.starts[b], A.n)); };
    int count = 0;
    for (int first = 0; first < A.batch.sequences; first += 64) {
        const int b = min(first + (int)(threadIdx.x & 63), A.batch.sequences);
        count += __popcll(__ballot(b < A.batch.sequences && start(b) * A.group / ROWS + b <= tile));
    }
    const int b = count - 1;
    if (b < 0) return false;
    const int s0 = same((int)start(b)), s1 = same((int)start(b + 1));
    const i64 first = ((i64)tile - b - (i64)s0 * A.group / ROWS) * ROWS;
    t->b = b, t->n = s1 - s0, t->s0 = s0, t->first = (int)first;
    return first >= 0 && first < (i64)t->n * A.group;         // less than 0 where starts does not rise
}

// ---- the pass over the keys ---------------------------------------------------------------------------------------
template <class F>
__global__ __launch_bounds__(F::THREADS, F::OCC) void k_attend(Args A) {
    constexpr int DT = F::DT, DP = F::DP, NB = F::NB, WM = F::WM, WK = F::WK, ROW = F::ROW, UNITS = F::UNITS;
    typedef typename type<DT>::t T;
    __shared__ alignas(16) char lds[F::LDS];
    __shared__ u32 masks[F::MASKS * MASK_WORDS];
    __shared__ int above[MAX_NODES];
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = same((int)threadIdx.x >> 6), wm = wave % WM, part = wave / WM;
    const int heads = (int)A.cache.heads, head = (int)blockIdx.x % heads, split = (int)blockIdx.x / heads % A.splits;
    const int tile = A.tiles - 1 - (int)blockIdx.x / heads / A.splits;         // the longest first, where a prompt's tiles differ

    if (A.clear) {                             // rows of no sequence
        const i64 s0 = A.batch.sequences ? max((i64)0, min((i64)A.batch.starts[0], A.n)) : A.n, s1 = A.batch.sequences ? max(s0, min((i64)A.batch.starts[A.batch.sequences], A.n)) : A.n;
        for (i64 r = blockIdx.x; r < s0 + A.n - s1; r += gridDim.x)
            for (int i = threadIdx.x; i < A.heads * A.cache.dim; i += F::THREADS)
                ((T *)A.out)[(r < s0 ? r : s1 + r - s0) * A.out_token + i / A.cache.dim * A.out_head + i % A.cache.dim] = (T)0.0f;
    }
    Tile t;
    if (!find_tile<F::ROWS>(A, tile, &t)) return;
    const int length = same((int)max((i64)0, min((i64)A.batch.lengths[t.b], A.batch.most))), context = same(A.batch.lengths[t.b]) - t.n;
    const bool tree = A.parents && t.n <= MAX_NODES;
    // key j < limit: the tokens of the tile's, and the wavefront's, first and last row; keys below `free` are masked for none of the wavefront's
    auto token = [&](int row) { return (int)((u32)row / (u32)A.group); };
    const int last = min(t.n - 1, token(t.first + F::ROWS - 1)), end = max(0, min(length, context + last + 1));
    const int row0 = t.first + wm * NB * 32, wave_first = token(row0), wave_last = min(t.n - 1, token(row0 + 32 * NB - 1));
    const int wave_end = wave_first < t.n ? min(end, context + wave_last + 1) : 0, wave_free = tree ? context : context + wave_first + 1;
    const int units = (end + F::KEYS * WK - 1) / (F::KEYS * WK);
    const int from = (int)((i64)split * units / A.splits), to = (int)((i64)(split + 1) * units / A.splits);
    const i64 slot = ((i64)tile * heads + head) * A.splits + split;
    if (A.splits > 1 && from == to) {
        for (int r = threadIdx.x; r < F::ROWS; r += F::THREADS) A.most[(slot * F::ROWS + r) * 2] = -INFINITY, A.most[(slot * F::ROWS + r) * 2 + 1] = 0.0f;
        return;
    }

    // the rows' ancestors among the new tokens, a bit each
    if (tree) {
        for (int i = threadIdx.x; i < t.n; i += F::THREADS) above[i] = A.parents[t.s0 + i];
        __syncthreads();
        for (int i = token(t.first) + (int)threadIdx.x; i <= last; i += F::THREADS) {
            u32 *bits = masks + (i - token(t.first)) * MASK_WORDS;
#pragma unroll
            for (int w = 0; w < MASK_WORDS; ++w) bits[w] = 0;
            for (int at = i;;) {
                bits[at >> 5] |= 1u << (at & 31);
                const int up = above[at];
                if (up < 0 || up >= at) break;
                at = up;
            }
        }
        __syncthreads();
    }

    // queries: unit (of eight columns) `chunk` of a row for half and step
    v4u q[NB][DP / 16];
    int limit[NB];                             // of the lane's row: keys below it (a chain's), its mask's place (a tree's); -1: no row
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const int row = row0 + 32 * nb + (lane & 31), tok = token(row), g = row - tok * A.group;
        const bool fine = tok < t.n;
        limit[nb] = !fine ? -1 : tree ? (tok - token(t.first)) * MASK_WORDS : max(0, context + tok + 1);
        const T *x = (const T *)A.q + (t.s0 + (fine ? tok : 0)) * A.q_token + (head * A.group + (fine ? g : 0)) * A.q_head;
#pragma unroll
        for (int st = 0; st < DP / 16; ++st) {
            const int chunk = F::I8 ? 4 * (st / 2) + 2 * half + st % 2 : 2 * st + half;
            q[nb][st] = v4u{0, 0, 0, 0};
            if (fine && chunk * 8 < A.cache.dim) q[nb][st] = load_any<v4u>(x + chunk * 8);
        }
    }

    // ---- stages
    const u32 lds_at = (u32)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    const char *keys = A.cache.half[0].at + head * A.cache.half[0].head, *values = A.cache.half[1].at + head * A.cache.half[1].head;
    const float *key_scales = A.cache.half[0].scales + head * A.cache.half[0].scale_head, *value_scales = A.cache.half[1].scales + head * A.cache.half[1].scale_head;
    const int full_units = A.cache.dim * (F::I8 ? 1 : 2) / 16;
    typedef const __attribute__((address_space(4))) int *Table;        // constant while the kernel runs: read by the scalar cache
    const Table pages = (Table)(A.batch.pages + t.b * A.batch.stride);
    const int stages = to - from;              // of each of the WK groups
    auto stage_key = [&](int it) { return ((from + it) * WK + part) * F::KEYS; };
    struct Page {
        i64 page;
        int row, valid;                        // row in the page of the first of sixteen keys; how many of them there are
    };
    auto page_of = [&](int j) {
        Page p = {0, 0, 0};
        if (j < end) {
            const int n = pages[j >> A.cache.shift];
            p.page = n, p.row = j & A.cache.mask;
            p.valid = n >= 0 && n < A.cache.pages ? min(16, end - j) : 0;
        }
        return p;
    };
    u32 partial = 0;                           // a bit for each slot whose stage has fewer loads than MINE
    auto fetch = [&](int it) {
        const int j = stage_key(it), into = it % F::ST;
        char *stage = lds + (part * F::ST + into) * F::STAGE;
        const u32 at = lds_at + (u32)((part * F::ST + into) * F::STAGE);
        bool some = false;
        Page page[F::GROUPS];
#pragma unroll
        for (int g = 0; g < F::GROUPS; ++g) page[g] = page_of(j + 16 * g), some |= page[g].valid < 16;
#pragma unroll
        for (int l = 0; l < 2 * F::GROUPS * F::LOADS / WM; ++l) {
            const int n = l * WM + wm, which = n / (F::GROUPS * F::LOADS), g = n / F::LOADS % F::GROUPS, i = n % F::LOADS;
            i64 number = page[0].page;
            int first = page[0].row, valid = page[0].valid;
#pragma unroll
            for (int o = 1; o < F::GROUPS; ++o)
                if (g == o) number = page[o].page, first = page[o].row, valid = page[o].valid;
            const i64 page_apart = which ? A.cache.half[1].page : A.cache.half[0].page, row_apart = which ? A.cache.half[1].row : A.cache.half[0].row;
            const char *base = (which ? values : keys) + number * page_apart + first * row_apart;
            const int row = i * F::PER_LOAD + lane / UNITS, unit = lane % UNITS ^ order<UNITS>(row);
            const u32 off = (u32)row * (u32)row_apart + (u32)unit * 16;
            const u32 place = (u32)(which * F::HALF + g * 16 * ROW + i * 1024);
            if (valid == 16 && full_units == UNITS) {
                fetch_to_lds(at + place, off, base);
            } else {
                if (row < valid && unit < full_units) fetch_to_lds(at + place, off, base);
                else *(v4u *)(stage + place + lane * 16) = v4u{0, 0, 0, 0};
            }
        }
        if constexpr (F::I8) {
            // lanes 0 .. 31 the scales of 32 keys, the others of as many values
#pragma unroll
            for (int kb = 0; kb < F::KBS; ++kb) {
                const bool second = lane & 16;
                const i64 number = second ? page[2 * kb + 1].page : page[2 * kb].page;
                const int first = second ? page[2 * kb + 1].row : page[2 * kb].row, valid = second ? page[2 * kb + 1].valid : page[2 * kb].valid;
                const float *base = half ? value_scales : key_scales;
                const i64 apart = half ? A.cache.half[1].scale_page : A.cache.half[0].scale_page;
                const u32 place = 2 * F::HALF + kb * 256;
                if ((lane & 15) < valid) fetch_words_to_lds(at + place, base + number * apart + first + (lane & 15));
                else *(float *)(stage + place + lane * 4) = 0.0f;
            }
        }
        partial = (partial & ~(1u << into)) | (u32)some << into;
    };

    v16f o[NB][DP / 32];
    float most[NB], relative[NB], sum[NB];     // largest score so far (or up to LATE behind), times c: what the sums are relative to
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        most[nb] = -INFINITY, relative[nb] = -INFINITY, sum[nb] = 0;
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) o[nb][db] = v16f{};
    }

    // 32 keys from j on, in the stage's block kb; the low and the high sixteen have so many
    auto block = [&](const char *stage, int kb, int j, int low, int high, auto masked) {
        constexpr bool MASKED = decltype(masked)::value;
        u32 window[NB];
        if constexpr (MASKED) {
            const u32 there = (low >= 16 ? 0xFFFFu : (1u << low) - 1) | (high >= 16 ? 0xFFFFu : (1u << high) - 1) << 16;
            bool any = false;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                u32 w = ~0u;
                if (limit[nb] >= 0) {
                    if (!tree) {
                        const int left = limit[nb] - j;
                        w = left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1;
                    } else {
                        const int node = j - context;
                        const u32 *bits = masks + limit[nb];
                        if (node <= -32) w = ~0u;
                        else if (node < 0) w = bits[0] << -node | ((1u << -node) - 1);
                        else if (node < MAX_NODES) w = (u32)(((u64)bits[(node >> 5) + 1] << 32 | bits[node >> 5]) >> (node & 31));
                        else w = 0;
                    }
                }
                window[nb] = w & there;
                any |= window[nb] != 0;
            }
            if (!__any(any)) return;
        }
        const char *k = stage + kb * 32 * ROW, *v = stage + F::HALF + kb * 32 * ROW;
        v16f s[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) s[nb] = v16f{};
        {
            const int row = lane & 31;
            const char *mine = k + row * ROW;
            const int o_ = order<UNITS>(row & 15);
            if constexpr (F::I8) {
#pragma unroll
                for (int st = 0; st < DP / 16; st += 2) {
                    const v4u w = *(const v4u *)(mine + ((st + half) ^ o_) * 16);
                    const v4u lo = widen(v2u{w.x, w.y}), hi = widen(v2u{w.z, w.w});
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) s[nb] = multiply<DT>(lo, q[nb][st], s[nb]);
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) s[nb] = multiply<DT>(hi, q[nb][st + 1], s[nb]);
                }
                v4f scale[4];
#pragma unroll
                for (int g = 0; g < 4; ++g) scale[g] = *(const v4f *)(stage + 2 * F::HALF + kb * 256 + (8 * g + 4 * half) * 4);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[nb][r] *= scale[r / 4][r % 4];
            } else {
#pragma unroll
                for (int st = 0; st < DP / 16; ++st) {
                    const v4u w = *(const v4u *)(mine + ((2 * st + half) ^ o_) * 16);
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) s[nb] = multiply<DT>(w, q[nb][st], s[nb]);
                }
            }
        }
        v4u p[NB][2];
        v4f value_scale[4];
        if constexpr (F::I8) {
#pragma unroll
            for (int g = 0; g < 4; ++g) value_scale[g] = *(const v4f *)(stage + 2 * F::HALF + kb * 256 + 128 + (8 * g + 4 * half) * 4);
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            if constexpr (MASKED) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (!(window[nb] >> (8 * (r / 4) + 4 * half + r % 4) & 1)) s[nb][r] = -INFINITY;
            }
            float top = s[nb][0];
#pragma unroll
            for (int r = 1; r < 16; ++r) top = fmaxf(top, s[nb][r]);
            top = most_of_halves(top);
            if (__any(top * A.c > relative[nb] + LATE)) {
                const float now = fmaxf(most[nb], top), then = now * A.c;
                const float by = relative[nb] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(relative[nb] - then);
                most[nb] = now, relative[nb] = then, sum[nb] *= by;
#pragma unroll
                for (int db = 0; db < DP / 32; ++db) o[nb][db] *= by;
            }
            const float base = relative[nb] == -INFINITY ? 0.0f : relative[nb];
            float e[16], add = 0;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                e[r] = __builtin_amdgcn_exp2f(fmaf(s[nb][r], A.c, -base));
                add += e[r];
            }
            sum[nb] += add;
            if constexpr (F::I8) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    e[r] *= value_scale[r / 4][r % 4];
                    if (MASKED && !(window[nb] >> (8 * (r / 4) + 4 * half + r % 4) & 1)) e[r] = 0;     // its scale may be a NaN
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) p[nb][i / 4][i % 4] = pack<DT>(e[2 * i], e[2 * i + 1]);
        }
        // V^T, keys in the order of the registers: four from 4 half on, four from 8 + 4 half on
        const int in = lane & 15, right = lane >> 4 & 1;
        auto columns = [&](int db, int st) {
            v2u two[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int row = 8 * i + 4 * half + (in >> 2), unit = (4 * db + 2 * right + (in >> 1 & 1)) ^ order<UNITS>(row);
                two[i] = read_columns16(v + (16 * st + row) * ROW + unit * 16 + (in & 1) * 8);
            }
            return v4u{two[0].x, two[0].y, two[1].x, two[1].y};
        };
        // 0 times an infinity or a NaN in a masked place would be a NaN: where there are any they are left out of the products, and what they
        // make of the sums is put in behind, by which kinds of them a row attends to
        constexpr u32 INF = DT == VI_BF16 ? 0x7F80u : 0x7C00u, ONE = DT == VI_BF16 ? 0x3F80u : 0x3C00u;
        auto is_wild = [&](u32 b) { return (b & INF) == INF; };
        bool wild = false;
        if constexpr (MASKED && !F::I8) {
#pragma unroll 1
            for (int u = half; u < UNITS; u += 2) {
                const v4u w = *(const v4u *)(v + (lane & 31) * ROW + u * 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) wild |= is_wild(w[i]) || is_wild(w[i] >> 16);
            }
            wild = __any(wild);
        }
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                v4u w;
                if constexpr (F::I8) {
                    const int row = (in >> 3) * 8 + 4 * half + (in >> 1 & 3), unit = (2 * db + right) ^ order<UNITS>(row);
                    w = widen(read_columns8(v + (16 * st + row) * ROW + unit * 16 + (in & 1) * 8));
                } else {
                    w = columns(db, st);
                    if (MASKED && wild)
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[i] &= (is_wild(w[i] & 0xFFFFu) ? 0 : 0xFFFFu) | (is_wild(w[i] >> 16) ? 0 : 0xFFFF0000u);
                }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) o[nb][db] = multiply<DT>(w, p[nb][st], o[nb][db]);
            }
        if constexpr (MASKED && !F::I8) {
            if (!wild) return;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                v4u counts[2];                 // ones at the keys that the row attends to
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const u32 bits = window[nb] >> (8 * (2 * i / 4) + 4 * half + 2 * i % 4);
                    counts[i / 4][i % 4] = (bits & 1 ? ONE : 0) | (bits & 2 ? ONE : 0) << 16;
                }
#pragma unroll
                for (int db = 0; db < DP / 32; ++db) {
                    const v4u w[2] = {columns(db, 0), columns(db, 1)};
                    v16f more = {};
#pragma unroll
                    for (int kind = 0; kind < 3; ++kind) {             // +inf, -inf, NaN: inf - inf is a NaN too
                        v16f n = {};
#pragma unroll
                        for (int st = 0; st < 2; ++st) {
                            auto one = [&](u32 b) { return (kind == 0 ? b == INF : kind == 1 ? b == (INF | 0x8000u) : (b & 0x7FFFu) > INF) ? ONE : 0; };
                            v4u ones;
#pragma unroll
                            for (int i = 0; i < 4; ++i) ones[i] = one(w[st][i] & 0xFFFFu) | one(w[st][i] >> 16) << 16;
                            n = multiply<DT>(ones, counts[st], n);
                        }
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (n[r] > 0) more[r] += kind == 0 ? INFINITY : kind == 1 ? -INFINITY : __uint_as_float(0x7FC00000u);
                    }
                    o[nb][db] += more;
                }
            }
        }
    };

#pragma unroll 1
    for (int it = 0; it < min(F::ST - 1, stages); ++it) fetch(it);
#pragma unroll 1
    for (int it = 0; it < stages; ++it) {
        // this stage's loads have arrived; those of the ones behind it may be on their way, where each has all its loads
        const u32 behind = partial & ~(1u << it % F::ST) & ~(1u << (it + F::ST - 1) % F::ST);
        if (F::ST == 2 || behind || it + F::ST - 2 >= stages) arrive<0>();
        else arrive<(F::ST - 2) * F::MINE>();
        if (WM > 1) meet_group();
        else meet_wave();
        if (it + F::ST - 1 < stages) fetch(it + F::ST - 1);
        const char *stage = lds + (part * F::ST + it % F::ST) * F::STAGE;
#pragma unroll 1
        for (int kb = 0; kb < F::KBS; ++kb) {
            const int j = stage_key(it) + 32 * kb;
            if (j >= wave_end) break;
            const int low = page_of(j).valid, high = page_of(j + 16).valid;
            if (low == 16 && high == 16 && j + 32 <= wave_free) block(stage, kb, j, low, high, std::false_type());
            else block(stage, kb, j, low, high, std::true_type());
        }
    }

    // ---- the WK groups' sums as one, and out
    arrive<0>();
    __syncthreads();
    float *buf = (float *)lds, *of_waves = buf + F::WAVES * NB * 32 * F::PITCH, *of_rows = of_waves + F::WAVES * NB * 32 * 2;
    float factor[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum[nb]), __float_as_uint(sum[nb]), false, false);
        sum[nb] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
        if (half == 0) {
            of_waves[((wave * NB + nb) * 32 + lane) * 2] = relative[nb];
            of_waves[((wave * NB + nb) * 32 + lane) * 2 + 1] = sum[nb];
        }
    }
    __syncthreads();
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        float top = -INFINITY, total = 0;
#pragma unroll
        for (int w = 0; w < WK; ++w) top = fmaxf(top, of_waves[(((w * WM + wm) * NB + nb) * 32 + (lane & 31)) * 2]);
        const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int w = 0; w < WK; ++w) {
            const float *x = of_waves + (((w * WM + wm) * NB + nb) * 32 + (lane & 31)) * 2;
            total += __builtin_amdgcn_exp2f(x[0] - base) * x[1];
        }
        factor[nb] = __builtin_amdgcn_exp2f(relative[nb] - base);
        if (part == 0 && half == 0) {
            of_rows[((wm * NB + nb) * 32 + lane) * 2] = top;
            of_rows[((wm * NB + nb) * 32 + lane) * 2 + 1] = total;
        }
    }
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) {
        if (db) __syncthreads();
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const v4f x = {o[nb][db][4 * g] * factor[nb], o[nb][db][4 * g + 1] * factor[nb], o[nb][db][4 * g + 2] * factor[nb], o[nb][db][4 * g + 3] * factor[nb]};
                *(v4f *)(buf + ((wave * NB + nb) * 32 + (lane & 31)) * F::PITCH + 8 * g + 4 * half) = x;
            }
        __syncthreads();
        for (int i = threadIdx.x; i < F::ROWS * 8; i += F::THREADS) {
            const int r = i / 8, col = 32 * db + i % 8 * 4, row = t.first + r, tok = token(row), g = row - tok * A.group;
            if (tok >= t.n || col >= A.cache.dim) continue;
            v4f x = *(const v4f *)(buf + r * F::PITCH + i % 8 * 4);
#pragma unroll
            for (int w = 1; w < WK; ++w) x += *(const v4f *)(buf + (w * F::ROWS + r) * F::PITCH + i % 8 * 4);
            if (A.splits > 1) {
                *(v4f *)(A.part + (slot * F::ROWS + r) * DP + col) = x;
            } else {
                const float total = of_rows[r * 2 + 1], per = total == 0.0f ? 0.0f : 1.0f / total;
                const v2u two = {pack<DT>(x.x * per, x.y * per), pack<DT>(x.z * per, x.w * per)};
                store_any((T *)A.out + (t.s0 + tok) * A.out_token + (head * A.group + g) * A.out_head + col, two);
            }
        }
    }
    if (A.splits > 1)
        for (int r = threadIdx.x; r < F::ROWS; r += F::THREADS) {
            A.most[(slot * F::ROWS + r) * 2] = of_rows[r * 2];
            A.most[(slot * F::ROWS + r) * 2 + 1] = of_rows[r * 2 + 1];
        }
}

// What the workgroups of a tile have left, as one.
constexpr int JOIN = 256;
template <int DT, int DP, int ROWS>
__global__ __launch_bounds__(JOIN) void k_join(Args A) {
    typedef typename type<DT>::t T;
    const int heads = (int)A.cache.heads, head = (int)blockIdx.x % heads, tile = (int)blockIdx.x / heads;
    Tile t;
    if (!find_tile<ROWS>(A, tile, &t)) return;
    const i64 slot = ((i64)tile * heads + head) * A.splits;
    for (int i = (int)blockIdx.y * JOIN + (int)threadIdx.x; i < ROWS * (DP / 4); i += (int)gridDim.y * JOIN) {
        const int r = i / (DP / 4), col = i % (DP / 4) * 4, row = t.first + r, tok = (int)((u32)row / (u32)A.group), g = row - tok * A.group;
        if (tok >= t.n || col >= A.cache.dim) continue;
        const float *most = A.most + (slot * ROWS + r) * 2, *part = A.part + (slot * ROWS + r) * DP + col;
        float top = -INFINITY, total = 0;
        for (int s = 0; s < A.splits; ++s) top = fmaxf(top, most[(i64)s * ROWS * 2]);
        const float base = top == -INFINITY ? 0.0f : top;
        v4f x = {0, 0, 0, 0};
#pragma unroll 4
        for (int s = 0; s < A.splits; ++s) {
            const float its = most[(i64)s * ROWS * 2], of = most[(i64)s * ROWS * 2 + 1], by = __builtin_amdgcn_exp2f(its - base);
            if (its == -INFINITY && of == 0.0f) continue;              // no keys: nothing was written
            total += by * of;
            x += by * *(const v4f *)(part + (i64)s * ROWS * DP);
        }
        const float per = total == 0.0f ? 0.0f : 1.0f / total;
        const v2u two = {pack<DT>(x.x * per, x.y * per), pack<DT>(x.z * per, x.w * per)};
        store_any((T *)A.out + (t.s0 + tok) * A.out_token + (head * A.group + g) * A.out_head + col, two);
    }
}

// ---- forms --------------------------------------------------------------------------------------------------------
// Up to 32 rows of a sequence: four wavefronts (two where columns are many) with keys of their own; up to 64: the same, two products of each operand of
// keys or values; more: four wavefronts' rows share the keys.
constexpr int key_groups(bool i8, int dp) { return dp > 128 && !i8 ? 2 : 4; }
constexpr int stages_of(bool i8, int dp) { return dp <= 128 && (i8 || dp == 64) ? 4 : 2; }
template <int DT, bool I8, int DP>
struct Few : Form<DT, I8, DP, 1, 1, key_groups(I8, DP), 1, stages_of(I8, DP), 1> {};
template <int DT, bool I8, int DP>
struct Some : Form<DT, I8, DP, 2, 1, key_groups(I8, DP), 1, stages_of(I8, DP), 1> {};
template <int DT, bool I8, int DP>
struct Many : Form<DT, I8, DP, 1, 4, 1, (DP > 128 ? 1 : 2), 2, (DP > 128 ? 1 : 2)> {};

enum { FEW, SOME, MANY };
struct Plan {
    int form, rows, dp, tiles, splits;
    size_t ws_bytes;
};
constexpr int CUS = 256;                       // of a whole card; on a part of one the choice of splits costs time, nothing else

Plan make_plan(int cache_dtype, i64 dim, i64 cache_heads, i64 n, i64 heads, i64 sequences, i64 longest) {
    Plan L = {};
    const i64 group = heads / cache_heads, rows = (n * group + sequences - 1) / sequences;           // of a sequence, on an average
    L.dp = dim <= 64 ? 64 : dim <= 128 ? 128 : 256;
    L.form = rows <= 32 ? FEW : rows <= 64 && L.dp <= 128 ? SOME : MANY;
    L.rows = L.form == FEW ? 32 : L.form == SOME ? 64 : 128;
    const i64 tiles = n * group / L.rows + sequences, busy = (n * group + L.rows - 1) / L.rows > sequences ? (n * group + L.rows - 1) / L.rows : sequences;
    L.tiles = (int)(tiles < MAX_BLOCKS ? tiles : MAX_BLOCKS);
    // as many parts of the keys as make two workgroups a CU, of 512 keys at least
    i64 splits = 2 * CUS / (busy * cache_heads), most = longest / 512;
    splits = splits < most ? splits : most;
    splits = splits < 64 ? splits : 64;
    L.splits = (int)(splits > 1 ? splits : 1);
    if (L.splits > 1) L.ws_bytes = (size_t)(tiles * cache_heads * L.splits * L.rows) * (L.dp + 2) * 4 + vi::WS_SLACK;
    (void)cache_dtype;
    return L;
}

template <class F>
void launch(const Args &A, hipStream_t s) {
    const i64 heads = A.cache.heads;
    hipLaunchKernelGGL(k_attend<F>, dim3((unsigned)(heads * A.tiles * A.splits)), dim3(F::THREADS), 0, s, A);
    if (A.splits > 1) {
        const int blocks = F::ROWS * (F::DP / 4) / JOIN;
        hipLaunchKernelGGL((k_join<F::DT, F::DP, F::ROWS>), dim3((unsigned)(heads * A.tiles), (unsigned)(heads * A.tiles < 2 * CUS ? blocks : 1)), dim3(JOIN), 0, s, A);
    }
}
template <int DT, bool I8, int DP>
void launch_form(int form, const Args &A, hipStream_t s) {
    if (form == FEW) return launch<Few<DT, I8, DP>>(A, s);
    if constexpr (DP <= 128)
        if (form == SOME) return launch<Some<DT, I8, DP>>(A, s);
    launch<Many<DT, I8, DP>>(A, s);
}
template <int DT, bool I8>
void launch_columns(const Plan &L, const Args &A, hipStream_t s) {
    if (L.dp == 64) launch_form<DT, I8, 64>(L.form, A, s);
    if (L.dp == 128) launch_form<DT, I8, 128>(L.form, A, s);
    if (L.dp == 256) launch_form<DT, I8, 256>(L.form, A, s);
}

bool sizes_fine(int dtype, i64 dim, i64 cache_heads, i64 n, i64 heads, i64 sequences, i64 longest) {
    return (dtype == VI_BF16 || dtype == VI_F16 || dtype == VI_I8) && dim >= 16 && dim <= 256 && cache_heads >= 1 && cache_heads <= 0xFFFF && n > 0 && heads >= cache_heads &&
           heads % cache_heads == 0 && heads <= 0xFFFF && n <= 0x7FFFFFFF / heads && sequences > 0 && sequences <= 0xFFFFFF && longest >= 0;
}

}  // namespace

extern "C" size_t vi_attend_cache_workspace_bytes(int cache_dtype, int64_t dim, int64_t cache_heads, int64_t n, int64_t heads, int64_t sequences, int64_t longest) {
    return sizes_fine(cache_dtype, dim, cache_heads, n, heads, sequences, longest) ? make_plan(cache_dtype, dim, cache_heads, n, heads, sequences, longest).ws_bytes : 0;
}

extern "C" int vi_attend_cache(const vi_cache *cache, const vi_batch *batch, int dtype, const void *q, int64_t n, int64_t heads, int64_t q_token, int64_t q_head,
                               const int32_t *parents, float scale, int64_t longest, int clear, void *out, int64_t out_token, int64_t out_head, void *ws,
                               size_t ws_bytes, void *stream) {
    const char *who = "vi_attend_cache";
    Args A = {};
    if (const int rc = take(who, cache, batch, &A.cache, &A.batch)) return rc;
    if (dtype != (cache->dtype == VI_F16 ? VI_F16 : VI_BF16)) return vi::fail(VI_EINVAL, "%s: queries of dtype %d over a cache of dtype %lld", who, dtype, (long long)cache->dtype);
    if (n < 0 || heads < 1 || heads > 0xFFFF || heads % cache->heads || n > 0x7FFFFFFF / heads)
        return vi::fail(VI_EINVAL, "%s: %lld tokens of %lld heads over a cache of %lld", who, (long long)n, (long long)heads, (long long)cache->heads);
    if (!(scale > 0 && scale < 1e30f)) return vi::fail(VI_EINVAL, "%s: a scale of %g", who, (double)scale);
    if (longest < 0) return vi::fail(VI_EINVAL, "%s: no sequence longer than %lld", who, (long long)longest);
    if (q_token < 0 || q_head < 0) return vi::fail(VI_EINVAL, "%s: tokens %lld apart", who, (long long)q_token);
    if ((n > 1 && out_token < cache->dim) || (heads > 1 && out_head < cache->dim)) return vi::fail(VI_EINVAL, "%s: heads that overlap", who);
    if (n == 0 || (batch->sequences == 0 && !clear)) return VI_OK;
    if (!q || !out) return vi::fail(VI_EINVAL, "%s: null pointer", who);
    const i64 sequences = batch->sequences > 0 ? batch->sequences : 1;
    const Plan L = make_plan((int)cache->dtype, cache->dim, cache->heads, n, heads, sequences, longest < A.batch.most ? longest : A.batch.most);
    if (cache->heads * (i64)L.tiles * L.splits > MAX_BLOCKS) return vi::fail(VI_EINVAL, "%s: %lld tokens of %lld sequences", who, (long long)n, (long long)sequences);
    if (ws_bytes < L.ws_bytes || (L.ws_bytes && !ws)) return vi::fail(VI_ENOMEM, "%s: workspace %zu < %zu bytes", who, ws_bytes, L.ws_bytes);
    A.q = q, A.out = out, A.q_token = q_token, A.q_head = q_head, A.out_token = out_token, A.out_head = out_head, A.n = n, A.parents = parents;
    A.heads = (int)heads, A.group = (int)(heads / cache->heads), A.tiles = L.tiles, A.splits = L.splits, A.clear = clear != 0, A.c = scale * 1.44269504f;
    if (L.splits > 1) {
        A.part = (float *)vi::align16(ws);
        A.most = A.part + (i64)L.tiles * cache->heads * L.splits * L.rows * L.dp;
    }
    const hipStream_t s = (hipStream_t)stream;
    if (cache->dtype == VI_I8) launch_columns<VI_BF16, true>(L, A, s);
    if (cache->dtype == VI_BF16) launch_columns<VI_BF16, false>(L, A, s);
    if (cache->dtype == VI_F16) launch_columns<VI_F16, false>(L, A, s);
    VI_LAUNCH_CHECK(who);
    return VI_OK;
}
