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
// Roundings: P to the type of the queries (as V has), to fp16 for 8-bit integers, relative to a largest score that may be up to 2^8 behind, fp16 with 2^7 of what it has room for
// above that; their sum is of them as rounded, but over 8-bit integers, where it is of the exponentials; all sums in 32 bits.  The matrix instructions take 16 bits, and P as a sum of
// two such numbers would be half as many products again; with one, a bf16 result is up to 1.4 times as far from 64 bits as its own rounding takes it.
//
// What bounds it (bf16, 8 heads of 128 columns for 32, where nothing else is said): 64 sequences of 4096 entries and a token each 202 us, 5.3 TB/s, as a large copy
// (118 to 124 us over 8-bit integers, 4.5 to 4.7); 4096 tokens of a prompt, 32 heads of the cache, fp16, 193 to 202 us, 680 to 712 TFLOP/s, where the matrix units are busy for a third of the time and
// the exponentials and their like, some 120 instructions to each 16 products, for half of it (180 us, 765 TFLOP/s, with four heads to one of the cache; 238 over 8-bit
// integers); a token over 1000 entries 12.5 us, over 128, of which a wavefront has one stage, 8.8 in one launch: loads behind each other, of sequence, page and keys.
//
// Columns that are none of 64, 128 or 256 leave units empty, which are zeros in LDS, written anew with each stage, whose loads are waited for at once: 64 tokens over 4096 entries of 80, 96 and
// 112 columns 143, 161 and 185 us, 4.7 to 5.1 TB/s, of 8-bit integers 124 to 138, 2.9 to 3.5; 4096 tokens of a prompt 231 to 233 us, of 128 columns 178 to 180.
#include <type_traits>

#include "cache.hpp"

namespace {

using namespace kv;

typedef u32 v4u __attribute__((ext_vector_type(4)));
typedef u32 v2u __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));

#define INLINE __attribute__((always_inline))

constexpr int MAX_NODES = 256;                 // of a tree
constexpr int MASK_WORDS = MAX_NODES / 32 + 1;
constexpr i64 MAX_BLOCKS = 1 << 22;            // of a launch, which has less than 2^32 threads
constexpr i64 MAX_HEADS = 1 << 30;             // of all tokens together
constexpr i64 MAX_PARTS = 128;                 // of a sequence's keys
constexpr int CLEARING = 64;                   // workgroups that look for rows of no sequence
constexpr float MAX_GAIN = 0x1p126f;
constexpr float LATE = 8.0f;                   // powers of two that scores may exceed what they are relative to

// DT: of queries and outputs; I8: the cache has 8-bit integers, whose products are taken in fp16; DP: columns, at least the cache's; OCC: workgroups of a CU
template <int DT_, bool I8_, int DP_, int WM_, int WK_, int OCC_>
struct Form {
    static constexpr int DT = DT_, CT = I8_ ? VI_F16 : DT_, DP = DP_, WM = WM_, WK = WK_, ST = WM > 1 ? 2 : 1;
    static constexpr bool I8 = I8_;
    static constexpr int WAVES = WM * WK, THREADS = 64 * WAVES, ROWS = 32 * WM, OCC = OCC_ * WAVES / 4 > 0 ? OCC_ * WAVES / 4 : 1;           // wavefronts of a SIMD
    static constexpr int KEYS = WM > 1 ? 64 : 32, GROUPS = KEYS / 16;  // of a stage; sixteen keys are of one page
    static constexpr int ROW = DP * (I8 ? 1 : 2), UNITS = ROW / 16, PER_LOAD = 64 / UNITS, LOADS = 16 / PER_LOAD;       // bytes, units; rows of a load, loads of a group
    static constexpr int SCALES = I8 ? KEYS * 4 : 0, HALF = KEYS * ROW + SCALES, STAGE = 2 * HALF;
    static constexpr int MINE = GROUPS * LOADS / WM, KINDS = LOADS > WM ? LOADS / WM : 1;              // loads of a wavefront in half a stage, different ones of a group
    // fp16's weights are 2^RAISED times as large, sums with them: up to 2^15, so that those 2^-21 of the largest still have all digits, and 2^-32 of it is half a step
    static constexpr float RAISED = DT_ == VI_F16 && !I8_ ? 7.0f : 0.0f;
    static constexpr int PITCH = 36;           // floats between rows of 32 on their way out
    static constexpr int OUT = WAVES * 32 * PITCH * 4 + WAVES * 32 * 8 + ROWS * 8;
    static constexpr int LDS = WK * ST * STAGE > OUT ? WK * ST * STAGE : OUT;
    static constexpr int MASKS = ROWS < MAX_NODES ? ROWS : MAX_NODES;
    static_assert(GROUPS * LOADS % WM == 0 && (LOADS % WM == 0 || WM % LOADS == 0) && (WM == 1 ? GROUPS == 2 : GROUPS == WM), "loads of a stage");
};

struct Args {
    Cache cache;
    Batch batch;
    const void *q;
    void *out;
    i64 q_token, q_head, out_token, out_head, n;
    const int *parents;
    int heads, group, tiles, splits, per_split, clear;                 // per_split: keys
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
    const u64 b = (u64)__builtin_amdgcn_readfirstlane((u32)((u64)base >> 32)) << 32 | (u32)__builtin_amdgcn_readfirstlane((u32)(u64)base);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(at), "v"(off), "s"(b) : "memory");
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
// its LDS accesses are done
__device__ __forceinline__ void read() { asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory"); }
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
// Eight 8-bit integers, + 128 and so 0 to 255, as the fp16 numbers that these are as they lie: 2^-24 of them, below the smallest normal number, which the matrix
// instructions take as it is.  Of each four the first and third come first, then the other two (in two_of's order).
constexpr float OF_BYTES = 0x1p24f, MIDDLE = 128.0f;
__device__ __forceinline__ v4u widen(v2u w) {
    v4u r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const u32 u = w[i] ^ 0x80808080u;
        r[2 * i] = u & 0x00FF00FFu, r[2 * i + 1] = __builtin_amdgcn_perm(u, u, 0x0C030C01u);
    }
    return r;
}

__device__ __forceinline__ int two_of(int i) { return i / 2 * 4 + i % 2; }            // the first of word i
__device__ __forceinline__ float element_of(v4u w, int i) { return (float)__builtin_bit_cast(_Float16, (unsigned short)(w[i / 2] >> (16 * (i & 1)))); }
// the sum of both halves of a word and c
template <int DT>
__device__ __forceinline__ float add_two(u32 w, float c) {
    typedef typename type<DT>::t v2t __attribute__((ext_vector_type(2)));
    const v2t ones = {(typename type<DT>::t)1.0f, (typename type<DT>::t)1.0f}, two = __builtin_bit_cast(v2t, w);
    if constexpr (DT == VI_BF16) return __builtin_amdgcn_fdot2_f32_bf16(two, ones, c, false);
    else return __builtin_amdgcn_fdot2(two, ones, c, false);
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
__device__ __forceinline__ float sum_of_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ int same(int v) { return (int)__builtin_amdgcn_readfirstlane((u32)v); }

// ---- which rows ---------------------------------------------------------------------------------------------------
// Sequence b's tiles begin at starts[b] group / rows + b: apart by at least as many as it needs, and no sequence's start has to be known to count them.
struct Tile {
    int b, n, first;                           // sequence, its new tokens, the tile's first row in it
    int s0, context, end;                      // its first row; entries before the new ones; the key behind the last that a row of the tile may attend to
};
template <int ROWS>
__device__ __forceinline__ bool find_tile(const Args &A, int tile, Tile *t) {
    int found = -1, s0 = 0, s1 = 0, length = 0;
    for (int first = 0; first < A.batch.sequences; first += 64) {
        const int b = min(first + (int)(threadIdx.x & 63), A.batch.sequences - 1);
        const i64 here = max((i64)0, min((i64)A.batch.starts[b], A.n)), next = max((i64)0, min((i64)A.batch.starts[b + 1], A.n));
        const int its = max(A.batch.lengths[b], 0);
        const int count = __popcll(__ballot(first + (int)(threadIdx.x & 63) < A.batch.sequences && here * A.group / ROWS + b <= tile));
        if (count == 0) break;                 // starts rises
        found = first + count - 1;
        s0 = __shfl((int)here, count - 1), s1 = __shfl((int)next, count - 1), length = __shfl(its, count - 1);
    }
    if (found < 0) return false;
    found = same(found), s0 = same(s0), s1 = same(s1), length = same(length);
    const i64 first = ((i64)tile - found - (i64)s0 * A.group / ROWS) * ROWS;
    t->b = found, t->n = s1 - s0, t->s0 = s0, t->first = (int)first, t->context = length - t->n;
    if (first < 0 || first >= (i64)t->n * A.group) return false;       // less than 0 where starts does not rise
    const int last = min(t->n - 1, (int)((u32)(t->first + ROWS - 1) / (u32)A.group));
    t->end = (int)max((i64)0, min(min((i64)length, A.batch.most), (i64)t->context + last + 1));
    return true;
}

// how many workgroups share a tile's keys: the last has what is left
__device__ __forceinline__ int parts_of(const Args &A, int end) { return max(1, min(A.splits, (end + A.per_split - 1) / A.per_split)); }

// ---- the pass over the keys ---------------------------------------------------------------------------------------
template <class F>
__global__ __launch_bounds__(F::THREADS, F::OCC) void k_attend(Args A) {
    constexpr int DT = F::DT, CT = F::CT, DP = F::DP, WM = F::WM, WK = F::WK, ROW = F::ROW, UNITS = F::UNITS;
    constexpr bool NARROW = F::I8;             // 8-bit integers in LDS
    typedef typename type<DT>::t T;
    __shared__ char lds[F::LDS] __attribute__((aligned(16)));
    __shared__ u32 masks[F::MASKS * MASK_WORDS];
    __shared__ int above[MAX_NODES];
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = same((int)threadIdx.x >> 6), wm = WM == 1 ? 0 : WK == 1 ? wave : wave % WM, part = WK == 1 ? 0 : WM == 1 ? wave : wave / WM;
    const int heads = (int)A.cache.heads, head = (int)blockIdx.x % heads, split = (int)blockIdx.x / heads % A.splits;
    const int tile = A.tiles - 1 - (int)blockIdx.x / heads / A.splits;         // the longest first, where a prompt's tiles differ

    if (A.clear && blockIdx.x < CLEARING) {    // rows of no sequence
        const i64 s0 = A.batch.sequences ? max((i64)0, min((i64)A.batch.starts[0], A.n)) : A.n, s1 = A.batch.sequences ? max(s0, min((i64)A.batch.starts[A.batch.sequences], A.n)) : A.n;
        for (i64 r = blockIdx.x; r < s0 + A.n - s1; r += min(CLEARING, (int)gridDim.x))
            for (int i = threadIdx.x; i < A.heads * A.cache.dim; i += F::THREADS)
                ((T *)A.out)[(r < s0 ? r : s1 + r - s0) * A.out_token + i / A.cache.dim * A.out_head + i % A.cache.dim] = (T)0.0f;
    }
    Tile t;
    if (!find_tile<F::ROWS>(A, tile, &t)) return;
    const int end = t.end, context = t.context;
    const bool tree = A.parents && t.n <= MAX_NODES;
    auto token = [&](int row) INLINE { return (int)((u32)row / (u32)A.group); };
    // a workgroup's part of the keys; where one has all of them it is done with that
    const int first_key = split * A.per_split, parts = parts_of(A, end);
    if (split >= parts) return;
    const int stages = ((split == parts - 1 ? end - first_key : A.per_split) + F::KEYS * WK - 1) / (F::KEYS * WK);       // of each of the WK groups
    const i64 slot = ((i64)tile * heads + head) * A.splits + split;
    // the wavefront's rows attend to keys below wave_end, all of them to those below wave_free
    const int row0 = t.first + wm * 32, wave_first = token(row0), wave_last = min(t.n - 1, token(row0 + 31));
    const int wave_end = wave_first < t.n ? min(end, context + wave_last + 1) : 0, wave_free = tree ? context : context + wave_first + 1;

    // queries: unit (of eight columns) `chunk` of a row for half and step
    const int row = row0 + (lane & 31), tok = token(row);
    const bool there = tok < t.n;
    v4u q[DP / 16];
    {
        const T *x = (const T *)A.q + ((i64)t.s0 + (there ? tok : 0)) * A.q_token + (head * A.group + (there ? row - tok * A.group : 0)) * A.q_head;
#pragma unroll
        for (int st = 0; st < DP / 16; ++st) {
            const int chunk = NARROW ? 4 * (st / 2) + 2 * half + st % 2 : 2 * st + half;
            q[st] = v4u{0, 0, 0, 0};
            if (there && chunk * 8 < A.cache.dim) q[st] = load_any<v4u>(x + chunk * 8);
        }
    }
    // For 8-bit integers a row's queries are fp16, their largest brought to 2^14 by a power of two, which goes into what its scores are multiplied by: exact, but for
    // numbers 2^28 times smaller than the largest.  What the integers are more than themselves is taken off from the start.
    float c = A.c, start = 0;
    if constexpr (F::I8) {
        auto number = [](const v4u &w, int i) INLINE { return __uint_as_float(i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16); };          // bfloat16
        float largest = 0;
#pragma unroll
        for (int st = 0; st < DP / 16; ++st)
#pragma unroll
            for (int i = 0; i < 8; ++i) largest = fmaxf(largest, fabsf(number(q[st], i)));
        const u32 exponent = __float_as_uint(most_of_halves(largest)) >> 23, e = exponent == 255 ? 141 : max(exponent, 15u);
        const float by = __uint_as_float((268 - e) << 23);
        c = fmaxf(c * OF_BYTES * __uint_as_float((e - 14) << 23), 0x1p-126f);      // nothing would make a NaN of a hidden key's -inf; scores that this is much for are nothing either
#pragma unroll
        for (int st = 0; st < DP / 16; ++st) {
            v4u r;
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = pack<CT>(number(q[st], two_of(i)) * by, number(q[st], two_of(i) + 2) * by);
            q[st] = r;
#pragma unroll
            for (int i = 0; i < 8; ++i) start += element_of(r, i);
        }
        start = sum_of_halves(start) * (-MIDDLE / OF_BYTES);
    }

    // ---- stages
    const u32 lds_at = (u32)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    const char *from[2];
    const float *scales_from[2];
    u32 page_apart[2], row_apart[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        from[h] = A.cache.half[h].at + head * A.cache.half[h].head, scales_from[h] = F::I8 ? A.cache.half[h].scales + head * A.cache.half[h].scale_head : nullptr;
        page_apart[h] = (u32)A.cache.half[h].page, row_apart[h] = (u32)A.cache.half[h].row;
    }
    const int full_units = A.cache.dim * (F::I8 ? 1 : 2) / 16, row_mask = A.cache.mask;
    const u32 n_pages = (u32)A.cache.pages;
    const bool one_page = row_mask >= F::KEYS - 1;                     // a stage has entries of one page
    typedef const __attribute__((address_space(4))) int *Table;        // constant while the kernel runs: read by the scalar cache
    const Table pages = (Table)(A.batch.pages + t.b * A.batch.stride);
    auto stage_key = [&](int it) INLINE { return first_key + (it * WK + part) * F::KEYS; };
    struct Pages {
        int number[F::GROUPS];                 // of sixteen keys each: only the first is looked at where a stage is in one page
    };
    auto look_up = [&](int it) INLINE {
        const int j = stage_key(it);
        Pages p;
#pragma unroll
        for (int g = 0; g < F::GROUPS; ++g) p.number[g] = pages[min(j + 16 * g, end - 1) >> A.cache.shift];
        return p;
    };
    auto number_of = [&](const Pages &p, int g) INLINE {
        const int first = p.number[0], own = p.number[g];
        return one_page ? first : own;
    };
    // how many of the sixteen keys from j on there are
    auto valid_of = [&](int number, int j) INLINE { return (u32)number < n_pages ? max(0, min(16, end - j)) : 0; };
    // whether a stage has all its keys, and columns fill the units
    auto whole = [&](const Pages &p, int j) INLINE {
        bool all = full_units == UNITS && j + F::KEYS <= end && (u32)p.number[0] < n_pages;
        if (!one_page) {
#pragma unroll
            for (int g = 1; g < F::GROUPS; ++g) all = all && (u32)p.number[g] < n_pages;
        }
        return all;
    };
    // A lane's unit of 16 bytes in a load: its row is lane / UNITS and a multiple of PER_LOAD behind, and rows differ in the order of their units.  A wavefront
    // has KINDS different loads of sixteen keys.
    const int lane_row = lane / UNITS, wave_load = F::LOADS >= WM ? wm : wm % F::LOADS;
    u32 lane_unit[F::KINDS], lane_off[2];
#pragma unroll
    for (int k = 0; k < F::KINDS; ++k) lane_unit[k] = (u32)(lane % UNITS ^ order<UNITS>((k * WM + wave_load) * F::PER_LOAD + lane_row)) * 16;
#pragma unroll
    for (int h = 0; h < 2; ++h) lane_off[h] = (u32)(wave_load * F::PER_LOAD + lane_row) * row_apart[h];
    // The keys (h = 0) or values of a stage on their way to its slot: MINE loads, and one of scales, where it is whole (fewer, and zeros in the places of
    // the others, elsewhere).
    auto fetch = [&](int h, u32 place, int j, const Pages &p, bool all) INLINE {
        const u32 wave_place = lds_at + place + (u32)(wave_load * 1024 + (F::LOADS >= WM ? 0 : wm / F::LOADS * 16 * ROW));
        // sixteen keys after sixteen; where a group has fewer loads than there are wavefronts, these are at several groups at a time
        constexpr int STEP = F::LOADS >= WM ? 1 : WM / F::LOADS;
        const int mine = F::LOADS >= WM ? 0 : wm / F::LOADS;
        if (all && one_page) {
            const char *b = from[h] + (u64)(u32)p.number[0] * page_apart[h] + (u32)((j & row_mask) + 16 * mine) * row_apart[h];
#pragma unroll
            for (int l = 0; l < F::MINE; ++l) {
                const int g = l / F::KINDS * STEP, k = l % F::KINDS;
                fetch_to_lds(wave_place + (u32)(g * 16 * ROW + k * WM * 1024), lane_off[h] + lane_unit[k], b + (u32)(16 * g + k * WM * F::PER_LOAD) * row_apart[h]);
            }
        } else {
#pragma unroll
            for (int l = 0; l < F::MINE; ++l) {
                const int g = l / F::KINDS * STEP, k = l % F::KINDS, jj = j + 16 * (g + mine);
                int number = number_of(p, g);
#pragma unroll
                for (int o = 1; o < STEP; ++o) number = mine == o ? number_of(p, g + o) : number;
                const u32 at = wave_place + (u32)(g * 16 * ROW + k * WM * 1024);
                const char *b = from[h] + (u64)(u32)number * page_apart[h] + (u32)((jj & row_mask) + k * WM * F::PER_LOAD) * row_apart[h];
                const int r = (k * WM + wave_load) * F::PER_LOAD + lane_row;
                if (r < valid_of(number, jj) && (int)lane_unit[k] < full_units * 16) fetch_to_lds(at, lane_off[h] + lane_unit[k], b);
                else *(v4u *)(lds + (at - lds_at) + lane * 16) = v4u{0, 0, 0, 0};
            }
        }
        if constexpr (F::I8) {                 // a scale a lane: a wavefront alone has the stage's 32, four have sixteen each
            constexpr int SCALES = F::KEYS / WM;
            const int g = WM == 1 ? lane >> 4 & 1 : wm, jj = j + 16 * g;
            int number = number_of(p, 0);
#pragma unroll
            for (int o = 1; o < F::GROUPS; ++o) number = g == o ? number_of(p, o) : number;
            const u32 at = place + F::KEYS * ROW + (WM == 1 ? 0 : wm * 64);
            if (lane < SCALES) {
                if ((lane & 15) < valid_of(number, jj)) fetch_words_to_lds(lds_at + at, scales_from[h] + number * A.cache.half[h].scale_page + (jj & row_mask) + (lane & 15));
                else *(float *)(lds + at + lane * 4) = 0.0f;
            }
        }
    };
    constexpr int LOADS_OF_HALF = F::MINE + (F::I8 ? 1 : 0);
    auto place_of = [&](int h, int into) INLINE { return (u32)((part * F::ST + into) * F::STAGE + h * F::HALF); };

    // the rows' ancestors among the new tokens, a bit each
    if (tree) {
        const int first = token(t.first), last = min(t.n - 1, token(t.first + F::ROWS - 1));
        for (int i = threadIdx.x; i < t.n; i += F::THREADS) above[i] = A.parents[t.s0 + i];
        __syncthreads();
        for (int i = first + (int)threadIdx.x; i <= last; i += F::THREADS) {
            u32 *bits = masks + (i - first) * MASK_WORDS;
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
    const u32 *mask = masks + (tree && there ? tok - token(t.first) : 0) * MASK_WORDS;

    v16f o[DP / 32];
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) o[db] = v16f{};
    // For 8-bit integers, exponentials times scales are multiplied by `gain` to be in fp16's range: a power of two at first, 2^14 at most of the largest so far.
    float gain = MAX_GAIN, weighed = 0;
    float most = -INFINITY, relative = -INFINITY, sum = 0, sum_odd = 0;             // largest score so far (or up to LATE behind), times c: what the sums are relative to

    // which of the 32 keys from j on the lane's row attends to; the low and the high sixteen have so many
    auto window_of = [&](int j, int low, int high) INLINE {
        u32 w = ~0u;
        if (there && !tree) {
            const int left = context + tok + 1 - j;
            w = left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1;
        } else if (there) {
            const int node = j - context;
            if (node >= MAX_NODES) w = 0;
            else if (node >= 0) w = (u32)(((u64)mask[(node >> 5) + 1] << 32 | mask[node >> 5]) >> (node & 31));
            else if (node > -32) w = mask[0] << -node | ((1u << -node) - 1);
        }
        return w & ((low >= 16 ? 0xFFFFu : (1u << low) - 1) | (high >= 16 ? 0xFFFFu : (1u << high) - 1) << 16);
    };
    auto bit_of = [&](int r) INLINE { return 8 * (r / 4) + 4 * half + r % 4; };

    // where a lane reads keys and values in a stage: kept in registers, the compiler would make them anew each time
    u32 key_at[DP / 16], value_at[DP / 32][2];
    {
        const int r_ = lane & 31, in = lane & 15, right = lane >> 4 & 1;
#pragma unroll
        for (int st = 0; st < (NARROW ? DP / 32 : DP / 16); ++st) key_at[st] = (u32)(r_ * ROW + ((2 * st + half) ^ order<UNITS>(r_ & 15)) * 16);
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int i = 0; i < (NARROW ? 1 : 2); ++i) {
                const int row8 = (in >> 3) * 8 + 4 * half + (in >> 1 & 3), row16 = 8 * i + 4 * half + (in >> 2);
                value_at[db][i] = NARROW ? (u32)(row8 * ROW + ((2 * db + right) ^ order<UNITS>(row8)) * 16 + (in & 1) * 8)
                                         : (u32)(row16 * ROW + ((4 * db + 2 * right + (in >> 1 & 1)) ^ order<UNITS>(row16)) * 16 + (in & 1) * 8);
            }
#pragma unroll
        for (int st = 0; st < (NARROW ? DP / 32 : DP / 16); ++st) asm volatile("" : "+v"(key_at[st]));
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int i = 0; i < (NARROW ? 1 : 2); ++i) asm volatile("" : "+v"(value_at[db][i]));
    }

    v16f starts;                               // kept in registers like those
#pragma unroll
    for (int r = 0; r < 16; ++r) starts[r] = start;
    if constexpr (F::I8) asm volatile("" : "+v"(starts));
    // Scores of 32 keys: k is their rows in LDS, `scales` theirs.  `beside(st)` is done between the products, two of the keys' units ahead of which are on their
    // way.
    auto scores_beside = [&](const char *k, const char *scales, auto beside) INLINE {
        constexpr int READS = DP / 16 / (NARROW ? 2 : 1);
        v16f s = {};
        if constexpr (NARROW) s = starts;
        v4u w[READS];
#pragma unroll
        for (int i = 0; i < 2; ++i) w[i] = *(const v4u *)(k + key_at[i]);
#pragma unroll
        for (int i = 0; i < READS; ++i) {
            if (i + 2 < READS) w[i + 2] = *(const v4u *)(k + key_at[i + 2]);
            if constexpr (NARROW) {
                s = multiply<CT>(widen(v2u{w[i].x, w[i].y}), q[2 * i], s);
                beside(2 * i);
                s = multiply<CT>(widen(v2u{w[i].z, w[i].w}), q[2 * i + 1], s);
                beside(2 * i + 1);
            } else {
                s = multiply<CT>(w[i], q[i], s);
                beside(i);
            }
        }
        if constexpr (F::I8) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const v4f f = *(const v4f *)(scales + (8 * g + 4 * half) * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) s[4 * g + i] *= f[i];
            }
        }
        return s;
    };
    auto scores = [&](const char *k, const char *scales) INLINE { return scores_beside(k, scales, [](int) INLINE {}); };

    // V^T of 32 columns and 16 keys, in the order of the registers: four from 4 half on, four from 8 + 4 half on
    auto columns = [&](const char *v, int db, int st) INLINE {
        if constexpr (NARROW) {
            const v2u w = read_columns8(v + value_at[db][0] + st * 16 * ROW);
            return v4u{w.x, w.y, 0, 0};
        } else {
            const v2u one = read_columns16(v + value_at[db][0] + st * 16 * ROW), two = read_columns16(v + value_at[db][1] + st * 16 * ROW);
            return v4u{one.x, one.y, two.x, two.y};
        }
    };

    // masked scores are none; the sums are kept relative to about the largest
    auto settle = [&](v16f &s, bool masked, u32 window) INLINE {
        if (masked) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = window >> bit_of(r) & 1 ? s[r] : -INFINITY;
        }
        float top = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
        top = most_of_halves(top);
        if (__any(top * c > relative + LATE)) {
            asm volatile("");                  // a branch: the compiler would multiply by one, each time
            const float now = fmaxf(most, top), then = now * c;
            const float by = relative == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(relative - then);
            most = now, relative = then, sum *= by, sum_odd *= by;
            float less = by;                   // of the products' sums: where they have a power of their own that follows
            if constexpr (F::I8) {
                // MAX_GAIN / gain may be beyond 32 bits where `by` is nothing; what both come to is 1 at most
                const float more = fminf(gain / by, MAX_GAIN);
                less = more < MAX_GAIN ? 1.0f : by * 0x1p63f / gain * (MAX_GAIN * 0x1p-63f);
                gain = more, weighed *= less;
            }
#pragma unroll
            for (int db = 0; db < DP / 32; ++db) o[db] *= less;
        }
    };
    auto base_of = [&](float relative) INLINE { return relative == -INFINITY ? 0.0f : relative - F::RAISED; };
    // The exponentials of scores, as the second operand of the product with V^T.
    struct Weights {
        float of[16];
    };
    // values' scales; in a masked place there may be anything
    auto scales_of = [&](const v16f &s, const char *scales, bool masked) INLINE {
        Weights f = {};
        if constexpr (F::I8) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const v4f four = *(const v4f *)(scales + (8 * g + 4 * half) * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) f.of[4 * g + i] = four[i];
            }
            if (masked) {
                asm volatile("");
#pragma unroll
                for (int r = 0; r < 16; ++r) f.of[r] = s[r] == -INFINITY ? 0.0f : f.of[r];
            }
        }
        return f;
    };
    // two exponentials, times their scales; the pair goes into word i of the operand
    auto weigh = [&](const v16f &s, Weights &f, float base, int i) INLINE {
        const int one = F::I8 ? i / 4 * 8 + two_of(i % 4) : 2 * i, two = F::I8 ? one + 2 : one + 1;
        const float a = __builtin_amdgcn_exp2f(fmaf(s[one], c, -base)), b = __builtin_amdgcn_exp2f(fmaf(s[two], c, -base));
        if (F::I8) sum += a + b;               // others as rounded (word_of)
        f.of[one] = F::I8 ? a * f.of[one] : a, f.of[two] = F::I8 ? b * f.of[two] : b;
    };
    // The sum is of what is multiplied, rounded, so that values all alike come out as they are (a prompt of 4096, four heads to one of the cache, 180 us, 176 with the sum of the exponentials
    // themselves, which was 0.3 per cent off beside one late key); in two, for an addition waits for the one before.  For 8-bit integers it cannot be, for their weights have scales in them.
    auto word_of = [&](const Weights &f, int i) INLINE {
        const int one = F::I8 ? i / 4 * 8 + two_of(i % 4) : 2 * i, two = F::I8 ? one + 2 : one + 1;
        const u32 word = F::I8 ? pack<CT>(f.of[one] * gain, f.of[two] * gain) : pack<CT>(f.of[one], f.of[two]);
        if constexpr (!F::I8) (i & 1 ? sum_odd : sum) = add_two<CT>(word, i & 1 ? sum_odd : sum);
        return word;
    };
    // For 8-bit integers: in fp16's range, and what the integers are more than themselves goes by them as rounded
    auto words_of = [&](const Weights &f, v4u (&p)[2]) INLINE {
        if constexpr (F::I8) {
            float top = 0;
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(f.of[r]));
            if (__any(top * gain > 0x1p14f)) {
                asm volatile("");
                float finite = 0;
#pragma unroll
                for (int r = 0; r < 16; ++r) finite = fmaxf(finite, fabsf(f.of[r]) < INFINITY ? fabsf(f.of[r]) : 0.0f);
                finite = most_of_halves(finite);
                if (finite * gain > 0x1p14f) {
                    const float now = __uint_as_float(max(254u - (__float_as_uint(finite) >> 23), 1u) << 23), by = now / gain;
                    gain = now, weighed *= by;
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db) o[db] *= by;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[i / 4][i % 4] = word_of(f, i);
            if constexpr (F::I8) weighed = add_two<CT>(p[i / 4][i % 4], weighed);
        }
    };
    auto weights = [&](const v16f &s, const char *scales, bool masked, v4u (&p)[2]) INLINE {
        Weights f = scales_of(s, scales, masked);
        const float base = base_of(relative);
#pragma unroll
        for (int i = 0; i < 8; ++i) weigh(s, f, base, i);
        words_of(f, p);
    };
    // The same with the next keys' scores beside them, product after product between the exponentials: in an order of its own, for the compiler would take the
    // products one after the other, each of which waits for the one before (4096 tokens of a prompt 206 us so, 201 in this order).
    auto weights_and_scores = [&](const v16f &s, const char *scales, bool masked, v4u (&p)[2], const char *k, const char *key_scales) INLINE {
        Weights f = scales_of(s, scales, masked);
        const float base = base_of(relative);
        constexpr int PRODUCTS = DP / 16;
        __builtin_amdgcn_sched_barrier(0);
        const v16f ahead = scores_beside(k, key_scales, [&](int st) INLINE {
#pragma unroll
            for (int i = st * 8 / PRODUCTS; i < (st + 1) * 8 / PRODUCTS; ++i) {
                weigh(s, f, base, i);
                if constexpr (!F::I8) {
                    u32 here = word_of(f, i);
                    asm volatile("" : "+v"(here));                     // not behind the branches that follow
                    p[i / 4][i % 4] = here;
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        });
        if constexpr (F::I8) words_of(f, p);
        return ahead;
    };

    // 0 times an infinity or a NaN in a masked place would be a NaN.  Where keys are masked such values are left out of the products, and seen once more behind
    // the pass, for the rows that attend to them.  (Those of 8-bit integers are in the scales.)
    constexpr u32 INF = DT == VI_BF16 ? 0x7F80u : 0x7C00u;
    bool wild = false;
    auto tame = [&](v4u &w) INLINE {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool low = (w[i] & INF) == INF, high = (w[i] & INF << 16) == INF << 16;
            w[i] = high ? w[i] & 0xFFFFu : w[i];
            w[i] = low ? w[i] & 0xFFFF0000u : w[i];
            wild = wild || low || high;
        }
    };
    auto add_values = [&](const char *v, const v4u (&p)[2], bool masked) INLINE {
        v4u w[DP / 32][2];
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int st = 0; st < 2; ++st) w[db][st] = columns(v, db, st);
        if constexpr (!F::I8) {
            if (masked) {
#pragma unroll
                for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                    for (int st = 0; st < 2; ++st) tame(w[db][st]);
            }
        }
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                if constexpr (NARROW) o[db] = multiply<CT>(widen(v2u{w[db][st].x, w[db][st].y}), p[st], o[db]);
                else o[db] = multiply<CT>(w[db][st], p[st], o[db]);
            }
    };

    if constexpr (WM == 1) {
        // A wavefront's own keys: each half of its stage is asked for anew as soon as it has been used, under the work on the other half.
        Pages now = {}, next = {};
        bool now_whole = false;
        if (stages) {
            now = look_up(0);
            now_whole = whole(now, stage_key(0));
            fetch(0, place_of(0, 0), stage_key(0), now, now_whole);
            fetch(1, place_of(1, 0), stage_key(0), now, now_whole);
        }
        if (stages > 1) next = look_up(1);
        const char *k = lds + part * F::STAGE, *v = k + F::HALF;
#pragma unroll 1
        for (int it = 0; it < stages; ++it) {
            const int j = stage_key(it);
            const bool more = it + 1 < stages, next_whole = more && whole(next, stage_key(it + 1)), needed = j < wave_end;
            if (now_whole) arrive<LOADS_OF_HALF>();
            else arrive<0>();
            meet_wave();
            v16f s;                            // of keys that are needed
            if (needed) s = scores(k, k + F::KEYS * ROW);
            if (more) {
                read();
                meet_wave();
                fetch(0, place_of(0, 0), stage_key(it + 1), next, next_whole);
            }
            const int low = now_whole ? 16 : valid_of(now.number[0], j), high = now_whole ? 16 : valid_of(number_of(now, 1), j + 16);
            const bool masked = low < 16 || high < 16 || j + 32 > wave_free;
            if (next_whole) arrive<LOADS_OF_HALF>();
            else arrive<0>();
            meet_wave();
            if (needed) {
                v4u p[2];
                settle(s, masked, masked ? window_of(j, low, high) : ~0u);
                weights(s, v + F::KEYS * ROW, masked, p);
                add_values(v, p, masked);
            }
            if (more) {
                read();
                meet_wave();
                fetch(1, place_of(1, 0), stage_key(it + 1), next, next_whole);
                now = next, now_whole = next_whole;
                if (it + 2 < stages) next = look_up(it + 2);
            }
        }
    } else {
        // Keys that WM wavefronts share, a stage of 64 in two steps of 32.  The scores of a step's keys are taken in the step before, under the exponentials there:
        // the second step of a stage is the last that reads the stage's values and the first that reads the next one's keys, so that the values of stage
        // it + 1 are asked for in the first step of stage it, and the keys of stage it + 2 in the second; both have two steps to come.
        auto key_rows = [&](int slot, int kb) INLINE { return lds + place_of(0, slot) + kb * 32 * ROW; };
        auto key_scales = [&](int slot, int kb) INLINE { return lds + place_of(0, slot) + F::KEYS * ROW + kb * 128; };
        v16f s = {};
        Pages next = {}, behind = {};          // of stages it + 1 and it + 2
        bool all = false, next_all = false;    // whether stages it and it + 1 are whole
        if (stages) {
            const Pages now = look_up(0);
            all = whole(now, stage_key(0));
            if (stages > 1) next = look_up(1);
            next_all = stages > 1 && whole(next, stage_key(1));
            if (stages > 2) behind = look_up(2);
            fetch(0, place_of(0, 0), stage_key(0), now, all);
            fetch(1, place_of(1, 0), stage_key(0), now, all);
            if (stages > 1) fetch(0, place_of(0, 1), stage_key(1), next, next_all);
            arrive<0>();
            meet_group();
            s = scores(key_rows(0, 0), key_scales(0, 0));
        }
        auto step = [&](int it, auto slot, int kb, const char *k, const char *scales) INLINE {
            const int j = stage_key(it) + 32 * kb;
            if (j >= wave_end) return;
            int low = 16, high = 16;
            if (!all) {
                const Pages p = look_up(it);
                low = valid_of(number_of(p, 2 * kb), j), high = valid_of(number_of(p, 2 * kb + 1), j + 16);
            }
            const bool masked = low < 16 || high < 16 || j + 32 > wave_free;
            settle(s, masked, masked ? window_of(j, low, high) : ~0u);
            v4u p[2];
            const v16f ahead = weights_and_scores(s, lds + place_of(1, decltype(slot)::value) + F::KEYS * ROW + kb * 128, masked, p, k, scales);      // behind the last stage: of what lies there, and not used
            add_values(lds + place_of(1, decltype(slot)::value) + kb * 32 * ROW, p, masked);
            s = ahead;
        };
        auto arrived = [&]() INLINE {          // all but what was asked for in the step before, which is of stage it + 1
            if (next_all) arrive<LOADS_OF_HALF>();
            else arrive<0>();
            meet_group();
        };
        // `slot` is it % 2 and known, so that places in LDS are in the instructions (201 us with it % 2 in registers, 198)
        auto stage = [&](int it, auto slot) INLINE {
            constexpr int own = decltype(slot)::value, other = 1 - own;
            arrived();
            if (it + 1 < stages) fetch(1, place_of(1, other), stage_key(it + 1), next, next_all);
            step(it, slot, 0, key_rows(own, 1), key_scales(own, 1));
            arrived();
            const bool behind_all = it + 2 < stages && whole(behind, stage_key(it + 2));
            if (it + 2 < stages) fetch(0, place_of(0, own), stage_key(it + 2), behind, behind_all);
            next = behind;
            if (it + 3 < stages) behind = look_up(it + 3);
            step(it, slot, 1, key_rows(other, 0), key_scales(other, 0));
            all = next_all, next_all = behind_all;
        };
#pragma unroll 1
        for (int it = 0; it < stages; it += 2) {
            stage(it, std::integral_constant<int, 0>());
            if (it + 1 < stages) stage(it + 1, std::integral_constant<int, 1>());
        }
    }

    // ---- the values that were left out, of the keys that some row of the wavefront does not attend to, by those that do
    if constexpr (!F::I8) {
        if (__any(wild)) {
#pragma unroll 1
            for (int i = 0; i < stages * (F::KEYS / 32); ++i) {
                const int it = i / (F::KEYS / 32), j = stage_key(it) + i % (F::KEYS / 32) * 32;
                if (j >= wave_end) break;
                const int one = pages[j >> A.cache.shift], two = pages[min(j + 16, end - 1) >> A.cache.shift], low = valid_of(one, j), high = valid_of(two, j + 16);
                if (low == 16 && high == 16 && j + 32 <= wave_free) continue;
                const u32 window = there ? window_of(j, low, high) : 0;
#pragma unroll 1
                for (int k = 0; k < 32; ++k) {
                    if (!(window >> k & 1)) continue;
                    const T *x = (const T *)(from[1] + (u64)(u32)(k < 16 ? one : two) * page_apart[1] + (u32)((j + k) & row_mask) * row_apart[1]);
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int col = 32 * db + bit_of(r);
                            const float f = col < A.cache.dim ? (float)x[col] : 0.0f;
                            if (!(fabsf(f) < INFINITY)) o[db][r] += f;
                        }
                }
            }
        }
    }

    // ---- the WK groups' sums as one, and out
    arrive<0>();
    __syncthreads();
    float *buf = (float *)lds, *of_waves = buf + F::WAVES * 32 * F::PITCH, *of_rows = of_waves + F::WAVES * 32 * 2;
    {
        sum = sum_of_halves(sum + sum_odd);
        if (half == 0) of_waves[(wave * 32 + lane) * 2] = relative, of_waves[(wave * 32 + lane) * 2 + 1] = sum;
    }
    __syncthreads();
    float top = -INFINITY, total = 0;
#pragma unroll
    for (int w = 0; w < WK; ++w) top = fmaxf(top, of_waves[((w * WM + wm) * 32 + (lane & 31)) * 2]);
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int w = 0; w < WK; ++w) {
        const float *x = of_waves + ((w * WM + wm) * 32 + (lane & 31)) * 2;
        total += __builtin_amdgcn_exp2f(x[0] - base) * x[1];
    }
    const float factor = __builtin_amdgcn_exp2f(relative - base) * (F::I8 ? 1.0f / gain : 1.0f);
    if constexpr (F::I8) {
        const float more = sum_of_halves(weighed) * -MIDDLE;
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[db][r] = fmaf(o[db][r], OF_BYTES, more);
    }
    if (part == 0 && half == 0) of_rows[(wm * 32 + lane) * 2] = top, of_rows[(wm * 32 + lane) * 2 + 1] = total;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) {
        if (db) __syncthreads();
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const v4f x = {o[db][4 * g] * factor, o[db][4 * g + 1] * factor, o[db][4 * g + 2] * factor, o[db][4 * g + 3] * factor};
            *(v4f *)(buf + (wave * 32 + (lane & 31)) * F::PITCH + 8 * g + 4 * half) = x;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < F::ROWS * 8; i += F::THREADS) {
            const int r = i / 8, col = 32 * db + i % 8 * 4, its = t.first + r, of = token(its);
            if (of >= t.n || col >= A.cache.dim) continue;
            v4f x = *(const v4f *)(buf + r * F::PITCH + i % 8 * 4);
#pragma unroll
            for (int w = 1; w < WK; ++w) x += *(const v4f *)(buf + (w * F::ROWS + r) * F::PITCH + i % 8 * 4);
            if (parts > 1) {
                *(v4f *)(A.part + (slot * F::ROWS + r) * DP + col) = x;
            } else {
                const float all = of_rows[r * 2 + 1], per = all == 0.0f ? 0.0f : 1.0f / all;
                const v2u two = {pack<DT>(x.x * per, x.y * per), pack<DT>(x.z * per, x.w * per)};
                store_any((T *)A.out + ((i64)t.s0 + of) * A.out_token + (head * A.group + its - of * A.group) * A.out_head + col, two);
            }
        }
    }
    if (parts > 1)
        for (int r = threadIdx.x; r < F::ROWS; r += F::THREADS) {
            A.most[(slot * F::ROWS + r) * 2] = of_rows[r * 2];
            A.most[(slot * F::ROWS + r) * 2 + 1] = of_rows[r * 2 + 1];
        }
}

// What the workgroups of a tile have left, as one.  A thread has four columns of a row and every GROUPS-th part: all of them where parts are few, so that a workgroup
// has several rows, else as many groups as a row leaves room for (64 parts of a token over 32768 entries, 8 heads: 20 us by one thread, 6 by eight).
constexpr int JOIN = 256, FEW_PARTS = 8;
template <int DT, int DP, int ROWS, bool MANY_PARTS>
__global__ __launch_bounds__(JOIN) void k_join(Args A) {
    typedef typename type<DT>::t T;
    constexpr int COLS = DP / 4, GROUPS = MANY_PARTS ? JOIN / COLS : 1, AT_ONCE = JOIN / COLS / GROUPS, MOST = MANY_PARTS ? (int)MAX_PARTS : FEW_PARTS;
    __shared__ float of_parts[AT_ONCE * MOST][2];
    __shared__ v4f of_groups[MANY_PARTS ? JOIN : 1];
    const int heads = (int)A.cache.heads, head = (int)blockIdx.x % heads, tile = (int)blockIdx.x / heads;
    const int col = (int)threadIdx.x % COLS * 4, group = (int)threadIdx.x / COLS % GROUPS, own = (int)threadIdx.x / COLS / GROUPS;
    Tile t;
    if (!find_tile<ROWS>(A, tile, &t)) return;
    const i64 slot = ((i64)tile * heads + head) * A.splits;
    const int parts = parts_of(A, t.end), rows = min(ROWS, t.n * A.group - t.first);
    if (parts <= 1) return;                    // the only one is done
    for (int first = (int)blockIdx.y * AT_ONCE; first < rows; first += (int)gridDim.y * AT_ONCE) {
        for (int i = threadIdx.x; i < AT_ONCE * parts; i += JOIN) {
            const int r = first + i / parts, s = i % parts;
            if (r < rows) __builtin_memcpy(of_parts[i], A.most + ((slot + s) * ROWS + r) * 2, 8);
        }
        __syncthreads();
        const int r = first + own, row = t.first + r, tok = (int)((u32)row / (u32)A.group), g = row - tok * A.group;
        const bool there = r < rows && col < A.cache.dim;
        float total = 0;
        v4f x = {0, 0, 0, 0};
        if (there) {
            const float(*its)[2] = of_parts + own * parts, *part = A.part + (slot * ROWS + r) * DP + col;
            float top = -INFINITY;
            for (int s = 0; s < parts; ++s) top = fmaxf(top, its[s][0]);
            const float base = top == -INFINITY ? 0.0f : top;
            for (int s = 0; s < parts; ++s) total += __builtin_amdgcn_exp2f(its[s][0] - base) * its[s][1];
#pragma unroll 8
            for (int s = group; s < parts; s += GROUPS) x += __builtin_amdgcn_exp2f(its[s][0] - base) * *(const v4f *)(part + (i64)s * ROWS * DP);
        }
        if constexpr (MANY_PARTS) {
            of_groups[threadIdx.x] = x;
            __syncthreads();
            if (group == 0) {
#pragma unroll
                for (int k = 1; k < GROUPS; ++k) x += of_groups[threadIdx.x + k * COLS];
            }
        }
        if (there && group == 0) {
            const float per = total == 0.0f ? 0.0f : 1.0f / total;
            const v2u two = {pack<DT>(x.x * per, x.y * per), pack<DT>(x.z * per, x.w * per)};
            store_any((T *)A.out + ((i64)t.s0 + tok) * A.out_token + (head * A.group + g) * A.out_head + col, two);
        }
        __syncthreads();                       // before the next rows' parts
    }
}

// ---- forms --------------------------------------------------------------------------------------------------------
// Few rows of a sequence: four wavefronts with keys of their own.  Many: four wavefronts' rows share the keys.
template <int DT, bool I8, int DP>
struct Few : Form<DT, I8, DP, 1, 4, (DP > 128 ? 1 : 2)> {};
template <int DT, bool I8, int DP>
struct Many : Form<DT, I8, DP, 4, 1, (DP > 128 ? 1 : 2)> {};

enum { FEW, MANY };
struct Plan {
    int form, rows, dp, tiles, splits, per_split;
    size_t ws_bytes;
};
constexpr int CUS = 256;                       // of a whole card; on a part of one the choice of splits costs time, nothing else

Plan make_plan(int cache_dtype, i64 dim, i64 cache_heads, i64 n, i64 heads, i64 sequences, i64 longest) {
    Plan L = {};
    const i64 group = heads / cache_heads, rows = (n * group + sequences - 1) / sequences;           // of a sequence, on an average
    L.dp = dim <= 64 ? 64 : dim <= 128 ? 128 : 256;
    // A tile of 128 rows reads its keys once, but its wavefronts wait for each other: 64 sequences of 64 rows over 4096 entries take 239 us as two tiles of
    // 32, 308 as one of 64 whose wavefronts share the keys; 16 of 100 rows 91 us as four tiles, 82 as one of 128, but over 8-bit integers, of which
    // there are half the bytes to read, 87 and 92.
    L.form = rows <= (cache_dtype == VI_I8 ? 128 : 64) ? FEW : MANY;
    L.rows = L.form == FEW ? 32 : 128;
    const i64 tiles = n * group / L.rows + sequences, full = (n * group + L.rows - 1) / L.rows, busy = full > sequences ? full : sequences;
    L.tiles = (int)(tiles < MAX_BLOCKS ? tiles : MAX_BLOCKS);
    // The keys are cut into parts of one size where there are few tiles: two workgroups a CU, as many as there is room for (a sequence of 32768 entries,
    // 8 heads: 38 us, 41 with four a CU; 16 trees of 25 78 and 90, 96 with one a CU), or four where sequences alone make two, for their lengths differ (64 of 500 to 8192: 224 us, 237 uncut).  A
    // part has 128 keys at least, a round of a workgroup's wavefronts, and 512 where there are many.
    const i64 all = busy * cache_heads, wanted = (all < 2 * CUS ? 2 : 4) * CUS, parts = wanted / all, round = 128, least = all >= CUS ? 4 * round : round;
    i64 keys = parts > 1 ? (longest + parts - 1) / parts : longest;
    keys = keys < least ? least : keys;
    keys = longest > keys * MAX_PARTS ? (longest + MAX_PARTS - 1) / MAX_PARTS : keys;
    L.per_split = (int)((keys + round - 1) / round * round);
    L.splits = (int)(longest > L.per_split ? (longest + L.per_split - 1) / L.per_split : 1);
    if (L.splits > 1) L.ws_bytes = (size_t)(tiles * cache_heads * L.splits * L.rows) * (L.dp + 2) * 4 + vi::WS_SLACK;
    return L;
}

template <class F>
void launch(const Args &A, hipStream_t s) {
    const i64 heads = A.cache.heads;
    hipLaunchKernelGGL(k_attend<F>, dim3((unsigned)(heads * A.tiles * A.splits)), dim3(F::THREADS), 0, s, A);
    if (A.splits > 1) {
        const bool many = A.splits > FEW_PARTS;
        const i64 tiles = heads * A.tiles, rows = many ? 1 : JOIN / (F::DP / 4);
        const dim3 grid((unsigned)tiles, (unsigned)(tiles < 2 * CUS ? F::ROWS / rows : 1));
        if (many) hipLaunchKernelGGL((k_join<F::DT, F::DP, F::ROWS, true>), grid, dim3(JOIN), 0, s, A);
        else hipLaunchKernelGGL((k_join<F::DT, F::DP, F::ROWS, false>), grid, dim3(JOIN), 0, s, A);
    }
}
template <int DT, bool I8, int DP>
void launch_form(int form, const Args &A, hipStream_t s) {
    if (form == FEW) return launch<Few<DT, I8, DP>>(A, s);
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
           heads % cache_heads == 0 && heads <= 0xFFFF && n <= MAX_HEADS / heads && sequences > 0 && sequences <= 0xFFFFFF && longest >= 0;
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
    if (n < 0 || heads < 1 || heads > 0xFFFF || heads % cache->heads || n > MAX_HEADS / heads)
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
    A.heads = (int)heads, A.group = (int)(heads / cache->heads), A.tiles = L.tiles, A.splits = L.splits, A.per_split = L.per_split, A.clear = clear != 0, A.c = scale * 1.44269504f;
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
