// Products of 8-bit integers with a scale for each row of A (token) and of B (channel), and the gated block of two of them.
//
//     S_ij = sum_l a_il b_jl          out = S, S mod p, or (S_ij a_scale_i) b_scale_j + bias_j
//     gated: act((S_ij a_scale_i) g_scale_j) ((T_ij a_scale_i) u_scale_j), S and T of the same A with two B
//
// Both operands have their inner dimension along the rows, so a wavefront's operands of a matrix instruction are 16 contiguous bytes a
// lane.  Sums are exact: |S| <= 2^14 k fits 32 bits up to MAX_K.
//
// What bounds them, by rows of A: up to some 32 the weights' way from memory (1 x 4096 x 11008 11-12 us, 4 TB/s).  Hundreds of rows, where a
// CU has one small tile and a SIMD one wavefront, what that wavefront waits for: 1000 x 4096 x 4096 takes 23 us, 1.45 POP/s (as field elements
// 27); its wavefronts are at a wait or barrier for 51 % of their cycles, the matrix cores work in 43 %, LDS is read in 23 %, and 27 bytes a cycle
// come from the L2s of 64 that the path takes.  More rows, the matrix cores at the clock that the power limit leaves them (4096 x 4096 x 11008
// 177-188 us by the card, 2.0 POP/s; 8192 x 8192 x 8192 462-480, 2.3; gated 1000 x 4096 x 11008 97-106, 1.8).
#include <type_traits>

#include "int8_gemm.hpp"

namespace {

using namespace i8;

constexpr int MAX_K = 131071;

// Where unit `unit` of row `row` is in a stage, in units: those of a row are in another order by the row, so that the sixteen lanes that LDS
// serves at a time, one unit of as many neighbouring rows, meet all 64 banks.
template <int U>
__device__ __forceinline__ int order(int row) { return U == 4 ? (row >> 2) & 3 : (row >> 1) & 7; }

// Column c of a tile's 64 WN virtual columns -> its row of B behind the tile's first, or of the second B where *second: a wavefront's
// first half of the columns are the gate's, its other half the same channels' of the up projection, so that both sums of an output
// are in one lane.
template <int WN, bool GATED>
__device__ __forceinline__ i64 channel(int c, bool *second) {
    if (!GATED) return c;
    const int wc = c / (32 * WN), in = c % (32 * WN);
    *second = in >= 16 * WN;
    return wc * (16 * WN) + in % (16 * WN);
}

// Words between the rows of a wavefront's sums in LDS: sixteen lanes' 16 bytes in neighbouring rows meet different banks.
constexpr int pitch(int wn) { return 32 * wn + 4; }

// a wavefront's own LDS accesses are in order for all its lanes
__device__ __forceinline__ void meet_wave() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A wavefront's sums acc[j][i]: columns 32 j, rows 32 i.  The weights are the first operand of the matrix instruction, so register r of a
// lane is column 8 (r / 4) + 4 half + r % 4 of row lane % 32: four neighbouring columns in neighbouring registers.
//
// This way out goes through LDS, 32 rows at a time in the wavefront's own part (after a barrier), with any number of columns.
template <int WM, int WN, bool GATED>
__device__ __forceinline__ void put_ragged(const Job &J, int *buf, const v16i (&acc)[WN][WM], i64 row0, i64 col0, int slice, int lane) {
    constexpr int WIDE = GATED ? 16 * WN : 32 * WN, VECS = WIDE / VEC, PITCH = pitch(WN);
    const int half = lane >> 5;
#pragma unroll
    for (int i = 0; i < WM; ++i) {
#pragma unroll
        for (int j = 0; j < WN; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const v4i v = {acc[j][i][4 * g], acc[j][i][4 * g + 1], acc[j][i][4 * g + 2], acc[j][i][4 * g + 3]};
                *(v4i *)(buf + (lane & 31) * PITCH + 32 * j + 8 * g + 4 * half) = v;
            }
        meet_wave();
#pragma unroll 1
        for (int it = 0; it < 32 * VECS / 64; ++it) {
            const int p = it * 64 + lane, lrow = p / VECS, lcol = p % VECS * VEC;
            const i64 row = row0 + 32 * i + lrow, col = col0 + lcol;
            const int count = (int)min(J.n - col, (i64)VEC);
            if (row >= J.m || count <= 0) continue;
            int v[VEC], w[VEC];
            __builtin_memcpy(v, __builtin_assume_aligned(buf + lrow * PITCH + lcol, 16), sizeof(v));
            if (GATED) __builtin_memcpy(w, __builtin_assume_aligned(buf + lrow * PITCH + WIDE + lcol, 16), sizeof(w));
            if (J.slices == 1) {
                finish<GATED>(J, row, col, count, v, w);
            } else {
#pragma unroll
                for (int h = 0; h < (GATED ? 2 : 1); ++h) {
                    int *o = J.partial + (((i64)slice * (GATED ? 2 : 1) + h) * J.m + row) * J.n + col;
#pragma unroll
                    for (int e = 0; e < VEC; ++e)
                        if (e < count) o[e] = h ? w[e] : v[e];
                }
            }
        }
        meet_wave();
    }
}

// The lower lanes get the eight columns of group 2 p of their row, the upper ones those of 2 p + 1: w[0] and w[1] are a lane's own four
// columns of either group.
__device__ __forceinline__ void swap_halves(u32 &a, u32 &b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}

// A sum as it is needed, here: without it the compiler converts all of a wavefront's sums in front of the branches that ask for their
// type, and has to put them into scratch memory.
__device__ __forceinline__ int here(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// two values as the 16-bit type, the first in the lower half
template <int DT>
__device__ __forceinline__ u32 pack(float a, float b) {
    typedef float v2f __attribute__((ext_vector_type(2)));
    typedef typename type<DT>::t v2t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(u32, __builtin_convertvector((v2f{a, b}), v2t));
}

// a sum as a residue mod p = 2^64 - 2^32 + 1, in words: s, or 2^64 + s - (2^32 - 1) below zero
__device__ __forceinline__ int residue_low(int s) { return s < 0 ? s + 1 : s; }
__device__ __forceinline__ int residue_high(int s) { return s < 0 && s + 1 != 0 ? -2 : s < 0 ? -1 : 0; }

// The way out for tiles whose columns all exist: 16 columns at a time (half a tile of the matrix instruction; the next ones' scales are on
// their way meanwhile), 32 rows through the wavefront's part of LDS as they go out, so that a store writes whole lines: 8192 x 1024 x 8192
// 103 us, 120 with 32 bytes of each of 32 rows in a store straight from the registers.
template <int DT, int WM, int WN, bool GATED>
__device__ __forceinline__ void put_rows(const Job &J, char *buf, const v16i (&acc)[WN][WM], i64 row0, i64 col0, int lane) {
    constexpr int Q = GATED ? WN : 2 * WN, SIZE = size_of(DT), ROW = Q * 16 * SIZE, PITCH = ROW + 16, UNITS = ROW / 16;     // bytes
    const int half = lane >> 5;
    float as[WM], bs[2][VEC], us[2][VEC];
    auto scales = [&](int q) {
        if (!is_float(DT)) return;
        auto some = [&](float (&to)[VEC], const float *from) {
#pragma unroll
            for (int g = 0; g < 2; ++g) __builtin_memcpy(to + 4 * g, from + col0 + 16 * q + 8 * g + 4 * half, 16);
        };
        some(bs[q & 1], J.b_scale);
        if (GATED) some(us[q & 1], J.b2_scale);
        else if (J.bias) some(us[q & 1], J.bias);
    };
    if (is_float(DT))
#pragma unroll
        for (int i = 0; i < WM; ++i) as[i] = J.a_scale[min(row0 + 32 * i + (lane & 31), J.m - 1)];
#pragma unroll
    for (int i = 0; i < WM; ++i) {
        char *mine = buf + (lane & 31) * PITCH;
        scales(0);
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            if (q + 1 < Q) scales(q + 1);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (!is_float(DT)) {
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    int s[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[e] = here(acc[q / 2][i][8 * (q % 2) + 4 * g + e]);
                    char *to = mine + (16 * q + 8 * g + 4 * half) * SIZE;
                    if constexpr (DT == VI_I32) {
                        *(v4i *)to = v4i{s[0], s[1], s[2], s[3]};
                    } else {
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            *(v4i *)(to + 16 * e) = v4i{residue_low(s[2 * e]), residue_high(s[2 * e]), residue_low(s[2 * e + 1]), residue_high(s[2 * e + 1])};
                    }
                }
                continue;
            }
            const float(&b)[VEC] = bs[q & 1], (&u)[VEC] = us[q & 1];
            float v[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = (float)here(acc[q / 2][i][8 * (q % 2) + e]) * as[i] * b[e];
            if constexpr (GATED) {
                activate(v, J.act);
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[e] *= (float)here(acc[(WN + q) / 2][i][8 * ((WN + q) % 2) + e]) * as[i] * u[e];
            } else if (J.bias) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[e] += u[e];
            }
            if constexpr (DT == VI_F32) {
#pragma unroll
                for (int g = 0; g < 2; ++g) *(v4i *)(mine + 64 * q + 32 * g + 16 * half) = __builtin_bit_cast(v4i, *(const float (*)[4])(v + 4 * g));
            } else if constexpr (is_float(DT)) {
                u32 w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = pack<DT>(v[2 * e], v[2 * e + 1]);
                swap_halves(w[0], w[2]);
                swap_halves(w[1], w[3]);
                *(v4i *)(mine + 32 * q + 16 * half) = v4i{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
            }
        }
        meet_wave();
#pragma unroll
        for (int p = 0; p < 32 * UNITS / 64; ++p) {
            const int at = p * 64 + lane, row = at / UNITS, unit = at % UNITS;
            const v4i w = *(const v4i *)(buf + row * PITCH + unit * 16);
            if (row0 + 32 * i + row < J.m) store_any((char *)J.out + ((row0 + 32 * i + row) * J.ldo + col0) * (i64)SIZE + unit * 16, w);
        }
        meet_wave();
    }
}

// The sums of a slice to its part of the scratch; those of the second weights `second` behind the first's.
template <int WM, int WN, bool GATED>
__device__ __forceinline__ void put_sums(const v16i (&acc)[WN][WM], int *out, i64 ld, i64 m, i64 second, i64 row0, i64 col0, int lane) {
    const int half = lane >> 5;
#pragma unroll
    for (int q = 0; q < 2 * WN; ++q)
#pragma unroll
        for (int i = 0; i < WM; ++i) {
            const i64 row = row0 + 32 * i + (lane & 31);
            const bool up = GATED && q >= WN;
            if (row < m) {
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const int r = 8 * (q % 2) + 4 * g;
                    const v4i v = {acc[q / 2][i][r], acc[q / 2][i][r + 1], acc[q / 2][i][r + 2], acc[q / 2][i][r + 3]};
                    store_any(out + row * ld + col0 + 16 * (up ? q - WN : q) + 8 * g + 4 * half + (up ? second : 0), v);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
}

template <int WM, int WN, bool GATED>
__device__ __forceinline__ void put(const Job &J, int *buf, const v16i (&acc)[WN][WM], int tm, int tn, int slice, int wave, int lane) {
    constexpr int WIDE = GATED ? 16 * WN : 32 * WN;
    const i64 row0 = (i64)tm * (64 * WM) + (wave >> 1) * (32 * WM), col0 = (i64)tn * (2 * WIDE) + (wave & 1) * WIDE;
    if (col0 + WIDE > J.n) {
        put_ragged<WM, WN, GATED>(J, buf, acc, row0, col0, slice, lane);
    } else if (J.slices > 1) {
        put_sums<WM, WN, GATED>(acc, J.partial + (i64)slice * (GATED ? 2 : 1) * J.m * J.n, J.n, J.m, J.m * J.n, row0, col0, lane);
    } else if (!GATED && J.dtype == VI_I32) {
        put_rows<VI_I32, WM, WN, false>(J, (char *)buf, acc, row0, col0, lane);
    } else if (!GATED && J.dtype == VI_FIELD) {
        put_rows<VI_FIELD, WM, WN, false>(J, (char *)buf, acc, row0, col0, lane);
    } else if (J.dtype == VI_BF16) {
        put_rows<VI_BF16, WM, WN, GATED>(J, (char *)buf, acc, row0, col0, lane);
    } else if (J.dtype == VI_F16) {
        put_rows<VI_F16, WM, WN, GATED>(J, (char *)buf, acc, row0, col0, lane);
    } else {
        put_rows<VI_F32, WM, WN, GATED>(J, (char *)buf, acc, row0, col0, lane);
    }
}

// Which tile a workgroup takes.  Workgroups go to the eight XCDs in turn: those of one XCD (id % 8) take neighbouring tiles, GROUP
// tiles down and as many across as there are, so that what they read at a time is in its L2.
constexpr int GROUP = 8;
__device__ __forceinline__ void place(const Job &J, int id, int *tm, int *tn) {
    const int total = J.mt * J.nt, xcd = id & 7, each = total >> 3, more = total & 7;
    id = xcd * each + min(xcd, more) + (id >> 3);
    const int strip = id / (GROUP * J.nt), first = strip * GROUP, rows = min(GROUP, J.mt - first), in = id - first * J.nt;
    *tm = first + in % rows;
    *tn = in / rows;
}

// ---- tiles --------------------------------------------------------------------------------------------------------
// 64 lanes' 16 bytes at base + off into 1 KiB of LDS, without a register in between, where fetch_from_here() says and 4 KiB on for each
// call; base is the same for the wavefront.  As instructions of their own the compiler does not wait for them before the next LDS read, as
// it does for its builtin: the waits are wait_and_meet's.  The place is in M0, a register that the compiler keeps nothing in: it sets it
// in front of instructions that read it, of which it makes none here.
// Wait states, which inside an asm block nothing inserts: one between a write of M0 and the load, five between a vector instruction's write
// of a scalar register (readfirstlane, where the compiler has kept the base in vector registers) and a load that reads it.
__device__ __forceinline__ void fetch_from_here(u32 at) { asm volatile("s_mov_b32 m0, %0" : : "s"(at) : "memory"); }
__device__ __forceinline__ void fetch_to_lds(const signed char *base, u32 off) {
    const u64 b = (u64)__builtin_amdgcn_readfirstlane((u32)((u64)base >> 32)) << 32 | (u32)__builtin_amdgcn_readfirstlane((u32)(u64)base);
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1\n\ts_add_u32 m0, m0, 0x1000" : : "v"(off), "s"(b) : "memory", "scc");
}
// all but the wavefront's last `n` loads have arrived and its LDS accesses are done, then the workgroup's barrier
template <int N>
__device__ __forceinline__ void wait_and_meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory");
}

// the same with all the loads, where there are any; the compiler waits for those to registers
template <bool LOADS>
__device__ __forceinline__ void meet() {
    if constexpr (LOADS) wait_and_meet<0>();
    else asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
}

template <int WM, int WN, int U, int ST>
union alignas(16) Lds {
    char in[ST * 64 * (WM + WN) * U * 16];
    int out[4][2 * 32 * pitch(WN)];            // 32 rows of a wavefront's sums or outputs, which may have 64 bits
};

// A tile of 64 WM rows and 64 WN (virtual) columns by four wavefronts in a square, in steps of U units of 16 inner indices.  ST stages of LDS,
// PER_CU workgroups to a CU.  The operands of the next 32 inner indices are read from LDS, and loads requested, between the products
// of these, so that the matrix cores have work throughout: they stop only where the workgroup meets, once a step.  The ragged end of
// the rows goes first, through registers.
// Whole lines: a step of four units is half a line of each row, and 64 KiB of lines do not stay in a CU's 32 KiB cache until the next step
// comes for the other half, so that the L2s would be asked for twice the operands (8192 x 8192 x 8192 in tiles of 256 x 128: 585 us, 509 in
// steps of eight units).  The large tiles, of whose steps of eight units LDS holds two, load two of four at a time (PAIR): five stages, two
// steps requested together, half a line behind the other, in every other step.
// DIRECT: operands at 16-byte boundaries go straight into LDS, ST - 1 steps ahead.  Others go through registers: loads of one step are
// under way while the next stage but one is written.
template <int WM, int WN, int U, int ST, int PER_CU, bool GATED, bool DIRECT>
__global__ __launch_bounds__(BLOCK, PER_CU) void k_tile(Job J) {
    constexpr int TM = 64 * WM, STEP = 16 * U, AHEAD = DIRECT ? ST - 1 : 2, N = WM * WN, T = U / 2;
    constexpr bool PAIR = DIRECT && U == 4;
    static_assert(!PAIR || ST == 5, "");
    constexpr int CHUNK_ROWS = 64 / U, NL = (WM + WN) * U / 4, A_LOADS = WM * U / 4, READS = WM + WN;
    constexpr u32 STAGE = 64 * (WM + WN) * U * 16;
    static_assert(DIRECT || ST == 3, "");
    __shared__ Lds<WM, WN, U, ST> lds;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int total = J.mt * J.nt;
    const int slice = __builtin_amdgcn_readfirstlane(blockIdx.x / total);
    int tm, tn;
    place(J, blockIdx.x % total, &tm, &tn);
    tm = __builtin_amdgcn_readfirstlane(tm);   // the divisions are vector instructions: what follows from them stays scalar this way
    tn = __builtin_amdgcn_readfirstlane(tn);
    const int s0 = slice * J.steps_per_slice, s1 = min(s0 + J.steps_per_slice, J.steps), steps = s1 - s0;

    // Load j of the wavefront is chunk 4 j + wave of a stage, 1 KiB: CHUNK_ROWS rows of A or B.  Rows that do not exist are the last
    // one again.  DIRECT: rows less than 2^23 apart, a tile's distances fit 32 bits.
    typedef typename std::conditional<DIRECT, u32, i64>::type Off;
    Off off[NL];
    bool other[NL];                            // of the second B
    const int in_row = lane / U, unit = ((lane % U) ^ order<U>(wave * CHUNK_ROWS + in_row)) * 16;
    static_assert(U == 4 || CHUNK_ROWS * 4 % 16 == 0, "");
    const i64 a_first = (i64)tm * TM, b_first = (i64)tn * (GATED ? 32 : 64) * WN;
    const signed char *pa = J.a + a_first * J.lda, *pb = J.b + b_first * J.ldb, *pb2 = GATED ? J.b2 + b_first * J.ldb2 : nullptr;
#pragma unroll
    for (int j = 0; j < NL; ++j) {
        other[j] = false;
        if (j < A_LOADS) {
            const i64 row = min((i64)((j * 4 + wave) * CHUNK_ROWS + in_row), J.m - 1 - a_first);
            off[j] = (Off)row * (Off)J.lda + unit;
        } else {
            const int c = ((j - A_LOADS) * 4 + wave) * CHUNK_ROWS;
            const i64 row = min(channel<WN, GATED>(c, &other[j]) + in_row, J.n - 1 - b_first);
            off[j] = (Off)row * (Off)(other[j] ? J.ldb2 : J.ldb) + unit;
        }
    }
    // position 0 is the ragged end, where this slice has it; position p else the step s0 + p - ragged
    const int ragged = s1 == J.steps && J.k % STEP ? 1 : 0;
    pa += (i64)s0 * STEP;
    pb += (i64)s0 * STEP;
    if (GATED) pb2 += (i64)s0 * STEP;
    auto source = [&](int j) { return j < A_LOADS ? pa : other[j] ? pb2 : pb; };
    const u32 lds0 = (u32)(uintptr_t)(__attribute__((address_space(3))) char *)lds.in;
    u32 put_at = ragged * STAGE;               // the stage that the next step is fetched to
    v4i in[NL];                                // !DIRECT: that step, on its way
    auto load = [&](int j) { in[j] = load_any<v4i>(source(j) + off[j]); };
    auto store = [&](int j) { *(v4i *)(lds.in + put_at + (j * 4 + wave) * 1024 + lane * 16) = in[j]; };
    auto advance = [&]() {
        pa += STEP;
        pb += STEP;
        if (GATED) pb2 += STEP;
    };
    auto next_stage = [](u32 s) { return s == (ST - 1) * STAGE ? 0 : s + STAGE; };
    // PAIR: of the next two steps at once
    auto fetch_two = [&](int j) {
        const u32 chunk = lds0 + wave * 1024 + j * 4096;
        fetch_from_here(chunk + put_at);
        fetch_to_lds(source(j), off[j]);
        fetch_from_here(chunk + next_stage(put_at));
        fetch_to_lds(source(j) + STEP, off[j]);
        if (j == NL - 1) {
            advance();
            advance();
            put_at = next_stage(next_stage(put_at));
        }
    };
    auto fetch = [&](int j) {
        if constexpr (DIRECT) {
            if (j == 0) fetch_from_here(lds0 + put_at + wave * 1024);
            fetch_to_lds(source(j), off[j]);
        } else {
            store(j);
            load(j);
        }
        if (j == NL - 1) {
            advance();
            put_at = next_stage(put_at);
        }
    };

    v16i acc[WN][WM];
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int j = 0; j < WN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[j][i][r] = 0;
    const int half = lane >> 5, row0 = (wave >> 1) * (32 * WM) + (lane & 31), col0 = TM + (wave & 1) * (32 * WN) + (lane & 31);
    u32 x_at[T], y_at[T];
#pragma unroll
    for (int t = 0; t < T; ++t) {
        x_at[t] = (row0 * U + ((2 * t + half) ^ order<U>(row0))) * 16;
        y_at[t] = (col0 * U + ((2 * t + half) ^ order<U>(col0))) * 16;
    }
    v4i x[2][WM], y[2][WN];
    // operand q of the 32 inner indices t of the stage at byte `from`, in the order in which the products take them
    auto read = [&](u32 from, int t, int q) {
        const char *xs = lds.in + from + x_at[t], *ys = lds.in + from + y_at[t];
        constexpr int APART = 32 * U * 16;
        if (q == 0) x[t & 1][0] = *(const v4i *)xs;
        else if (q <= WN) y[t & 1][q - 1] = *(const v4i *)(ys + APART * (q - 1));
        else x[t & 1][q - WN] = *(const v4i *)(xs + APART * (q - WN));
    };
    // the products of part t, `between(c)` behind the c-th
    auto multiply = [&](int t, auto between) {
#pragma unroll
        for (int c = 0; c < N; ++c) {
            const int i = c / WN, j = c % WN;
            acc[j][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(y[t & 1][j], x[t & 1][i], acc[j][i], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
            between(c);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    u32 take = 0;                              // the stage that is multiplied
    // All parts of a step but the last, the next part's reads and the loads of a step to come (LOADS) among them; then, behind `wait`, the
    // last with the reads of the next step's first.  PAIR: half of two steps' loads in each of the two parts.
    constexpr int FIRST = PAIR ? NL / 2 : NL;
    auto step = [&](auto loads, auto last, auto wait) {
        constexpr bool LOADS = decltype(loads)::value, LAST = decltype(last)::value;
#pragma unroll
        for (int t = 0; t < T - 1; ++t)
            multiply(t, [&](int c) {
                const int from = t * FIRST / (T - 1), ops = READS + (LOADS ? (t + 1) * FIRST / (T - 1) - from : 0);
#pragma unroll
                for (int q = c * ops / N; q < (c + 1) * ops / N; ++q) {
                    if (q < READS) read(take, t + 1, q);
                    else if constexpr (PAIR) fetch_two(from + q - READS);
                    else fetch(from + q - READS);
                }
            });
        wait();
        take = next_stage(take);
        multiply(T - 1, [&](int c) {
            if constexpr (PAIR && LOADS) {
                constexpr int OPS = READS + NL - FIRST;
#pragma unroll
                for (int q = c * OPS / N; q < (c + 1) * OPS / N; ++q) {
                    if (q < READS) read(take, 0, q);
                    else fetch_two(FIRST + q - READS);
                }
            } else if constexpr (!LAST) {
                constexpr int EACH = (READS + N - 1) / N;
#pragma unroll
                for (int q = c * EACH; q < (c + 1) * EACH && q < READS; ++q) read(take, 0, q);
            }
        });
    };
    const auto yes = std::true_type();
    const auto no = std::false_type();

    if (steps > 0) {
        v4i end[NL];
        if (ragged) {
            const i64 at = (i64)(J.steps - 1 - s0) * STEP;
#pragma unroll
            for (int j = 0; j < NL; ++j) end[j] = load_end(source(j) + at + off[j], J.k - (i64)(J.steps - 1) * STEP - unit, J.k);
        }
        // behind the other loads' requests
        auto store_end = [&]() {
            if (ragged) {
#pragma unroll
                for (int j = 0; j < NL; ++j) *(v4i *)(lds.in + (j * 4 + wave) * 1024 + lane * 16) = end[j];
            }
        };
        // how far the loads go in front of the loop, and the first position there
        if constexpr (PAIR) {
            // two steps, then two more, or one: positions from `ragged` on
            const int pairs = ragged ? 1 : 2, left = steps - ragged;
            for (int i = 0; i < pairs && 2 * i < left; ++i) {
                if (2 * i + 1 < left) {
#pragma unroll
                    for (int j = 0; j < NL; ++j) fetch_two(j);
                } else {
#pragma unroll
                    for (int j = 0; j < NL; ++j) fetch(j);
                }
            }
            store_end();
            if (left >= 2 * pairs) wait_and_meet<2 * NL>();            // all but the last pair
            else wait_and_meet<0>();
        } else if constexpr (DIRECT) {
#pragma unroll
            for (int p = 0; p < AHEAD; ++p)
                if (p < steps && p >= ragged) {
#pragma unroll
                    for (int j = 0; j < NL; ++j) fetch(j);
                }
            store_end();
            if (steps >= AHEAD) wait_and_meet<(AHEAD - 1) * NL>();
            else wait_and_meet<0>();
        } else {
            if (steps > ragged) {
#pragma unroll
                for (int j = 0; j < NL; ++j) load(j);
                advance();
#pragma unroll
                for (int p = 0; p < AHEAD; ++p)
                    if (p < steps && p >= ragged) {
                        if (p + 1 < steps) {
#pragma unroll
                            for (int j = 0; j < NL; ++j) fetch(j);
                        } else {
#pragma unroll
                            for (int j = 0; j < NL; ++j) store(j);
                        }
                    }
            }
            store_end();
            meet<false>();
        }
#pragma unroll
        for (int q = 0; q < READS; ++q) read(take, 0, q);
        int p = 0;
        if constexpr (PAIR) {
            // At a step with loads the three positions from its own on are in LDS or on their way, and the next two are requested; those
            // of the step before the last one with loads have arrived behind it.
            if (!ragged && steps > 1) {
                step(no, no, [] { wait_and_meet<2 * NL>(); });
                p = 1;
            }
            while (p + 4 < steps) {
                step(yes, no, [] { wait_and_meet<2 * FIRST>(); });
                step(no, no, [] { wait_and_meet<2 * NL>(); });
                p += 2;
            }
            if (p + 3 < steps) {
#pragma unroll
                for (int j = 0; j < NL; ++j) fetch(j);
            }
        } else {
            // the last load of !DIRECT would be one step too many
            for (; p + AHEAD + (DIRECT ? 0 : 1) < steps; ++p)
                step(yes, no, [] {
                    if constexpr (DIRECT) wait_and_meet<(AHEAD - 1) * NL>();
                    else meet<false>();
                });
            if constexpr (!DIRECT) {
                if (p + AHEAD < steps) {
#pragma unroll
                    for (int j = 0; j < NL; ++j) store(j);
                }
            }
        }
        for (; p + 1 < steps; ++p) step(no, no, [] { meet<DIRECT>(); });
        step(no, yes, [] {});
        __syncthreads();
    }
    put<WM, WN, GATED>(J, lds.out[wave], acc, tm, tn, slice, wave, lane);
}

// ---- rows at any address, to 16-byte boundaries -------------------------------------------------------------------
// Up to three matrices in one launch, 16 bytes a thread, zero behind the last of a row: whole lines, and whole steps of any tile, so that no
// row has a ragged end any more.
constexpr i64 LINE = 128;
i64 whole_lines(i64 k) { return (k + LINE - 1) / LINE * LINE; }

struct Pack {
    const signed char *from[3];
    v4i *to[3];
    i64 ld[3], rows[3];                        // rows: up to and with this matrix
    i64 k, units;                              // units of a row
};

__global__ __launch_bounds__(BLOCK) void k_pack(Pack P) {
    const i64 total = P.rows[2] * P.units;
    for (i64 p = (i64)blockIdx.x * BLOCK + threadIdx.x; p < total; p += (i64)gridDim.x * BLOCK) {
        i64 row = p / P.units;
        const i64 at = p - row * P.units;
        const int which = row < P.rows[0] ? 0 : row < P.rows[1] ? 1 : 2;
        if (which) row -= P.rows[which - 1];
        P.to[which][row * P.units + at] = load_end(P.from[which] + row * P.ld[which] + at * 16, P.k - at * 16, P.k);
    }
}

// ---- few rows -----------------------------------------------------------------------------------------------------
// Up to 16 MT rows: the weights are read once and hardly used, so they go from memory to the matrix instruction without LDS.  A workgroup
// takes 16 channels (of both weights), its eight wavefronts parts of the inner dimension: a lane has channel lane % 16, 16 inner indices of
// each 64 by lane / 16, FEW_BLOCKS loads of either operand under way at once.  The parts meet in LDS.
constexpr int FEW_BLOCKS = 8, FEW_WAVES = 8;

template <int MT, bool GATED>
__global__ __launch_bounds__(64 * FEW_WAVES) void k_few(Job J) {
    constexpr int W = FEW_WAVES;
    constexpr int NT = GATED ? 2 : 1;
    __shared__ int parts[W][NT * MT * 256];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const i64 first = (i64)blockIdx.x * 16, ch = min(first + (lane & 15), J.n - 1);
    const signed char *w[NT], *x[MT];
    w[0] = J.b + ch * J.ldb + (lane >> 4) * 16;
    if (GATED) w[NT - 1] = J.b2 + ch * J.ldb2 + (lane >> 4) * 16;
#pragma unroll
    for (int i = 0; i < MT; ++i) x[i] = J.a + min((i64)(16 * i + (lane & 15)), J.m - 1) * J.lda + (lane >> 4) * 16;
    v4i acc[NT][MT];
#pragma unroll
    for (int h = 0; h < NT; ++h)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[h][i] = v4i{0, 0, 0, 0};
    const int blocks = (int)(J.k / 64);
    int b = (int)((i64)blocks * wave / W);
    const int end = (int)((i64)blocks * (wave + 1) / W);
    auto some = [&](auto count) {
        constexpr int C = decltype(count)::value;
        v4i wv[C][NT], xv[C][MT];
#pragma unroll
        for (int u = 0; u < C; ++u) {
#pragma unroll
            for (int h = 0; h < NT; ++h) wv[u][h] = load_any<v4i>(w[h] + (i64)(b + u) * 64);
#pragma unroll
            for (int i = 0; i < MT; ++i) xv[u][i] = load_any<v4i>(x[i] + (i64)(b + u) * 64);
        }
#pragma unroll
        for (int u = 0; u < C; ++u)
#pragma unroll
            for (int h = 0; h < NT; ++h)
#pragma unroll
                for (int i = 0; i < MT; ++i) acc[h][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[u][h], xv[u][i], acc[h][i], 0, 0, 0);
        b += C;
    };
    while (b + FEW_BLOCKS <= end) some(std::integral_constant<int, FEW_BLOCKS>());
    if (b + 4 <= end) some(std::integral_constant<int, 4>());
    if (b + 2 <= end) some(std::integral_constant<int, 2>());
    if (b + 1 <= end) some(std::integral_constant<int, 1>());
    if (wave == W - 1 && J.k % 64) {
        const i64 at = (i64)blocks * 64, left = J.k - at - (lane >> 4) * 16;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const v4i xv = load_end(x[i] + at, left, J.k);
#pragma unroll
            for (int h = 0; h < NT; ++h) acc[h][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(load_end(w[h] + at, left, J.k), xv, acc[h][i], 0, 0, 0);
        }
    }
    // register r of a lane is channel 4 (lane / 16) + r of row lane % 16
#pragma unroll
    for (int h = 0; h < NT; ++h)
#pragma unroll
        for (int i = 0; i < MT; ++i) *(v4i *)&parts[wave][(h * MT + i) * 256 + (lane & 15) * 16 + (lane >> 4) * 4] = acc[h][i];
    __syncthreads();
    for (int e = threadIdx.x; e < MT * 256; e += 64 * W) {
        const i64 row = e / 16, col = first + e % 16;
        if (row >= J.m || col >= J.n) continue;
        int s = 0, t = 0;
#pragma unroll
        for (int v = 0; v < W; ++v) {
            s += parts[v][e];
            if (GATED) t += parts[v][MT * 256 + e];
        }
        finish_one<GATED>(J, row, col, s, t);
    }
}

// the sums of the slices, finished
template <bool GATED>
__global__ __launch_bounds__(BLOCK) void k_join(Job J) {
    const i64 per_row = (J.n + VEC - 1) / VEC, total = per_row * J.m, mn = J.m * J.n;
    for (i64 p = (i64)blockIdx.x * BLOCK + threadIdx.x; p < total; p += (i64)gridDim.x * BLOCK) {
        const i64 row = p / per_row, col = (p - row * per_row) * VEC;
        const int count = (int)min(J.n - col, (i64)VEC);
        int v[VEC] = {0}, w[VEC] = {0};
        const int *s = J.partial + row * J.n + col;
        if (count == VEC) {
#pragma unroll 4
            for (int q = 0; q < J.slices; ++q)
#pragma unroll
                for (int h = 0; h < (GATED ? 2 : 1); ++h, s += mn) {
                    int part[VEC];
                    __builtin_memcpy(part, s, sizeof(part));
#pragma unroll
                    for (int e = 0; e < VEC; ++e) (h ? w : v)[e] += part[e];
                }
        } else {
            for (int q = 0; q < J.slices; ++q)
#pragma unroll
                for (int h = 0; h < (GATED ? 2 : 1); ++h, s += mn)
#pragma unroll
                    for (int e = 0; e < VEC; ++e)
                        if (e < count) (h ? w : v)[e] += s[e];
        }
        finish<GATED>(J, row, col, count, v, w);
    }
}

// What a call is done with: the cheapest of these by their times in us, measured on this chip.
//
// Tiles, in units of 64 rows and 64 (virtual) columns: a step of one workgroup alone on its CU and of two that share it (0: there is
// room for one), all CUs busy; what a tile takes beside its steps (first loads, scaling, stores), and what of that shows where two share a
// CU; a step with operands through registers, and of two such.  Larger tiles read less a product (a CU's path to LDS takes 64 bytes a
// cycle, which 128 x 128 tiles would use up) and waste more where the last round of tiles is not full.
struct Tile {
    int wm, wn, units;
    double alone, shared, rest, between, staged, staged_shared;
};
constexpr Tile TILES[] = {{4, 4, 4, 0.85, 0, 7, 0, 1.45, 0},          // 8192 x 8192 x 8192 462 us; 256 x 192 tiles 524, 256 x 128 494, 128 x 128 588
                          {4, 3, 4, 0.6, 0, 9, 0, 1.2, 0},            // 1000 x 4096 x 11008 58 us; 256 x 256: 58, 256 x 128: 65, 128 x 128: 74
                          {4, 2, 8, 0.9, 0, 6.5, 0, 1.5, 0},          // 2000 x 4096 x 4096 37 us; 256 x 256: 51, 128 x 128: 41; gated 1000 x 4096 x 11008 103, 256 x 192: 106
                          {2, 2, 8, 0.48, 1.0, 4.5, 1.3, 1.2, 0},     // 1000 x 4096 x 4096 23 us; 256 x 128: 26, 64 x 128: 24
                          {1, 2, 8, 0.27, 0.62, 3, 0.5, 0.75, 1.25}};  // 128 x 4096 x 4096 12 us; 128 x 128: 16
constexpr int N_TILES = sizeof(TILES) / sizeof(TILES[0]), CUS = 256;                    // of a whole card; on a part of one the choices cost time, nothing else
constexpr int FEW = N_TILES;                   // k_few, up to FEW_ROWS rows
constexpr i64 FEW_ROWS = 32;
constexpr i64 MAX_GROUPS = (1 << 24) - 1;     // a launch has less than 2^32 threads: of 256, and half as many workgroups of 512

struct Plan {
    int tile, slices, steps_per_slice, steps, mt, nt;
    bool pack;
    size_t pack_bytes, ws_bytes;
};

// aligned: all operands' rows at 16-byte boundaries; may_pack: others may be copied
Plan make_plan(i64 m, i64 k, i64 n, bool gated, bool aligned, bool may_pack) {
    const double two = gated ? 2 : 1, weights = two * (double)n * k;
    Plan best = {};
    double least = 1e30;
    if (m <= FEW_ROWS && (n + 15) / 16 <= MAX_GROUPS / 2) {
        // weights from memory, rows of A once for each 16 channels from the L2s, and a wavefront's blocks of loads one after the other: 1 x 4096 x
        // 11008 12.0 us (64 x 128 tiles in slices 14.6), 16 rows 16.6 (15.7), 32 rows of 4096 x 4096 8.3 (10.2); gated 1 x 12288 x 1280
        // unaligned 34 (13.5 in eight slices)
        const double blocks = k / 64.0 / FEW_WAVES / FEW_BLOCKS;
        least = weights / (aligned ? 5.0e6 : 3.9e6) + (double)n * k * m / 16 / (m > 16 ? 7.5e6 : 9.5e6) + blocks * (aligned ? 1 : 5) * (gated ? 1.5 : 1);
        best.tile = FEW;
        best.slices = 1;
    }
    // copying unaligned operands: two passes over them and a launch
    const double pack_cost = aligned ? 0 : 4 + 2 * ((double)m * k + weights) / 4e6;
    for (int t = 0; t < N_TILES; ++t) {
        const Tile &T = TILES[t];
        const i64 rows = 64 * T.wm, cols = (gated ? 32 : 64) * T.wn, mt = (m + rows - 1) / rows, nt = (n + cols - 1) / cols, per_step = 16 * T.units;
        const int steps = (int)((k + per_step - 1) / per_step);
        for (int slices = 1; slices <= 16 && (slices == 1 || (steps / slices >= 4 && (double)mt * nt * slices <= 4 * CUS)); slices *= 2) {
            int each = (steps + slices - 1) / slices;
            if (T.units == 4) each += each & 1;         // whole lines
            const int used = each ? (steps + each - 1) / each : 1;
            const double groups = (double)mt * nt * used;
            if (groups > MAX_GROUPS) continue;
            const double join = used > 1 ? 4.5 + (double)used * m * n * two * 8 / 3.5e6 : 0;
            for (int pack = 0; pack < (may_pack && !aligned ? 2 : 1); ++pack) {
                const bool staged = !aligned && !pack;
                // rounds of all CUs, with as many workgroups as share one, then a last that may leave them alone
                const double alone = staged ? T.staged : T.alone, two_share = staged ? T.staged_shared : T.shared, rest = T.rest * (gated ? 1.5 : 1);
                const int share = two_share > 0 ? 2 : 1;
                const double full = each * (share == 2 ? two_share : alone), rounds = (double)(i64)(groups / (CUS * share)), left = groups - rounds * CUS * share;
                const double cost = join + (pack ? pack_cost : 0) + rounds * (full + (share == 2 ? T.between : rest)) +
                                    (left > CUS ? full + rest : left > 0 ? each * alone + rest : share == 2 ? rest : 0);
                if (cost < least) {
                    least = cost;
                    best = {t, used, each, steps, (int)mt, (int)nt, pack != 0, 0, 0};
                }
            }
        }
    }
    if (best.pack) best.pack_bytes = (size_t)whole_lines(k) * (m + (gated ? 2 : 1) * n);
    best.ws_bytes = best.pack_bytes + (best.slices > 1 ? (size_t)4 * best.slices * (gated ? 2 : 1) * m * n : 0);
    if (best.ws_bytes) best.ws_bytes += vi::WS_SLACK;
    return best;
}

// for operands wherever they are; may_pack: with copies of those that are not aligned
size_t workspace_bytes(i64 m, i64 k, i64 n, bool gated, bool may_pack) {
    if (m <= 0 || k < 0 || n <= 0 || k > MAX_K) return 0;
    const size_t a = make_plan(m, k, n, gated, true, false).ws_bytes, b = make_plan(m, k, n, gated, false, false).ws_bytes;
    const size_t c = may_pack ? make_plan(m, k, n, gated, false, true).ws_bytes : 0;
    return a > b ? (a > c ? a : c) : (b > c ? b : c);
}

bool aligned_rows(const void *p, i64 ld) { return ((uintptr_t)p & 15) == 0 && (ld & 15) == 0 && ld < (i64)1 << 23; }

// what is the same to check of both entries
int check(const char *who, const Job &J, bool gated) {
    if (J.m < 0 || J.k < 0 || J.n < 0) return vi::fail(VI_EINVAL, "%s: %lld x %lld x %lld", who, (long long)J.m, (long long)J.k, (long long)J.n);
    if (J.k > MAX_K) return vi::fail(VI_EINVAL, "%s: an inner dimension of %lld, sums of more than %d do not fit 32 bits", who, (long long)J.k, MAX_K);
    if (J.lda < J.k || J.ldb < J.k || (gated && J.ldb2 < J.k) || J.ldo < J.n)
        return vi::fail(VI_EINVAL, "%s: rows overlap (%lld, %lld, %lld and %lld apart)", who, (long long)J.lda, (long long)J.ldb, (long long)J.ldb2, (long long)J.ldo);
    if (J.m == 0 || J.n == 0) return VI_OK;
    if (J.m > (i64)1 << 31 || J.n > (i64)1 << 31) return vi::fail(VI_EINVAL, "%s: %lld x %lld outputs", who, (long long)J.m, (long long)J.n);
    if (!J.out || (J.k && (!J.a || !J.b || (gated && !J.b2)))) return vi::fail(VI_EINVAL, "%s: null pointer", who);
    if (is_float(J.dtype) && (!J.a_scale || !J.b_scale || (gated && !J.b2_scale))) return vi::fail(VI_EINVAL, "%s: scales missing", who);
    return VI_OK;
}

template <bool GATED, bool DIRECT>
void launch_tile(const Plan &L, const Job &J, hipStream_t s) {
    const int groups = L.mt * L.nt * L.slices;
    const dim3 grid((unsigned)groups);
    const bool few = groups <= CUS;            // deeper prefetch where no CU has two: 1000 x 4096 x 4096 23 us, 30 without; 128 x 4096 x 4096 12.1, 12.8
#define GO(WM, WN, U, ST, CU) hipLaunchKernelGGL((k_tile<WM, WN, U, ST, CU, GATED, DIRECT>), grid, dim3(BLOCK), 0, s, J)
    if constexpr (DIRECT) {
        if (L.tile == 0) GO(4, 4, 4, 5, 1);
        if (L.tile == 1) GO(4, 3, 4, 5, 1);
        if (L.tile == 2) GO(4, 2, 8, 3, 1);
        if (L.tile == 3 && few) GO(2, 2, 8, 4, 1);
        if (L.tile == 3 && !few) GO(2, 2, 8, 2, 2);
        if (L.tile == 4 && few) GO(1, 2, 8, 6, 1);
        if (L.tile == 4 && !few) GO(1, 2, 8, 3, 2);
    } else {
        if (L.tile == 0) GO(4, 4, 4, 3, 1);
        if (L.tile == 1) GO(4, 3, 4, 3, 1);
        if (L.tile == 2) GO(4, 2, 8, 3, 1);
        if (L.tile == 3) GO(2, 2, 8, 3, 1);
        if (L.tile == 4) GO(1, 2, 8, 3, 2);
    }
#undef GO
}

// a call as planned; ws is large enough
template <bool GATED>
int run(const char *who, const Plan &L, Job J, bool aligned, void *ws, hipStream_t s) {
    if (L.tile == FEW) {
        const dim3 grid((unsigned)((J.n + 15) / 16));
        if (J.m <= 16) hipLaunchKernelGGL((k_few<1, GATED>), grid, dim3(64 * FEW_WAVES), 0, s, J);
        else hipLaunchKernelGGL((k_few<2, GATED>), grid, dim3(64 * FEW_WAVES), 0, s, J);
        VI_LAUNCH_CHECK(who);
        return VI_OK;
    }
    char *at = (char *)vi::align16(ws);
    J.partial = (int *)(at + L.pack_bytes);
    J.slices = L.slices;
    J.steps_per_slice = L.steps_per_slice;
    J.steps = L.steps;
    J.mt = L.mt;
    J.nt = L.nt;
    if (L.pack) {
        Pack P = {};
        P.k = J.k;
        P.units = whole_lines(J.k) / 16;
        J.k = J.steps * (16 * TILES[L.tile].units);
        const signed char **from[3] = {&J.a, &J.b, &J.b2};
        i64 *ld[3] = {&J.lda, &J.ldb, &J.ldb2}, rows = 0;
        for (int i = 0; i < 3; ++i) {
            const i64 here = i == 0 ? J.m : i == 1 || GATED ? J.n : 0;
            P.from[i] = *from[i];
            P.ld[i] = *ld[i];
            P.to[i] = (v4i *)at;
            P.rows[i] = rows += here;
            *from[i] = (const signed char *)at;
            *ld[i] = P.units * 16;
            at += here * P.units * 16;
        }
        const i64 blocks = (rows * P.units + BLOCK - 1) / BLOCK;
        hipLaunchKernelGGL(k_pack, dim3((unsigned)(blocks < 16 * CUS ? blocks : 16 * CUS)), dim3(BLOCK), 0, s, P);
        VI_LAUNCH_CHECK(who);
    }
    if (aligned || L.pack) launch_tile<GATED, true>(L, J, s);
    else launch_tile<GATED, false>(L, J, s);
    VI_LAUNCH_CHECK(who);
    if (L.slices > 1) {
        const i64 blocks = ((J.n + VEC - 1) / VEC * J.m + BLOCK - 1) / BLOCK;
        hipLaunchKernelGGL(k_join<GATED>, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(BLOCK), 0, s, J);
        VI_LAUNCH_CHECK(who);
    }
    return VI_OK;
}

template <bool GATED>
int launch(const char *who, const Job &J, void *ws, size_t ws_bytes, hipStream_t s) {
    const bool aligned = aligned_rows(J.a, J.lda) && aligned_rows(J.b, J.ldb) && (!GATED || aligned_rows(J.b2, J.ldb2));
    // the sizes of a call are often those of the thread's last one, and the plan is a good half of a microsecond
    static thread_local struct {
        i64 m, k, n;
        bool aligned;
        Plan plan;
    } last = {};
    if (last.m != J.m || last.k != J.k || last.n != J.n || last.aligned != aligned) last = {J.m, J.k, J.n, aligned, make_plan(J.m, J.k, J.n, GATED, aligned, true)};
    Plan L = last.plan;
    if (L.pack && (!ws || ws_bytes < L.ws_bytes)) L = make_plan(J.m, J.k, J.n, GATED, aligned, false);
    if (ws_bytes < L.ws_bytes || (L.ws_bytes && !ws)) return vi::fail(VI_ENOMEM, "%s: workspace %zu < %zu bytes", who, ws_bytes, L.ws_bytes);
    if (L.tile != FEW && !L.mt) return vi::fail(VI_EINVAL, "%s: %lld x %lld outputs", who, (long long)J.m, (long long)J.n);
    return run<GATED>(who, L, J, aligned, ws, s);
}

}  // namespace

extern "C" size_t vi_int8_matmul_workspace_bytes(int64_t m, int64_t k, int64_t n) { return workspace_bytes(m, k, n, false, false); }
extern "C" size_t vi_int8_matmul_best_workspace_bytes(int64_t m, int64_t k, int64_t n) { return workspace_bytes(m, k, n, false, true); }
extern "C" size_t vi_int8_gated_workspace_bytes(int64_t m, int64_t k, int64_t n) { return workspace_bytes(m, k, n, true, false); }
extern "C" size_t vi_int8_gated_best_workspace_bytes(int64_t m, int64_t k, int64_t n) { return workspace_bytes(m, k, n, true, true); }

extern "C" int vi_int8_matmul(const int8_t *a, int64_t lda, const int8_t *b, int64_t ldb, int64_t m, int64_t k, int64_t n,
                              const float *a_scale, const float *b_scale, const float *bias, int dtype, void *out, int64_t ldo, void *ws,
                              size_t ws_bytes, void *stream) {
    if (!is_float(dtype) && dtype != VI_I32 && dtype != VI_FIELD) return vi::fail(VI_EINVAL, "vi_int8_matmul: dtype %d", dtype);
    Job J = {};
    J.a = (const signed char *)a, J.b = (const signed char *)b, J.lda = lda, J.ldb = ldb, J.m = m, J.k = k, J.n = n;
    J.a_scale = a_scale, J.b_scale = b_scale, J.bias = bias, J.dtype = dtype, J.out = out, J.ldo = ldo;
    if (int rc = check("vi_int8_matmul", J, false)) return rc;
    if (m == 0 || n == 0) return VI_OK;
    return launch<false>("vi_int8_matmul", J, ws, ws_bytes, (hipStream_t)stream);
}

extern "C" int vi_int8_gated(const int8_t *a, int64_t lda, const int8_t *gate, int64_t ldg, const int8_t *up, int64_t ldu, int64_t m, int64_t k,
                             int64_t n, const float *a_scale, const float *gate_scale, const float *up_scale, int activation, int dtype,
                             void *out, int64_t ldo, void *ws, size_t ws_bytes, void *stream) {
    if (!is_float(dtype)) return vi::fail(VI_EINVAL, "vi_int8_gated: dtype %d is none of VI_F32, VI_BF16, VI_F16", dtype);
    if (activation != VI_SILU && activation != VI_GELU) return vi::fail(VI_EINVAL, "vi_int8_gated: activation %d", activation);
    Job J = {};
    J.a = (const signed char *)a, J.b = (const signed char *)gate, J.b2 = (const signed char *)up, J.lda = lda, J.ldb = ldg, J.ldb2 = ldu;
    J.m = m, J.k = k, J.n = n, J.a_scale = a_scale, J.b_scale = gate_scale, J.b2_scale = up_scale, J.act = activation;
    J.dtype = dtype, J.out = out, J.ldo = ldo;
    if (int rc = check("vi_int8_gated", J, true)) return rc;
    if (m == 0 || n == 0) return VI_OK;
    return launch<true>("vi_int8_gated", J, ws, ws_bytes, (hipStream_t)stream);
}
