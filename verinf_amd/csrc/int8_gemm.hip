// Products of 8-bit integers with a scale for each row of A (token) and of B (channel), and the gated block of two of them.
//
//     S_ij = sum_l a_il b_jl          out = S, S mod p, or (S_ij a_scale_i) b_scale_j + bias_j
//     gated: act((S_ij a_scale_i) g_scale_j) ((T_ij a_scale_i) u_scale_j), S and T of the same A with two B
//
// Both operands have their inner dimension along the rows, so a wavefront's operands of a matrix instruction are 16 contiguous bytes a
// lane.  Sums are exact: |S| <= 2^14 k fits 32 bits up to MAX_K.
#include "int8_gemm.hpp"

namespace {

using namespace i8;

constexpr int MAX_K = 131071;
constexpr int STEP = 64;                       // inner indices of a step
constexpr int UNITS = STEP / 16;

// units of a row are stored in another order, by the row, so that lanes that read one unit of neighbouring rows meet different banks
__device__ __forceinline__ int slot(int row, int unit) { return row * UNITS + (unit ^ ((row >> 1) & 3)); }

// column c of a tile's 64 WN virtual columns -> its row of B, or of the second B where *second: a wavefront's first half of the
// columns are the gate's, its other half the same channels' of the up projection, so that both sums of an output are in one lane
template <int WN, bool GATED>
__device__ __forceinline__ i64 channel(int tn, int c, bool *second) {
    if (!GATED) {
        *second = false;
        return (i64)tn * (64 * WN) + c;
    }
    const int wc = c / (32 * WN), in = c % (32 * WN), half = in / (16 * WN);
    *second = half;
    return (i64)tn * (32 * WN) + wc * (16 * WN) + in % (16 * WN);
}

template <int WM, int WN>
struct Lds {
    v4i a[64 * WM * UNITS], b[64 * WN * UNITS];
};

// A tile of 64 WM rows and 64 WN (virtual) columns by four wavefronts in a square.
template <int WM, int WN, bool GATED>
__global__ __launch_bounds__(BLOCK) void k_tile(Job J) {
    constexpr int TM = 64 * WM, TN = 64 * WN, PITCH = 32 * WN + 8;
    __shared__ union {
        Lds<WM, WN> in;
        int out[4][32 * PITCH];
    } lds;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int total = J.mt * J.nt;
    const int slice = blockIdx.x / total, id = blockIdx.x % total, tm = id % J.mt, tn = id / J.mt;
    const int s0 = slice * J.steps_per_slice, s1 = min(s0 + J.steps_per_slice, J.steps);

    const signed char *src[WM + WN];
#pragma unroll
    for (int j = 0; j < WM + WN; ++j) {
        const int row = (j < WM ? j : j - WM) * 64 + (tid >> 2);
        if (j < WM) {
            src[j] = J.a + min((i64)tm * TM + row, J.m - 1) * J.lda;
        } else {
            bool second;
            const i64 c = min(channel<WN, GATED>(tn, row, &second), J.n - 1);
            src[j] = second ? J.b2 + c * J.ldb2 : J.b + c * J.ldb;
        }
        src[j] += (tid & 3) * 16;
    }
    v16i acc[WM][WN];
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int j = 0; j < WN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
    const int row0 = (wave >> 1) * (32 * WM) + (lane & 31), col0 = (wave & 1) * (32 * WN) + (lane & 31), half = lane >> 5;
    for (int s = s0; s < s1; ++s) {
        const i64 at = (i64)s * STEP;
        v4i in[WM + WN];
#pragma unroll
        for (int j = 0; j < WM + WN; ++j) in[j] = load_part(src[j] + at, J.k - at - (tid & 3) * 16);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < WM + WN; ++j) {
            const int row = (j < WM ? j : j - WM) * 64 + (tid >> 2);
            (j < WM ? lds.in.a : lds.in.b)[slot(row, tid & 3)] = in[j];
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < UNITS / 2; ++t) {
            v4i x[WM], y[WN];
#pragma unroll
            for (int i = 0; i < WM; ++i) x[i] = lds.in.a[slot(row0 + 32 * i, 2 * t + half)];
#pragma unroll
            for (int j = 0; j < WN; ++j) y[j] = lds.in.b[slot(col0 + 32 * j, 2 * t + half)];
#pragma unroll
            for (int i = 0; i < WM; ++i)
#pragma unroll
                for (int j = 0; j < WN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(x[i], y[j], acc[i][j], 0, 0, 0);
        }
    }

    // 32 rows at a time through the wavefront's own part of LDS, so that a lane has neighbouring columns: register r of a
    // tile is row 8 (r / 4) + 4 half + r % 4, column lane % 32
    __syncthreads();
    int *buf = lds.out[wave];
    constexpr int WIDE = GATED ? 16 * WN : 32 * WN, VECS = WIDE / VEC;
#pragma unroll
    for (int i = 0; i < WM; ++i) {
#pragma unroll
        for (int j = 0; j < WN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) buf[(8 * (r / 4) + 4 * half + r % 4) * PITCH + 32 * j + (lane & 31)] = acc[i][j][r];
        __syncthreads();
        for (int it = 0; it < 32 * VECS / 64; ++it) {
            const int p = it * 64 + lane, lrow = p / VECS, lcol = p % VECS * VEC;
            const i64 row = (i64)tm * TM + (wave >> 1) * (32 * WM) + 32 * i + lrow, col = (i64)tn * (GATED ? TN / 2 : TN) + (wave & 1) * WIDE + lcol;
            const int count = (int)min(J.n - col, (i64)VEC);
            if (row >= J.m || count <= 0) continue;
            int v[VEC], w[VEC];
            __builtin_memcpy(v, buf + lrow * PITCH + lcol, sizeof(v));
            if (GATED) __builtin_memcpy(w, buf + lrow * PITCH + WIDE + lcol, sizeof(w));
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
        __syncthreads();
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
        for (int q = 0; q < J.slices; ++q)
#pragma unroll
            for (int h = 0; h < (GATED ? 2 : 1); ++h) {
                const int *s = J.partial + ((i64)q * (GATED ? 2 : 1) + h) * mn + row * J.n + col;
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (e < count) (h ? w : v)[e] += s[e];
            }
        finish<GATED>(J, row, col, count, v, w);
    }
}

struct Plan {
    int slices, steps_per_slice, steps, mt, nt;
    size_t ws_bytes;
};

Plan make_plan(i64 m, i64 k, i64 n, bool gated) {
    Plan L;
    const i64 cols = gated ? 64 : 128, mt = (m + 127) / 128, nt = (n + cols - 1) / cols;
    L.mt = (int)mt;
    L.nt = (int)nt;
    L.steps = (int)((k + STEP - 1) / STEP);
    // slices of the inner dimension until there are two tiles for every CU, of at least 8 steps
    i64 slices = 1;
    while (mt * nt * slices * 2 <= 512 && L.steps / (slices * 2) >= 8) slices *= 2;
    L.steps_per_slice = (int)((L.steps + slices - 1) / slices);
    L.slices = L.steps ? (L.steps + L.steps_per_slice - 1) / L.steps_per_slice : 1;
    L.ws_bytes = L.slices > 1 ? (size_t)4 * L.slices * (gated ? 2 : 1) * m * n + vi::WS_SLACK : 0;
    return L;
}

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

template <bool GATED>
int launch(const char *who, Job J, void *ws, size_t ws_bytes, hipStream_t s) {
    const Plan L = make_plan(J.m, J.k, J.n, GATED);
    if (ws_bytes < L.ws_bytes || (L.ws_bytes && !ws)) return vi::fail(VI_ENOMEM, "%s: workspace %zu < %zu bytes", who, ws_bytes, L.ws_bytes);
    if ((i64)L.mt * L.nt * L.slices > 0x7FFFFFFF) return vi::fail(VI_EINVAL, "%s: %lld x %lld outputs", who, (long long)J.m, (long long)J.n);
    J.partial = (int *)vi::align16(ws);
    J.slices = L.slices;
    J.steps_per_slice = L.steps_per_slice;
    J.steps = L.steps;
    J.mt = L.mt;
    J.nt = L.nt;
    hipLaunchKernelGGL((k_tile<2, 2, GATED>), dim3((unsigned)(L.mt * L.nt * L.slices)), dim3(BLOCK), 0, s, J);
    VI_LAUNCH_CHECK(who);
    if (L.slices > 1) {
        const i64 blocks = ((J.n + VEC - 1) / VEC * J.m + BLOCK - 1) / BLOCK;
        hipLaunchKernelGGL(k_join<GATED>, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(BLOCK), 0, s, J);
        VI_LAUNCH_CHECK(who);
    }
    return VI_OK;
}

}  // namespace

extern "C" size_t vi_int8_matmul_workspace_bytes(int64_t m, int64_t k, int64_t n) {
    return m > 0 && k >= 0 && n > 0 && k <= MAX_K ? make_plan(m, k, n, false).ws_bytes : 0;
}

extern "C" size_t vi_int8_gated_workspace_bytes(int64_t m, int64_t k, int64_t n) {
    return m > 0 && k >= 0 && n > 0 && k <= MAX_K ? make_plan(m, k, n, true).ws_bytes : 0;
}

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
