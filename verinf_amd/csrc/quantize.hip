// Rows of floats to 8-bit integers with a scale each.
//
//     A = max |x_j|    s = A / 127    r = 127 / A (both rounded to 32 bits)    q_j = rint(x_j r), half to even
//
// The product x_j r is rounded to 32 bits before rint: one multiplication an element, and |q| <= 127 since |x_j| <= A.
// A row whose scale would be no normal number (A < 127 2^-126) is zero: its r would overflow.  A NaN or an infinity makes the
// row's scale NaN and its integers zero, so that it shows in every product with them.
#include "number_types.hpp"

namespace {

using namespace num;

constexpr int BLOCK = 256;

template <int DT>
__global__ __launch_bounds__(BLOCK) void k_quantize(const typename type<DT>::t *x, i64 k, i64 ldx, signed char *q, i64 ldq, float *scale) {
    __shared__ u32 seen[BLOCK / 64];
    const i64 row = blockIdx.x;
    x += row * ldx;
    q += row * ldq;
    // as bit patterns: |x| in order, infinity above every number and NaN above that
    u32 top = 0;
    for (i64 j = threadIdx.x; j < k; j += BLOCK) top = max(top, __float_as_uint((float)x[j]) & 0x7FFFFFFFu);
#pragma unroll
    for (int d = 32; d; d >>= 1) top = max(top, (u32)__shfl_xor((int)top, d));
    if ((threadIdx.x & 63) == 0) seen[threadIdx.x / 64] = top;
    __syncthreads();
    for (int w = 0; w < BLOCK / 64; ++w) top = max(top, seen[w]);
    const float most = __uint_as_float(top);
    const bool none = most < 127.0f * 0x1p-126f, bad = top >= 0x7F800000u;
    const float r = none || bad ? 0.0f : 127.0f / most;
    if (threadIdx.x == 0) scale[row] = bad ? __uint_as_float(0x7FC00000u) : none ? 0.0f : most / 127.0f;
    for (i64 j = threadIdx.x; j < k; j += BLOCK) q[j] = bad ? 0 : (signed char)(int)rintf((float)x[j] * r);
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
    if (dtype == VI_F32) hipLaunchKernelGGL(k_quantize<VI_F32>, dim3((unsigned)m), dim3(BLOCK), 0, s, (const float *)x, k, ldx, (signed char *)q, ldq, scale);
    if (dtype == VI_BF16) hipLaunchKernelGGL(k_quantize<VI_BF16>, dim3((unsigned)m), dim3(BLOCK), 0, s, (const __bf16 *)x, k, ldx, (signed char *)q, ldq, scale);
    if (dtype == VI_F16) hipLaunchKernelGGL(k_quantize<VI_F16>, dim3((unsigned)m), dim3(BLOCK), 0, s, (const _Float16 *)x, k, ldx, (signed char *)q, ldq, scale);
    VI_LAUNCH_CHECK("quantize_rows");
    return VI_OK;
}
