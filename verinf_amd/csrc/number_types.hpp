// The number types of the forward pass's operators (VI_F32 ...), as kernels see them: unaligned vectors in, floats out and back.
#pragma once

#include "common.hpp"

namespace num {

typedef int64_t i64;
typedef uint32_t u32;
typedef uint64_t u64;

template <int DT> struct type;
template <> struct type<VI_F32> { typedef float t; };
template <> struct type<VI_BF16> { typedef __bf16 t; };
template <> struct type<VI_F16> { typedef _Float16 t; };

constexpr int size_of(int dtype) { return dtype == VI_F32 || dtype == VI_I32 ? 4 : dtype == VI_FIELD ? 8 : 2; }
constexpr bool is_float(int dtype) { return dtype == VI_F32 || dtype == VI_BF16 || dtype == VI_F16; }

// N bytes at any address: one access where the hardware has one of that width (it takes any alignment)
template <class V, class P>
__device__ __forceinline__ V load_any(const P *p) {
    V v;
    __builtin_memcpy(&v, p, sizeof(V));
    return v;
}
template <class V, class P>
__device__ __forceinline__ void store_any(P *p, const V &v) {
    __builtin_memcpy(p, &v, sizeof(V));
}

// element e of 16 loaded bytes as a float
template <int DT>
__device__ __forceinline__ float element(const u32 *w, int e) {
    if constexpr (DT == VI_F32) return __uint_as_float(w[e]);
    if constexpr (DT == VI_BF16) return __uint_as_float(e & 1 ? w[e / 2] & 0xFFFF0000u : w[e / 2] << 16);
    const unsigned short h = (unsigned short)(e & 1 ? w[e / 2] >> 16 : w[e / 2]);
    return (float)__builtin_bit_cast(_Float16, h);
}

}  // namespace num
