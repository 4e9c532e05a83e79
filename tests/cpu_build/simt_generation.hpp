// What the kernels of the cache, the attention over it and the drafts use beside simt_inference.hpp: products of 16-bit numbers, LDS reads that transpose,
// loads of 16 and of 4 bytes straight into LDS at addresses of their own.
//
// With SIMT_LATE=1 a load arrives when a wait for it is reached and not before.  A lane counts its own loads, so that this shows for stages in which all lanes load
// alike: those of 16-bit numbers whose columns fill the units.
#pragma once
#include "simt_inference.hpp"

inline int __ffsll(unsigned long long v) { return __builtin_ffsll((long long)v); }
inline int __clzll(long long v) { return v ? __builtin_clzll((unsigned long long)v) : 64; }
template <class T>
T __shfl(T v, int lane) { return simt::lane_value(v, lane); }
using ::fma;
using ::fmax;

namespace simt {

struct Piece {
    char *to;
    const char *from;
    int bytes;
};
inline std::deque<Piece> pieces[1024];
inline void piece(uint32_t at, const char *from, int bytes) {
    if ((uintptr_t)from % bytes) {
        fprintf(stderr, "a load of %d bytes to LDS from %p\n", bytes, (const void *)from);
        abort();
    }
    const Piece p = {lds_memory + at + (threadIdx.x & 63) * bytes, from, bytes};
    if (late()) pieces[threadIdx.x].push_back(p);
    else memcpy(p.to, p.from, bytes);
}
inline void fetch16(uint32_t at, uint32_t off, uint64_t base) { piece(at, (const char *)base + off, 16); }
inline void fetch4(uint32_t at, const float *from) { piece(at, (const char *)from, 4); }
inline void arrived_but(size_t n) {
    auto &mine = pieces[threadIdx.x];
    for (; mine.size() > n; mine.pop_front()) memcpy(mine.front().to, mine.front().from, mine.front().bytes);
}
inline void no_pieces() {
    for (auto &of : pieces)
        if (!of.empty()) {
            fprintf(stderr, "a load that nothing waits for\n");
            abort();
        }
}

// of each sixteen lanes, lane i gets column i of `rows` rows, whose pieces of 8 bytes are at the lanes' addresses one after the other
template <class V, class E, int ROWS>
V transposed(const void *from) {
    const int lane = threadIdx.x & 63, group = lane & ~15, column = lane & 15, each = 16 / ROWS, per = 8 / sizeof(E);
    const uint64_t *places = all_say((uint64_t)from);
    E e[ROWS];
    for (int r = 0; r < ROWS; ++r) memcpy(&e[r], (const E *)places[group + r * each + column / per] + column % per, sizeof(E));
    V v;
    memcpy(&v, e, sizeof(v));
    __builtin_amdgcn_wave_barrier();           // nobody overwrites what another still reads
    return v;
}

inline float halves_a[16][64][8], halves_b[16][64][8];
template <class V, class C>
__attribute__((no_sanitize("address", "undefined"))) C mfma_32x32x16(const V &a, const V &b, C c) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = 0; i < 8; ++i) halves_a[wave][lane][i] = (float)a[i], halves_b[wave][lane][i] = (float)b[i];
    __builtin_amdgcn_wave_barrier();
    for (int r = 0; r < 16; ++r) {
        const int row = 8 * (r / 4) + 4 * (lane / 32) + r % 4;
        float sum = c[r];
        for (int part = 0; part < 64; part += 32)
            for (int i = 0; i < 8; ++i) sum += halves_a[wave][row + part][i] * halves_b[wave][lane % 32 + part][i];
        c[r] = sum;
    }
    __builtin_amdgcn_wave_barrier();
    return c;
}

}  // namespace simt

template <class V>
float simt_dot2(V a, V b, float c) { return (float)a[0] * (float)b[0] + (float)a[1] * (float)b[1] + c; }
#define __builtin_amdgcn_sched_barrier(mask)
#define __builtin_amdgcn_fdot2(a, b, c, clamp) simt_dot2(a, b, c)
#define __builtin_amdgcn_fdot2_f32_bf16(a, b, c, clamp) simt_dot2(a, b, c)
#define __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, x, y, z) simt::mfma_32x32x16(a, b, c)
#define __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, x, y, z) simt::mfma_32x32x16(a, b, c)
#define __builtin_amdgcn_ds_read_tr16_b64_v4i16(p) simt::transposed<v4s, short, 4>(p)
#define __builtin_amdgcn_ds_read_tr8_b64_v2i32(p) simt::transposed<v2i, char, 8>(p)
