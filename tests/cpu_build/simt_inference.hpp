// What the kernels of the forward pass in 8-bit integers use beside the rest of cpu_build/simt, for clang: their 16-bit number types,
// vectors of them and element-wise operations are that compiler's own.  LDS is static here, so that AddressSanitizer sees its ends.
//
// Loads straight into LDS.  A lane's load arrives at once, which shows a place that is overwritten while it is still read, or (SIMT_LATE=1) when a
// wait for it is reached and not before, which shows a wait that is missing.
//
// Fibers change places by a switch of their own: AddressSanitizer clears the whole stack's shadow at every swapcontext, and these kernels
// meet at every vote of the lanes.
#pragma once
#include <sanitizer/asan_interface.h>
#include <ucontext.h>

extern "C" void simt_switch(greg_t *from, greg_t to);                 // rbp, rbx and r12 to r15 on the stack, whose end is kept
__asm__(".text\n.type simt_switch, @function\nsimt_switch:\n\tpush %rbp\n\tpush %rbx\n\tpush %r12\n\tpush %r13\n\tpush %r14\n\tpush %r15\n\t"
        "mov %rsp, (%rdi)\n\tmov %rsi, %rsp\n\tpop %r15\n\tpop %r14\n\tpop %r13\n\tpop %r12\n\tpop %rbx\n\tpop %rbp\n\tret\n");
inline void simt_make(ucontext_t *c, void (*start)(), int) {
    __asan_unpoison_memory_region(c->uc_stack.ss_sp, c->uc_stack.ss_size);
    uint64_t *top = (uint64_t *)((char *)c->uc_stack.ss_sp + c->uc_stack.ss_size) - 10;               // six registers, the start, its caller
    for (int i = 0; i < 10; ++i) top[i] = i == 6 ? (uint64_t)start : 0;
    c->uc_mcontext.gregs[REG_RSP] = (greg_t)top;
}
#define makecontext simt_make
#define swapcontext(from, to) simt_switch(&(from)->uc_mcontext.gregs[REG_RSP], (to)->uc_mcontext.gregs[REG_RSP])
#define getcontext(c) ((void)0)
#include <hip/hip_runtime.h>

#include <atomic>
#include <cfloat>
#include <cmath>
#include <cstdarg>
#include <deque>
#include <type_traits>

#undef ext_vector_type
#undef __shared__
#define __shared__ static

using ::fabsf;
using ::fmaxf;
using ::fminf;

inline int max(int a, int b) { return a > b ? a : b; }
inline int64_t min(int64_t a, int64_t b) { return a < b ? a : b; }
inline int64_t max(int64_t a, int64_t b) { return a > b ? a : b; }
inline uint64_t max(uint64_t a, uint64_t b) { return a > b ? a : b; }
inline float __uint_as_float(uint32_t u) { float f; memcpy(&f, &u, 4); return f; }
inline int __float_as_int(float f) { int i; memcpy(&i, &f, 4); return i; }
inline int __popcll(uint64_t v) { return __builtin_popcountll(v); }

namespace simt {

inline long groups_met = 0;                                           // how often a workgroup's first thread has come to a barrier

// a lane's loads to LDS that have not arrived, oldest first, and where its next one goes
struct Load {
    char *to;
    const char *from;
};
inline std::deque<Load> loads[1024];
inline char *lds_memory;
inline uint32_t lds_next[1024];
inline bool late() {
    static const bool is = getenv("SIMT_LATE") != nullptr;
    return is;
}
inline uint32_t lds_base(char *memory) {
    lds_memory = memory;
    return 0;
}
inline void arrive(const Load &l) { memcpy(l.to, l.from, 16); }
inline void fetch_at(uint32_t at) { lds_next[threadIdx.x] = at; }
inline void fetch(uint32_t off, uint64_t base) {
    uint32_t &at = lds_next[threadIdx.x];
    const Load l = {lds_memory + at + (threadIdx.x & 63) * 16, (const char *)base + off};
    if ((uintptr_t)l.from & 15) {
        fprintf(stderr, "a load to LDS from %p\n", (const void *)l.from);
        abort();
    }
    at += 0x1000;
    if (late()) loads[threadIdx.x].push_back(l);
    else arrive(l);
}
inline void wait_for_loads_but(size_t n) {
    auto &mine = loads[threadIdx.x];
    for (; mine.size() > n; mine.pop_front()) arrive(mine.front());
}
inline void none_under_way() {
    for (auto &of : loads)
        if (!of.empty()) {
            fprintf(stderr, "a load that nothing waits for\n");
            abort();
        }
}

// What all lanes of a wavefront say, in one meeting: the words of one are read before the next, and there are two places in turn.  For
// code where the same lanes take part every time.
inline uint64_t said[16][2][64];
inline bool turn[1024];
inline const uint64_t *all_say(uint64_t v) {
    uint64_t *lanes = said[threadIdx.x >> 6][turn[threadIdx.x] ^= true];
    lanes[threadIdx.x & 63] = v;
    wait_at(AT_LANES);
    return lanes;
}
template <class T>
T lane_value(T v, int from) {
    uint64_t w = 0;
    memcpy(&w, &v, sizeof(v));
    w = all_say(w)[from];
    memcpy(&v, &w, sizeof(v));
    return v;
}

// Matrix instructions on signed bytes, 16 * PARTS inner indices: lane l holds row (column) l % N of A (B), the sixteen inner indices from
// 16 (l / N); at(r) is the row of the result's register r, whose column is l % N.
template <int N, int REGS, class At>
__attribute__((no_sanitize("address", "undefined"))) void multiply(const int8_t (*a)[16], const int8_t (*b)[16], int32_t *c, int lane, At at) {
    for (int r = 0; r < REGS; ++r)
        for (int part = 0; part < 64; part += N) {
            const int8_t *x = a[at(r) + part], *y = b[lane % N + part];
            int sum = 0;
            for (int i = 0; i < 16; ++i) sum += x[i] * y[i];
            c[r] += sum;
        }
}
inline int8_t bytes_a[16][64][16], bytes_b[16][64][16];
template <int N, int REGS, class V, class C, class At>
void mfma(const V &a, const V &b, C &c, At at) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    memcpy(bytes_a[wave][lane], &a, 16);
    memcpy(bytes_b[wave][lane], &b, 16);
    __builtin_amdgcn_wave_barrier();
    int32_t sums[REGS];
    memcpy(sums, &c, sizeof(sums));
    multiply<N, REGS>(bytes_a[wave], bytes_b[wave], sums, lane, at);
    memcpy(&c, sums, sizeof(sums));
    __builtin_amdgcn_wave_barrier();
}
template <class V, class C>
C mfma_32x32x32(const V &a, const V &b, C c) {
    mfma<32, 16>(a, b, c, [half = (int)(threadIdx.x & 63) / 32](int r) { return 8 * (r / 4) + 4 * half + r % 4; });
    return c;
}
template <class V, class C>
C mfma_16x16x64(const V &a, const V &b, C c) {
    mfma<16, 4>(a, b, c, [part = (int)(threadIdx.x & 63) / 16](int r) { return 4 * part + r; });
    return c;
}

struct Two {
    uint32_t v[2];
    uint32_t operator[](int i) const { return v[i]; }
};
// the upper 32 lanes of a and the lower ones of b change places
inline Two swap_halves(uint32_t a, uint32_t b) {
    const int lane = threadIdx.x & 63;
    const uint32_t from_b = lane_value(b, lane ^ 32), from_a = lane_value(a, lane ^ 32);
    return lane < 32 ? Two{{a, from_a}} : Two{{from_b, b}};
}

}  // namespace simt

template <class T>
T __shfl_xor(T v, int mask) { return simt::lane_value(v, (int)(threadIdx.x & 63) ^ mask); }
__attribute__((no_sanitize("address", "undefined"))) inline uint64_t __ballot(bool v) {                                    // where all lanes are
    const uint64_t *lanes = simt::all_say(v);
    uint64_t all = 0;
    for (int i = 0; i < 64; ++i) all |= lanes[i] << i;
    return all;
}
inline void simt_meet() {
    simt::groups_met += threadIdx.x == 0;
    simt::wait_at(simt::AT_GROUP);
}
#define __syncthreads() simt_meet()
#define __builtin_amdgcn_sched_barrier(x) ((void)0)
#define __builtin_amdgcn_permlane32_swap(a, b, x, y) simt::swap_halves(a, b)
#undef __builtin_amdgcn_mfma_i32_32x32x32_i8
#define __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, x, y, z) simt::mfma_32x32x32(a, b, c)
#define __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, x, y, z) simt::mfma_16x16x64(a, b, c)
// results below the least normal number are zero
inline float simt_exp2(float x) {
    const float r = ::exp2f(x);
    return r < FLT_MIN ? 0.0f : r;
}
#define __builtin_amdgcn_exp2f(x) simt_exp2(x)
#define __builtin_amdgcn_rcpf(x) (1.0f / (x))
