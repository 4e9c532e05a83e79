// Drafted tokens held against the target's probabilities, and the accepted ones' cache entries moved to the front.
//
// A node's children are tried in their order, which is that of the nodes, so that one walk over a sequence's nodes tries them all.  With
// p and q the target's and the draft model's probabilities behind the node, R = p at first, child c with token x is accepted where
// u_c q(x) sum(R) < R(x), and behind a refused one R = max(R / sum(R) - q, 0).  Up to a factor that is
//
//     R = max(p - a q, 0)        a = 0 at first, a <- a + sum(R) at each refusal, sum(R) with the p and q that sum to one
//
// since max(max(p - a q, 0) - W q, 0) = max(p - (a + W) q, 0): nothing is stored of it but a.  Without the draft's probabilities R loses
// the refused tokens and is otherwise p.
//
// Whole numbers come of it, decided by comparisons next to borders, of which the last token's have as many as there are tokens: all in 64
// bits, exponentials too (4e-16 off).
//
// All rows' largest entries and sums, in slices (k_stats), and the sums behind a first refusal, for nodes with other children (k_first), are taken by the whole
// chip; a workgroup a sequence walks (k_walk), with a pass over two rows for each further refusal; the whole chip adds up what is left behind the paths
// (k_left), and a workgroup a sequence looks for the token (k_pick).
//
// What bounds them: some 16 instructions an exponential, twelve of them in 64 bits, which issue every 5 cycles.  64 trees of 16 nodes, 32000 bf16 logits of both models:
// 116 us over three sets of inputs, 108 to 118 by the sequence with the most refusals, 9 us each.  The parts of a set that takes 131: 46 all rows' sums, 24 first refusals, 54 the walk,
// 11 the last tokens.  Half of all rows' sums are of leaves of the trees, which nobody asks for; what is needed could be read in 9 us.  With the 11 powers of a series on [-1/2, 1/2] and no
// table it was 149 us, with the table and four powers, 1.6e-13 off, 126 then and 3 % less than now.  One chain of five nodes, f32: 16 us, the latency of four launches.
#include "cache.hpp"

namespace {

using namespace kv;

constexpr int BLOCK = 256, WALK = 1024;        // threads
constexpr i64 MAX_V = 1 << 20;
constexpr i64 MAX_BLOCKS = 1 << 23;            // of a launch, which has less than 2^32 threads
constexpr int MAX_NODES = 1024, MAX_DEPTH = 256;
constexpr int EIGHT = 8;                       // neighbouring entries of a thread
constexpr double MARGIN = 64;                  // bits
constexpr double CLOSE = 0x1p-40;              // sums of up to 2^20 probabilities, 4096 a thread, are 2^-41 off at most

struct Part {                                  // of a slice: an entry of its largest (NaN: it has a NaN or +inf), sum of 2^((x - most) c / 32)
    double z;
    float most, pad;
};
struct Row {                                   // of a row: the largest, which its sum is relative to; 1 / sum, 0 where it has none (or NaN, +inf among its entries)
    double most, per_z;
};

// 2^(d c / 32) of N numbers side by side (one alone waits for itself at each step), d c up to 0 or hardly above, less than LEAST from where it would be that: the whole part by an
// addition whose result has units of one, its last five bits from a table, the others into the exponent, the rest by a polynomial (over Chebyshev's nodes, 1.4e-16).
// d is a difference of entries, taken before the product: c times an entry of 10^38 has no digits that c times another could be taken from.
// The table has 256 bytes, a pair of banks to each entry; the exponent comes into the entry by adding the whole part as it is, 15 bits up in the upper half, from
// where the entry has lost its own number before.
constexpr int STEPS = 32;
constexpr double LEAST = 0x1p-1022;            // what is below it stands for anything down to nothing: of a masked entry, say
constexpr double DEEPEST = -1022.25 * STEPS;   // of d c: a quarter of a power of two below LEAST, so that no rounding of it is above
struct Scale {                                 // of a launch: 32 log2(e) / temperature, DEEPEST / c
    double c, deepest;
};
__device__ const double TABLE[STEPS] = {0x1.0000000000000p+0, 0x1.059b0d3158574p+0, 0x1.0b5586cf9890fp+0, 0x1.11301d0125b51p+0, 0x1.172b83c7d517bp+0, 0x1.1d4873168b9aap+0,
                                      0x1.2387a6e756238p+0, 0x1.29e9df51fdee1p+0, 0x1.306fe0a31b715p+0, 0x1.371a7373aa9cbp+0, 0x1.3dea64c123422p+0, 0x1.44e086061892dp+0,
                                      0x1.4bfdad5362a27p+0, 0x1.5342b569d4f82p+0, 0x1.5ab07dd485429p+0, 0x1.6247eb03a5585p+0, 0x1.6a09e667f3bcdp+0, 0x1.71f75e8ec5f74p+0,
                                      0x1.7a11473eb0187p+0, 0x1.82589994cce13p+0, 0x1.8ace5422aa0dbp+0, 0x1.93737b0cdc5e5p+0, 0x1.9c49182a3f090p+0, 0x1.a5503b23e255dp+0,
                                      0x1.ae89f995ad3adp+0, 0x1.b7f76f2fb5e47p+0, 0x1.c199bdd85529cp+0, 0x1.cb720dcef9069p+0, 0x1.d5818dcfba487p+0, 0x1.dfc97337b9b5fp+0,
                                      0x1.ea4afa2a490dap+0, 0x1.f50765b6e4540p+0};
__device__ __forceinline__ void take_table(double *table) {        // a barrier has to follow
    if (threadIdx.x < STEPS) table[threadIdx.x] = __builtin_bit_cast(double, __builtin_bit_cast(u64, TABLE[threadIdx.x]) - ((u64)threadIdx.x << 47));
}
template <int N>
__device__ __forceinline__ void exp2_64(const double *table, const Scale &S, double (&d)[N], double (&scale)[N]) {         // times scale
    constexpr double C[] = {3.9737238568525983e-11, 9.172607532092245e-09, 1.6938509724285119e-06, 0.0002345961981994449, 0.021660849392498290, 1.0};
    double m[N], f[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
        d[e] = fmax(d[e], S.deepest);
        m[e] = fma(d[e], S.c, 6755399441055744.0);
        f[e] = fma(d[e], S.c, -(m[e] - 6755399441055744.0));
        const u32 k = (u32)__builtin_bit_cast(u64, m[e]);
        const u64 entry = __builtin_bit_cast(u64, table[k % STEPS]);
        scale[e] = __builtin_bit_cast(double, (u64)((u32)(entry >> 32) + (k << 15)) << 32 | (u32)entry);
        d[e] = C[0];
    }
#pragma unroll
    for (int i = 1; i < 6; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e) d[e] = fma(d[e], f[e], C[i]);
}
__device__ __forceinline__ double exp2_64(const double *table, const Scale &S, double d) {
    double one[1] = {d}, scale[1];
    exp2_64(table, S, one, scale);
    return one[0] * scale[0];
}
// an entry's part of its row's sum as a probability: none where it is LEAST
__device__ __forceinline__ double probability(double part, double per_z) { return part > LEAST ? part * per_z : 0.0; }

template <int DT>
struct Entries {                               // as they come
    u32 w[DT == VI_F32 ? 8 : 4];
};
template <int DT>
__device__ __forceinline__ float entry(const Entries<DT> &v, int e) {
    if constexpr (DT == VI_F32) return __uint_as_float(v.w[e]);
    else return element<DT>(v.w, e);
}
// the eight entries from `at` on; -inf behind the row's end
template <int DT>
__device__ __forceinline__ Entries<DT> eight(const typename type<DT>::t *x, i64 at, i64 v) {
    if (at + EIGHT <= v) return load_any<Entries<DT>>(x + at);
    typename type<DT>::t e[EIGHT];
#pragma unroll
    for (int i = 0; i < EIGHT; ++i) e[i] = at + i < v ? x[at + i] : (typename type<DT>::t)-INFINITY;
    Entries<DT> r;
    __builtin_memcpy(&r, e, sizeof(r));
    return r;
}
// the eight from `at` on where there are eight, anything otherwise: asked for ahead of their use
template <int DT>
__device__ __forceinline__ Entries<DT> first_eight(const typename type<DT>::t *x, i64 at, i64 end) {
    Entries<DT> r = {};
    if (at + EIGHT <= end) r = load_any<Entries<DT>>(x + at);
    return r;
}

// e^(x - most) of eight entries, in 64 bits: t times scale, to(i, t, scale)
template <int DT, class To>
__device__ __forceinline__ void exponentials(const double *table, const Scale &S, const Entries<DT> &v, double most, To to) {
#pragma unroll
    for (int h = 0; h < EIGHT; h += 4) {
        double t[4], scale[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = (double)entry<DT>(v, h + e) - most;
        exp2_64(table, S, t, scale);
#pragma unroll
        for (int e = 0; e < 4; ++e) to(h + e, t[e], scale[e]);
    }
}
template <int DT>
__device__ __forceinline__ void exponentials(const double *table, const Scale &S, const Entries<DT> &v, double most, double (&r)[EIGHT]) {
    exponentials<DT>(table, S, v, most, [&](int i, double t, double scale) __attribute__((always_inline)) { r[i] = t * scale; });
}

// The sum of max(e^(x - most) - ratio e^(y - most), 0) of eight entries of two rows.  (LEAST in the place of nothing: too
// little to change what comes of a sum.)
template <int DT>
__device__ __forceinline__ void add_left(const double *table, const Scale &S, const Entries<DT> &e, const Entries<DT> &f, double p_most, double q_most, double ratio, double &sum) {
    double o[EIGHT];
    exponentials<DT>(table, S, f, q_most, [&](int i, double t, double scale) __attribute__((always_inline)) { o[i] = t * (scale * ratio); });
    exponentials<DT>(table, S, e, p_most, [&](int i, double t, double scale) __attribute__((always_inline)) { sum += fmax(fma(t, scale, -o[i]), 0.0); });
}

struct Job {
    const void *x[2];                          // the target's logits, the draft's
    i64 ld[2], n, v;
    int slices, per_slice, firsts, sequences, apart, depth, drafted;           // apart: nodes of a sequence, on an average
    Scale scale;
    Part *parts;                               // [2 n][slices]
    double *first;                             // [n][firsts]: the sum of max(p - q, 0) of a slice
    Row *rows;                                 // [2 n]
    struct End *ends;                          // [sequences]
    double *segments;                          // [sequences][segments of a row]
    const i64 *tokens;
    const int *starts, *parents;
    const double *uniforms;
    i64 *counts, *nodes, *out;
};

// How many children the node of a row has, two at most, by a wavefront that asks for one row
__device__ __forceinline__ int children(const Job &A, i64 row) {
    int found = -1;
    i64 s0 = 0, s1 = 0;
    for (int first = 0; first < A.sequences; first += 64) {
        const int b = min(first + (int)(threadIdx.x & 63), A.sequences - 1);
        const i64 start = A.starts[b], next = A.starts[b + 1];
        const int count = __popcll(__ballot(first + (int)(threadIdx.x & 63) < A.sequences && start <= row));
        if (count == 0) break;
        found = first + count - 1;
        s0 = __shfl((int)start, count - 1), s1 = __shfl((int)next, count - 1);
    }
    s0 = max(s0, (i64)0), s1 = min(s1, A.n);
    if (found < 0 || row >= s1) return 0;
    if (!A.parents) return row + 1 < s1;
    int count = 0;
    for (i64 j = row + 1; j < min(s1, s0 + MAX_NODES) && count < 2; j += 64) {
        const i64 i = j + (threadIdx.x & 63);
        count += __popcll(__ballot(i < min(s1, s0 + MAX_NODES) && s0 + A.parents[min(i, s1 - 1)] == row));
    }
    return min(count, 2);
}

// The sum of a slice.  A thread's is relative to the largest of the first entries that it has seen, or of later ones where they are 2^MARGIN times those.
template <int DT>
__global__ __launch_bounds__(BLOCK) void k_stats(Job A) {
    typedef typename type<DT>::t T;
    __shared__ float most_of[BLOCK / 64];
    __shared__ double sum_of[BLOCK / 64], table[STEPS];
    const i64 row = blockIdx.x / A.slices;
    const int slice = (int)(blockIdx.x % A.slices), which = row >= A.n, lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    const T *x = (const T *)A.x[which] + (row - (which ? A.n : 0)) * A.ld[which];
    const i64 end = min(A.v, (i64)(slice + 1) * A.per_slice);
    i64 at = (i64)slice * A.per_slice + (int)threadIdx.x * EIGHT;
    Entries<DT> v = first_eight<DT>(x, at, end);
    if (which && children(A, row - A.n) == 0) return;                  // nobody asks
    take_table(table);
    __syncthreads();
    const float margin = (float)(MARGIN * STEPS / A.scale.c);
    float most = -INFINITY, bound = -INFINITY;
    double z = 0, from = 0;
    bool bad = false;
    auto add = [&](const Entries<DT> &e) __attribute__((always_inline)) {
        float here = entry<DT>(e, 0);
#pragma unroll
        for (int i = 1; i < EIGHT; ++i) here = __builtin_elementwise_maximum(here, entry<DT>(e, i));           // NaN where there is one
        bad |= !(here < INFINITY);
        if (here > bound && !bad) {
            z = z > 0 ? z * exp2_64(table, A.scale, from - (double)here) : 0.0;
            most = here, bound = here + margin, from = (double)here;
        }
        if (most > -INFINITY) {
            exponentials<DT>(table, A.scale, e, from, [&](int, double t, double scale) __attribute__((always_inline)) { z = fma(t, scale, z); });
        }
    };
    while (at + EIGHT <= end) {
        const i64 next = at + BLOCK * EIGHT;
        const Entries<DT> ahead = first_eight<DT>(x, next, end);
        add(v);
        v = ahead, at = next;
    }
    if (at < end) add(eight<DT>(x, at, end));
    if (bad) most = INFINITY;
    const float own = most;
#pragma unroll
    for (int d = 32; d; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
    if (lane == 0) most_of[wave] = most;
    __syncthreads();
    most = fmaxf(fmaxf(most_of[0], most_of[1]), fmaxf(most_of[2], most_of[3]));
    z = own > -INFINITY && most < INFINITY ? z * exp2_64(table, A.scale, from - (double)most) : 0.0;
#pragma unroll
    for (int d = 32; d; d >>= 1) z += __shfl_xor(z, d);
    if (lane == 0) sum_of[wave] = z;
    __syncthreads();
    if (threadIdx.x == 0) A.parts[blockIdx.x] = {(sum_of[0] + sum_of[1]) + (sum_of[2] + sum_of[3]), most == INFINITY ? __uint_as_float(0x7FC00000u) : most, 0.0f};
}

struct End {                                   // where a path ends: its node's row (-1: no sequence), its number, what is left of its probabilities
    double a;
    i64 row;
    int node, refused, count, pad;
};
struct Tree {                                  // -1: none, also of nodes that cannot be accepted
    int parent[MAX_NODES], token[MAX_NODES];
};
// a sequence's nodes
template <int THREADS>
__device__ __forceinline__ int take_tree(const Job &A, int b, Tree &tree, i64 *first) {
    const i64 s0 = max((i64)0, min((i64)A.starts[b], A.n)), s1 = max(s0, min((i64)A.starts[b + 1], A.n));
    const int nodes = (int)min(s1 - s0, (i64)MAX_NODES);
    for (int i = threadIdx.x; i < nodes; i += THREADS) {
        const int parent = i ? A.parents ? A.parents[s0 + i] : i - 1 : -1;
        const i64 token = A.tokens[s0 + i];
        const bool fine = parent >= 0 && parent < i && token >= 0 && token < A.v;
        tree.parent[i] = fine ? parent : -1;
        tree.token[i] = fine ? (int)token : -1;
    }
    *first = s0;
    return nodes;
}

struct Shared {
    Tree tree;
    double have[MAX_NODES], said[MAX_NODES], u[MAX_NODES];             // p and q of a node's token behind its parent
    double sums[WALK / 64], table[STEPS];
};

// the sum of the wavefront's values up to this lane's
__device__ __forceinline__ double sum_up_to(double v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double o = __shfl(v, max(lane - d, 0));
        if (lane >= d) v += o;
    }
    return v;
}
// the first lane whose sum is above the threshold, the last with anything where none is; -1: nothing anywhere
__device__ __forceinline__ int first_above(double sum, double own, double threshold) {
    const u64 above = __ballot(sum > threshold && own > 0), any = __ballot(own > 0);
    return above ? __ffsll((unsigned long long)above) - 1 : any ? 63 - __clzll((long long)any) : -1;
}

// What is left of a row: R(j) = max(p - a q, 0), or p without the tokens of the refused children of `cur`
template <int DT>
struct Left {
    const typename type<DT>::t *x, *y;
    Row p, q;
    double a;
    Scale scale;
    i64 v;
    const Tree *tree;
    const double *table;
    int nodes, cur;                            // the refused are the children of cur (-1: none are)

    __device__ __forceinline__ void eight_at(i64 at, double (&r)[EIGHT]) const {
        of(at, eight<DT>(x, at, v), a > 0 ? eight<DT>(y, at, v) : Entries<DT>{}, r);
    }
    __device__ __forceinline__ void of(i64 at, const Entries<DT> &e, const Entries<DT> &f, double (&r)[EIGHT]) const {
        exponentials<DT>(table, scale, e, p.most, r);
#pragma unroll
        for (int i = 0; i < EIGHT; ++i) r[i] = probability(r[i], p.per_z);
        if (a > 0) {
            const double per = a * q.per_z;
            double o[EIGHT];
            exponentials<DT>(table, scale, f, q.most, o);
#pragma unroll
            for (int i = 0; i < EIGHT; ++i) r[i] = fmax(r[i] - o[i] * per, 0.0);
        }
        if (cur >= 0) {
            for (int j = 1; j < nodes; ++j) {
                const i64 place = tree->token[j] - at;
                if (tree->parent[j] == cur && place >= 0 && place < EIGHT) {
#pragma unroll
                    for (int i = 0; i < EIGHT; ++i)
                        if (place == i) r[i] = 0;
                }
            }
        }
    }
};

__device__ __forceinline__ int segments_of(i64 v) { return (int)((v + 64 * EIGHT - 1) / (64 * EIGHT)); }
// the sum of a segment, 64 times eight entries, by a wavefront
template <int DT>
__device__ __forceinline__ double sum_segment(const Left<DT> &left, int segment) {
    double r[EIGHT], sum = 0;
    left.eight_at((i64)(segment * 64 + (int)(threadIdx.x & 63)) * EIGHT, r);
#pragma unroll
    for (int i = 0; i < EIGHT; ++i) sum += r[i];
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    return sum;
}

// a wavefront's of what WALK threads add up of a row, with the draft's
template <int DT>
__device__ __forceinline__ double sum_own(const Left<DT> &left) {
    i64 at = (i64)threadIdx.x * EIGHT;
    Entries<DT> e = first_eight<DT>(left.x, at, left.v), f = first_eight<DT>(left.y, at, left.v);
    double sum = 0;
    const double ratio = left.a * left.q.per_z / left.p.per_z;
    auto add = [&](const Entries<DT> &e, const Entries<DT> &f) __attribute__((always_inline)) { add_left<DT>(left.table, left.scale, e, f, left.p.most, left.q.most, ratio, sum); };
    while (at + EIGHT <= left.v) {
        const i64 next = at + WALK * EIGHT;
        const Entries<DT> e_ahead = first_eight<DT>(left.x, next, left.v), f_ahead = first_eight<DT>(left.y, next, left.v);
        add(e, f);
        e = e_ahead, f = f_ahead, at = next;
    }
    if (at < left.v) add(eight<DT>(left.x, at, left.v), eight<DT>(left.y, at, left.v));
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    return sum * left.p.per_z;
}

// the smallest j with R(0) + ... + R(j) > u sum(R); by a wavefront, from the sums of the segments
template <int DT>
__device__ int find_left(const double *segment_sums, const Left<DT> &left, double u, double *total) {
    const int lane = threadIdx.x & 63, segments = segments_of(left.v), each = (segments + 63) / 64;
    double own = 0;
    for (int s = lane * each; s < min(segments, (lane + 1) * each); ++s) own += segment_sums[s];
    double sum = sum_up_to(own);
    *total = __shfl(sum, 63);
    const double threshold = u * *total;
    int at = first_above(sum, own, threshold);
    if (at < 0) return -1;
    double before = __shfl(sum, max(at - 1, 0));
    if (at == 0) before = 0;
    int segment = -1;
    double base = 0;                           // what lies in front of the segment
    for (int s = at * each; s < min(segments, (at + 1) * each); ++s) {               // the same for all lanes
        const double here = segment_sums[s];
        if (here > 0) {
            segment = s, base = before;
            if (before + here > threshold) break;
        }
        before += here;
    }
    if (segment < 0) return -1;
    double r[EIGHT];
    own = 0;
    left.eight_at((i64)(segment * 64 + lane) * EIGHT, r);
#pragma unroll
    for (int i = 0; i < EIGHT; ++i) own += r[i];
    sum = base + sum_up_to(own);
    at = first_above(sum, own, threshold);
    if (at < 0) return -1;
    double here = __shfl(sum, max(at - 1, 0));
    if (at == 0) here = base;
    int j = -1;
    bool done = false;
#pragma unroll
    for (int i = 0; i < EIGHT; ++i) {
        if (!done && r[i] > 0) j = i;
        here += r[i];
        done |= r[i] > 0 && here > threshold;
    }
    return __shfl(j < 0 ? -1 : (segment * 64 + lane) * EIGHT + j, at);
}

// The largest entry and the sum of a row of its slices', by a wavefront
__device__ __forceinline__ Row join(const double *table, const Scale &S, const Part *parts, int slices) {
    const int lane = threadIdx.x & 63;
    Part p = {0.0, -INFINITY, 0.0f};
    if (lane < slices) p = parts[lane];
    const bool bad = __ballot(!(p.most == p.most)) != 0;
    float most = p.most;
#pragma unroll
    for (int d = 32; d; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
    if (bad || !(most > -INFINITY)) return {0.0, 0.0};
    double z = p.most > -INFINITY ? p.z * exp2_64(table, S, (double)p.most - (double)most) : 0.0;
#pragma unroll
    for (int d = 32; d; d >>= 1) z += __shfl_xor(z, d);
    return {(double)most, 1.0 / z};
}

// The sum behind a first refusal, max(p - q, 0), where another child is tried behind it.
template <int DT>
__global__ __launch_bounds__(BLOCK) void k_first(Job A) {
    typedef typename type<DT>::t T;
    __shared__ double sum_of[BLOCK / 64], table[STEPS];
    // neighbours in the launch are nodes of one number in different trees, as far as these are alike: first nodes have more children, and what has to be done lies evenly (64 trees of 16: 23 us, 30 in
    // the order of the rows)
    const int turn = blockIdx.x / A.firsts, slice = (int)(blockIdx.x % A.firsts);
    const i64 row = (i64)(turn % A.sequences) * A.apart + turn / A.sequences;
    if (row >= A.n) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    const T *x = (const T *)A.x[0] + row * A.ld[0], *y = (const T *)A.x[1] + row * A.ld[1];
    i64 at = ((i64)slice * BLOCK + threadIdx.x) * EIGHT;
    if (children(A, row) < 2) return;
    Entries<DT> e = first_eight<DT>(x, at, A.v), f = first_eight<DT>(y, at, A.v);
    take_table(table);
    __syncthreads();
    const Row p = join(table, A.scale, A.parts + row * A.slices, A.slices), q = join(table, A.scale, A.parts + (A.n + row) * A.slices, A.slices);
    double sum = 0;
    const double ratio = q.per_z / p.per_z;
    auto add = [&](const Entries<DT> &e, const Entries<DT> &f) __attribute__((always_inline)) { add_left<DT>(table, A.scale, e, f, p.most, q.most, ratio, sum); };
    while (at + EIGHT <= A.v) {
        const i64 next = at + (i64)A.firsts * (BLOCK * EIGHT);
        const Entries<DT> e_ahead = first_eight<DT>(x, next, A.v), f_ahead = first_eight<DT>(y, next, A.v);
        add(e, f);
        e = e_ahead, f = f_ahead, at = next;
    }
    if (at < A.v) add(eight<DT>(x, at, A.v), eight<DT>(y, at, A.v));
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if (lane == 0) sum_of[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) A.first[row * A.firsts + slice] = ((sum_of[0] + sum_of[1]) + (sum_of[2] + sum_of[3])) * p.per_z;
}

template <int DT>
__global__ __launch_bounds__(WALK) void k_walk(Job A) {
    typedef typename type<DT>::t T;
    __shared__ Shared sh;
    const int b = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t / 64;
    i64 s0;
    const int nodes = take_tree<WALK>(A, b, sh.tree, &s0);
    take_table(sh.table);
    __syncthreads();
    for (int d = t; d < A.depth; d += WALK) A.nodes[(i64)b * A.depth + d] = -1;
    for (int d = t; d <= A.depth; d += WALK) A.out[(i64)b * (A.depth + 1) + d] = -1;
    for (int r = wave; r < nodes * (A.drafted ? 2 : 1); r += WALK / 64) {
        const i64 row = r < nodes ? s0 + r : A.n + s0 + r - nodes;
        const Row joined = join(sh.table, A.scale, A.parts + row * A.slices, A.slices);
        if (lane == 0) A.rows[row] = joined;
    }
    __syncthreads();
    for (int i = t; i < nodes; i += WALK) {
        const int parent = sh.tree.parent[i], token = sh.tree.token[i];
        sh.u[i] = A.uniforms[s0 + i];
        sh.have[i] = sh.said[i] = 0;
        if (parent >= 0) {
            auto of = [&](int which) {
                const Row r = A.rows[(which ? A.n : 0) + s0 + parent];
                if (r.per_z == 0) return 0.0;
                return probability(exp2_64(sh.table, A.scale, (double)(float)((const T *)A.x[which])[(s0 + parent) * A.ld[which] + token] - r.most), r.per_z);
            };
            sh.have[i] = of(0);
            sh.said[i] = A.drafted ? of(1) : 1.0;
        }
    }
    __syncthreads();
    // from here on all threads do the same
    Left<DT> left = {};
    left.scale = A.scale, left.v = A.v, left.tree = &sh.tree, left.table = sh.table, left.nodes = nodes;
    int cur = 0, count = 0, refusals = 0;
    auto stand_at = [&](int node) {
        cur = node, left.a = 0, left.cur = -1, refusals = 0;
        if (node < nodes) {
            left.x = (const T *)A.x[0] + (s0 + node) * A.ld[0], left.p = A.rows[s0 + node];
            if (A.drafted) left.y = (const T *)A.x[1] + (s0 + node) * A.ld[1], left.q = A.rows[A.n + s0 + node];
        }
    };
    stand_at(0);
    auto sum_of_waves = [&](double own) {
        __syncthreads();
        if (lane == 0) sh.sums[wave] = own;
        __syncthreads();
        double sum = 0;
        for (int k = 0; k < WALK / 64; ++k) sum += sh.sums[k];
        return sum;
    };
    double w = 1;                              // the sum of what is left
    for (int i = 1; i < nodes; ++i) {
        if (sh.tree.parent[i] != cur || count == A.depth || left.p.per_z == 0 || (A.drafted && left.q.per_z == 0)) continue;
        double have = sh.have[i];
        if (!A.drafted) {
            for (int j = 1; j < i; ++j)
                if (sh.tree.parent[j] == cur && sh.tree.token[j] == sh.tree.token[i]) have = 0;        // refused before
            // w is one without the refused, whose sum is CLOSE to right: summed anew where that might decide
            if (left.cur >= 0 && have > 0 && fabs(sh.u[i] * w - have) <= CLOSE) {
                left.nodes = i;
                w = 0;
                for (int s = wave; s < segments_of(A.v); s += WALK / 64) w += sum_segment(left, s);
                w = sum_of_waves(w);
            }
        } else if (refusals) {
            if (refusals == 1) {
                w = 0;
                for (int k = 0; k < A.firsts; ++k) w += A.first[(s0 + cur) * A.firsts + k];
            } else {
                w = sum_of_waves(sum_own(left));
            }
            have = fmax(have - left.a * sh.said[i], 0.0);
        }
        if (sh.u[i] * sh.said[i] * w < have) {
            if (t == 0) {
                A.nodes[(i64)b * A.depth + count] = i;
                A.out[(i64)b * (A.depth + 1) + count] = sh.tree.token[i];
            }
            ++count;
            stand_at(i);
            w = 1;
        } else if (A.drafted) {
            left.a += w;
            ++refusals;
        } else {
            w -= have;
            left.cur = cur;
        }
    }
    if (t == 0) {
        A.counts[b] = count;
        A.ends[b] = {left.a, nodes > 0 && left.p.per_z != 0 ? s0 + cur : -1, cur, left.cur >= 0, count, 0};
    }
}

// what is left at the end of a sequence's path
template <int DT, int THREADS>
__device__ __forceinline__ Left<DT> left_at(const Job &A, int b, const End &end, Tree &tree, double *table) {
    typedef typename type<DT>::t T;
    Left<DT> left = {};
    left.scale = A.scale, left.v = A.v, left.tree = &tree, left.table = table, left.a = end.a, left.cur = end.refused ? end.node : -1;
    take_table(table);
    if (end.refused) {
        i64 s0;
        left.nodes = take_tree<THREADS>(A, b, tree, &s0);
    }
    __syncthreads();
    left.x = (const T *)A.x[0] + end.row * A.ld[0], left.p = A.rows[end.row];
    if (A.drafted) left.y = (const T *)A.x[1] + end.row * A.ld[1], left.q = A.rows[A.n + end.row];
    return left;
}

template <int DT>
__global__ __launch_bounds__(BLOCK) void k_left(Job A) {
    __shared__ Tree tree;
    __shared__ double table[STEPS];
    const int groups = (segments_of(A.v) + BLOCK / 64 - 1) / (BLOCK / 64), b = (int)(blockIdx.x / groups), segment = (int)(blockIdx.x % groups) * (BLOCK / 64) + (int)threadIdx.x / 64;
    const End end = A.ends[b];
    if (end.row < 0) return;
    const Left<DT> left = left_at<DT, BLOCK>(A, b, end, tree, table);
    if (segment >= segments_of(A.v)) return;
    const double sum = sum_segment(left, segment);
    if ((threadIdx.x & 63) == 0) A.segments[(i64)b * segments_of(A.v) + segment] = sum;
}

template <int DT>
__global__ __launch_bounds__(64) void k_pick(Job A) {
    __shared__ Tree tree;
    __shared__ double table[STEPS];
    const int b = blockIdx.x;
    const End end = A.ends[b];
    if (end.row < 0) return;                   // -1 is there
    Left<DT> left = left_at<DT, 64>(A, b, end, tree, table);
    double *segments = A.segments + (i64)b * segments_of(A.v), total;
    const double u = A.uniforms[max((i64)0, (i64)A.starts[b])];
    int last = find_left(segments, left, u, &total);
    if (!(total > 0)) {                        // nothing: of the target's probabilities
        left.a = 0, left.cur = -1;
        for (int s = 0; s < segments_of(A.v); ++s) {
            const double sum = sum_segment(left, s);
            if (threadIdx.x == 0) segments[s] = sum;
        }
        __syncthreads();
        last = find_left(segments, left, u, &total);
    }
    if (threadIdx.x == 0) A.out[(i64)b * (A.depth + 1) + end.count] = last;
}

// Entries of a slice of a row: as many as leave 8192 workgroups, 2048 at least, and 64 slices at most
i64 per_slice_of(int64_t v, int64_t rows) {
    const i64 at_once = BLOCK * EIGHT, all = (v + at_once - 1) / at_once, slices = min(min(all, (i64)64), max((i64)1, 8192 / max(rows, (i64)1)));
    return (all + slices - 1) / slices * at_once;
}
i64 slices_of(int64_t v, int64_t rows) { return (v + per_slice_of(v, rows) - 1) / per_slice_of(v, rows); }
// slices of a sum behind a first refusal: its rows are some of the nodes'
i64 firsts_of(int64_t v, int64_t n) { return min((v + BLOCK * EIGHT - 1) / (BLOCK * EIGHT), max((i64)4, min((i64)16, 4096 / max(n, (i64)1)))); }

// ---- the path's entries -------------------------------------------------------------------------------------------
// A thread moves one place of all entries of a path.  64 paths of up to eight entries in 256 heads of 128 columns and 8 bits: 14 us, of which reading and writing the rows,
// 128 bytes each in pages of their own, would be 7; a path in 8 heads 4.7: a load behind the other, of numbers, page and entry.
struct Keep {
    Cache cache;
    Batch batch;
    const i64 *nodes, *counts;
    int depth;
    int *lengths;
};

__global__ __launch_bounds__(BLOCK) void k_keep(Keep A) {
    struct Move {
        i64 from_page, to_page;
        int from_row, to_row, fine;
    };
    __shared__ int node[MAX_DEPTH];
    __shared__ Move moves[MAX_DEPTH];
    __shared__ int path;
    const int b = blockIdx.x, t = threadIdx.x, heads = (int)A.cache.heads;
    const int nodes = max(A.batch.starts[b + 1] - A.batch.starts[b], 0);
    const i64 length = A.batch.lengths[b], first = length - nodes;
    const int count = (int)max((i64)0, min(A.counts[b], (i64)A.depth));
    for (int d = t; d < count; d += BLOCK) node[d] = (int)max((i64)0, min(A.nodes[(i64)b * A.depth + d], (i64)0x7FFFFFFF));
    __syncthreads();
    if (t == 0) {
        int d = 0;
        for (int before = 0; d < count && node[d] > before && node[d] < nodes; ++d) before = node[d];
        path = d;
        if (blockIdx.y == 0) A.lengths[b] = (int)max((i64)0, nodes ? first + 1 + d : length);
    }
    __syncthreads();
    const int n = path;
    for (int d = t; d < n; d += BLOCK) {
        Move m = {0, 0, 0, 0, 0};
        m.fine = node[d] != d + 1 && find_entry(A.cache, A.batch, b, first + node[d], &m.from_page, &m.from_row) &&
                 find_entry(A.cache, A.batch, b, first + d + 1, &m.to_page, &m.to_row);
        moves[d] = m;
    }
    __syncthreads();
    // A thread has one place in all entries of the path: 16 bytes of a head's, or a scale.  Numbers rise, so that an entry never comes from where an
    // earlier one went: eight are read before the first is written.
    const int units = A.cache.dim * A.cache.size / 16, all = heads * 2 * units;
    const int item = (int)blockIdx.y * BLOCK + t;
    if (item < all) {
        typedef u32 v4u __attribute__((ext_vector_type(4)));
        const Half &h = A.cache.half[item / (heads * units)];
        const int head = item / units % heads;
        char *at = h.at + head * h.head + item % units * 16;
        for (int d = 0; d < n; d += 8) {
            v4u v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (d + i < n && moves[d + i].fine) v[i] = *(const v4u *)(at + moves[d + i].from_page * h.page + moves[d + i].from_row * h.row);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (d + i < n && moves[d + i].fine) *(v4u *)(at + moves[d + i].to_page * h.page + moves[d + i].to_row * h.row) = v[i];
        }
    } else if (A.cache.dtype == VI_I8 && item < all + 2 * heads) {
        const Half &h = A.cache.half[(item - all) / heads];
        float *at = h.scales + (item - all) % heads * h.scale_head;
        for (int d = 0; d < n; d += 8) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (d + i < n && moves[d + i].fine) v[i] = at[moves[d + i].from_page * h.scale_page + moves[d + i].from_row];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (d + i < n && moves[d + i].fine) at[moves[d + i].to_page * h.scale_page + moves[d + i].to_row] = v[i];
        }
    }
}

}  // namespace

extern "C" size_t vi_verify_drafts_workspace_bytes(int dtype, int64_t n, int64_t v, int64_t sequences, int drafted) {
    if (!is_float(dtype) || n < 0 || n > MAX_BLOCKS || v <= 0 || v > MAX_V || sequences < 0 || sequences > 0xFFFFFF) return 0;
    const i64 rows = drafted ? 2 * n : n, slices = slices_of(v, rows);
    return (size_t)(2 * n) * sizeof(Row) + (size_t)(rows * slices) * sizeof(Part) + (size_t)sequences * (sizeof(End) + 8 * ((v + 64 * EIGHT - 1) / (64 * EIGHT))) +
           (drafted ? (size_t)(n * firsts_of(v, n)) * 8 : 0) + vi::WS_SLACK;
}

extern "C" int vi_verify_drafts(int dtype, const void *logits, int64_t n, int64_t v, int64_t ld, const void *draft, int64_t ld_draft, const int64_t *tokens,
                                const int32_t *starts, int64_t sequences, const int32_t *parents, const double *uniforms, double temperature, int64_t depth,
                                int64_t *counts, int64_t *nodes, int64_t *out, void *ws, size_t ws_bytes, void *stream) {
    const char *who = "vi_verify_drafts";
    if (!is_float(dtype)) return vi::fail(VI_EINVAL, "%s: dtype %d is none of VI_F32, VI_BF16, VI_F16", who, dtype);
    if (n < 0 || n > MAX_BLOCKS || v < 1 || v > MAX_V) return vi::fail(VI_EINVAL, "%s: %lld rows of %lld logits (1 to %lld)", who, (long long)n, (long long)v, (long long)MAX_V);
    if (ld < v || (draft && ld_draft < v)) return vi::fail(VI_EINVAL, "%s: rows of %lld logits %lld apart", who, (long long)v, (long long)(ld < v ? ld : ld_draft));
    if (sequences < 0 || sequences > 0xFFFFFF) return vi::fail(VI_EINVAL, "%s: %lld sequences", who, (long long)sequences);
    if (depth < 0 || depth > MAX_DEPTH) return vi::fail(VI_EINVAL, "%s: a depth of %lld (%d at most)", who, (long long)depth, MAX_DEPTH);
    if (!(temperature >= 1e-3 && temperature <= 1e3)) return vi::fail(VI_EINVAL, "%s: temperature %g", who, temperature);
    if (sequences == 0) return VI_OK;
    if (!starts || !counts || !out || (depth && !nodes) || (n && (!logits || !tokens || !uniforms))) return vi::fail(VI_EINVAL, "%s: null pointer", who);
    const i64 rows = draft ? 2 * n : n, segments = (v + 64 * EIGHT - 1) / (64 * EIGHT), groups = (segments + BLOCK / 64 - 1) / (BLOCK / 64);
    if (rows * slices_of(v, rows) > MAX_BLOCKS || sequences * groups > MAX_BLOCKS || (n + sequences) * firsts_of(v, n) > MAX_BLOCKS)
        return vi::fail(VI_EINVAL, "%s: %lld rows of %lld logits, %lld sequences", who, (long long)n, (long long)v, (long long)sequences);
    const size_t need = vi_verify_drafts_workspace_bytes(dtype, n, v, sequences, draft != nullptr);
    if (ws_bytes < need || !ws) return vi::fail(VI_ENOMEM, "%s: workspace %zu < %zu bytes", who, ws_bytes, need);
    const hipStream_t s = (hipStream_t)stream;
    Job J = {};
    J.x[0] = logits, J.x[1] = draft, J.ld[0] = ld, J.ld[1] = ld_draft, J.n = n, J.v = v, J.slices = (int)slices_of(v, rows), J.per_slice = (int)per_slice_of(v, rows), J.firsts = (int)firsts_of(v, n), J.sequences = (int)sequences;
    J.apart = (int)((n + sequences - 1) / sequences), J.depth = (int)depth, J.drafted = draft != nullptr, J.scale.c = STEPS * 1.4426950408889634 / temperature, J.scale.deepest = DEEPEST / J.scale.c, J.tokens = tokens, J.starts = starts, J.parents = parents;
    J.uniforms = uniforms, J.counts = counts, J.nodes = nodes, J.out = out;
    J.rows = (Row *)vi::align16(ws);
    J.parts = (Part *)(J.rows + 2 * n);
    J.ends = (End *)(J.parts + rows * J.slices);
    J.segments = (double *)(J.ends + sequences);
    J.first = J.segments + sequences * segments;
    const dim3 of_rows((unsigned)(rows * J.slices)), of_nodes((unsigned)((i64)J.apart * sequences * J.firsts)), of_groups((unsigned)(sequences * groups)), of_sequences((unsigned)sequences);
#define GO(TYPE)                                                                                    \
    do {                                                                                            \
        constexpr int DT = TYPE;                                                                    \
        if (n) hipLaunchKernelGGL(k_stats<DT>, of_rows, dim3(BLOCK), 0, s, J);                      \
        VI_LAUNCH_CHECK(who);                                                                       \
        if (n && draft && parents) hipLaunchKernelGGL(k_first<DT>, of_nodes, dim3(BLOCK), 0, s, J); \
        VI_LAUNCH_CHECK(who);                                                                       \
        hipLaunchKernelGGL(k_walk<DT>, of_sequences, dim3(WALK), 0, s, J);                          \
        VI_LAUNCH_CHECK(who);                                                                       \
        hipLaunchKernelGGL(k_left<DT>, of_groups, dim3(BLOCK), 0, s, J);                            \
        VI_LAUNCH_CHECK(who);                                                                       \
        hipLaunchKernelGGL(k_pick<DT>, of_sequences, dim3(64), 0, s, J);                            \
        VI_LAUNCH_CHECK(who);                                                                       \
    } while (0)
    if (dtype == VI_F32) GO(VI_F32);
    if (dtype == VI_BF16) GO(VI_BF16);
    if (dtype == VI_F16) GO(VI_F16);
#undef GO
    return VI_OK;
}

extern "C" int vi_keep_drafts(const vi_cache *cache, const vi_batch *batch, const int64_t *nodes, int64_t depth, const int64_t *counts, int32_t *lengths,
                              void *stream) {
    const char *who = "vi_keep_drafts";
    Keep A = {};
    if (const int rc = take(who, cache, batch, &A.cache, &A.batch)) return rc;
    if (depth < 0 || depth > MAX_DEPTH) return vi::fail(VI_EINVAL, "%s: a depth of %lld (%d at most)", who, (long long)depth, MAX_DEPTH);
    if (batch->sequences == 0) return VI_OK;
    if (!counts || !lengths || (depth && !nodes)) return vi::fail(VI_EINVAL, "%s: null pointer", who);
    if (lengths == batch->lengths) return vi::fail(VI_EINVAL, "%s: the new lengths in the place of the old", who);
    A.nodes = nodes, A.counts = counts, A.depth = (int)depth, A.lengths = lengths;
    const i64 items = (i64)cache->heads * 2 * (cache->dim * A.cache.size / 16) + (cache->dtype == VI_I8 ? 2 * cache->heads : 0);
    if (items / BLOCK >= 65535) return vi::fail(VI_EINVAL, "%s: %lld heads", who, (long long)cache->heads);
    hipLaunchKernelGGL(k_keep, dim3((unsigned)batch->sequences, (unsigned)((items + BLOCK - 1) / BLOCK)), dim3(BLOCK), 0, (hipStream_t)stream, A);
    VI_LAUNCH_CHECK(who);
    return VI_OK;
}
