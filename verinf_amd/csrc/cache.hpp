// The paged cache of keys and values, as the kernels that write, read and move its entries see it.
#pragma once

#include "number_types.hpp"

namespace kv {

using namespace num;

struct Half {                                  // the keys, or the values
    char *at;
    float *scales;
    i64 page, head, row;                       // bytes apart
    i64 scale_page, scale_head;                // floats apart
};
struct Cache {
    Half half[2];
    i64 pages, heads;
    int shift, mask;                           // of the number of an entry: its page in the sequence, its row in the page
    int dim, size;                             // numbers of an entry, bytes of one
    int dtype;
};
struct Batch {
    const int *starts, *lengths, *pages;
    i64 stride;
    int sequences;
    i64 most;                                  // entries that a row of `pages` can name
};

// Where entry j of sequence b lies: false where no page of the cache holds it
__device__ __forceinline__ bool find_entry(const Cache &c, const Batch &t, int b, i64 j, i64 *page, int *row) {
    if (j < 0 || j >= t.most) return false;
    *page = t.pages[b * t.stride + (j >> c.shift)];
    *row = (int)(j & c.mask);
    return *page >= 0 && *page < c.pages;
}

// The sequence that a row of the new tokens belongs to, by a wavefront, all of whose lanes ask for the same row: -1, none
__device__ __forceinline__ int find_sequence(const Batch &t, i64 row) {
    int count = 0;
    for (int first = 0; first < t.sequences; first += 64) {
        const int b = first + (int)(threadIdx.x & 63);
        count += __popcll(__ballot(b < t.sequences && t.starts[min(b, t.sequences)] <= row));
    }
    const int b = count - 1;
    return b >= 0 && t.starts[b] <= row && row < t.starts[b + 1] ? b : -1;
}

inline int size_of_entry(int dtype) { return dtype == VI_I8 ? 1 : 2; }

// What is wrong with a cache or batch, and both as the kernels take them
inline int take(const char *who, const vi_cache *c, const vi_batch *b, Cache *to, Batch *t) {
    if (!c || !b) return vi::fail(VI_EINVAL, "%s: null pointer", who);
    if (c->dtype != VI_BF16 && c->dtype != VI_F16 && c->dtype != VI_I8) return vi::fail(VI_EINVAL, "%s: a cache of dtype %lld", who, (long long)c->dtype);
    if (c->dim < 16 || c->dim > 256 || c->dim % 16) return vi::fail(VI_EINVAL, "%s: heads of %lld numbers (multiples of 16 up to 256)", who, (long long)c->dim);
    if (c->page_size < 16 || c->page_size > 1024 || !vi::is_pow2(c->page_size))
        return vi::fail(VI_EINVAL, "%s: pages of %lld entries (powers of two from 16 to 1024)", who, (long long)c->page_size);
    if (c->pages < 0 || c->pages > 0x7FFFFFFF || c->heads < 1 || c->heads > 0xFFFF) return vi::fail(VI_EINVAL, "%s: %lld pages of %lld heads", who, (long long)c->pages, (long long)c->heads);
    if (b->sequences < 0 || b->sequences > 0xFFFFFF || b->width < 0 || b->width > (1 << 30) / c->page_size || (b->sequences > 1 && b->stride < b->width))
        return vi::fail(VI_EINVAL, "%s: %lld sequences of %lld pages", who, (long long)b->sequences, (long long)b->width);
    if (!b->starts || (b->sequences && (!b->lengths || (b->width && !b->pages)))) return vi::fail(VI_EINVAL, "%s: null pointer", who);
    if (c->pages && (!c->keys || !c->values || (c->dtype == VI_I8 && (!c->key_scales || !c->value_scales)))) return vi::fail(VI_EINVAL, "%s: null pointer", who);
    const int size = size_of_entry((int)c->dtype);
    for (int h = 0; h < 2; ++h) {
        const int64_t *s = h ? c->value_strides : c->key_strides, *e = h ? c->value_scale_strides : c->key_scale_strides;
        const uintptr_t at = (uintptr_t)(h ? c->values : c->keys);
        if ((at | s[0] * size | s[1] * size | s[2] * size) & 15) return vi::fail(VI_EINVAL, "%s: a cache whose entries do not start at multiples of 16 bytes", who);
        // an entry's place in its page is taken in 32 bits
        if (s[0] < 0 || s[1] < 0 || s[2] < 0 || s[2] > (1 << 20) || s[0] * size >= (1ll << 32))
            return vi::fail(VI_EINVAL, "%s: a cache of pages %lld, entries %lld apart", who, (long long)s[0], (long long)s[2]);
        to->half[h] = {(char *)at, h ? c->value_scales : c->key_scales, s[0] * size, s[1] * size, s[2] * size, e[0], e[1]};
    }
    to->pages = c->pages, to->heads = c->heads, to->shift = vi::ilog2(c->page_size), to->mask = (int)c->page_size - 1;
    to->dim = (int)c->dim, to->size = size, to->dtype = (int)c->dtype;
    *t = {b->starts, b->lengths, b->pages, b->stride, (int)b->sequences, b->width * c->page_size};
    return VI_OK;
}

}  // namespace kv
