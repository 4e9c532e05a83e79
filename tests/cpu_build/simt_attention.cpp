// Attention over the cache (verinf_amd/csrc/attention.hip) on the CPU, launches and all; with any form and cut of the keys, which the library chooses by size.
#include "simt_generation.hpp"
#include "attention.hip"
extern "C" const char *simt_error() { return vi::err_buf(); }

// form 0: a wavefront's own keys, 1: shared ones
extern "C" int simt_attend(int form, int splits, int per_split, const vi_cache *cache, const vi_batch *batch, int dtype, const void *q, int64_t n, int64_t heads, int64_t q_token,
                           int64_t q_head, const int32_t *parents, float scale, void *out, float *ws) {
    Args A = {};
    if (const int rc = take("simt", cache, batch, &A.cache, &A.batch)) return rc;
    const int rows = form ? 128 : 32;
    A.q = q, A.out = out, A.q_token = q_token, A.q_head = q_head, A.out_token = heads * cache->dim, A.out_head = cache->dim, A.n = n, A.parents = parents;
    A.heads = (int)heads, A.group = (int)(heads / cache->heads), A.tiles = (int)(n * A.group / rows + batch->sequences), A.splits = splits, A.per_split = per_split;
    A.clear = 1, A.c = scale * 1.44269504f;
    const int dp = cache->dim <= 64 ? 64 : cache->dim <= 128 ? 128 : 256;
    A.part = ws, A.most = ws + (i64)A.tiles * cache->heads * splits * rows * dp;
    Plan L = {};
    L.form = form, L.dp = dp;
    if (cache->dtype == VI_I8) launch_columns<VI_BF16, true>(L, A, nullptr);
    if (cache->dtype == VI_BF16) launch_columns<VI_BF16, false>(L, A, nullptr);
    if (cache->dtype == VI_F16) launch_columns<VI_F16, false>(L, A, nullptr);
    (void)dtype;
    simt::no_pieces();
    return VI_OK;
}
extern "C" int64_t simt_ws_floats(int form, int splits, int64_t n, int64_t heads, int64_t cache_heads, int64_t sequences, int64_t dim) {
    const int rows = form ? 128 : 32, dp = dim <= 64 ? 64 : dim <= 128 ? 128 : 256;
    return (n * (heads / cache_heads) / rows + sequences) * cache_heads * splits * rows * (dp + 2);
}
