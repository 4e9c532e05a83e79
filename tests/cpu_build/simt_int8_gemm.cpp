// Products of 8-bit integers (verinf_amd/csrc/int8_gemm.hip) on the CPU, launches and all; with any tile, number of slices and copy of the
// operands, which the library chooses by size.
#include "simt_inference.hpp"
#include "int8_gemm.hip"
extern "C" const char *simt_error() { return vi::err_buf(); }
extern "C" int simt_tiles() { return N_TILES; }
// the tile (N_TILES: few rows) of a call, and its slices and copy
extern "C" void simt_plan(int64_t m, int64_t k, int64_t n, int gated, int aligned, int *out) {
    const Plan L = make_plan(m, k, n, gated, aligned, true);
    out[0] = L.tile, out[1] = L.slices, out[2] = L.pack;
}

static Plan forced(int tile, int slices, int pack, i64 m, i64 k, i64 n, bool gated) {
    Plan L = {};
    L.tile = tile;
    if (tile == FEW) return L;
    const Tile &T = TILES[tile];
    const i64 rows = 64 * T.wm, cols = (gated ? 32 : 64) * T.wn, step = 16 * T.units;
    L.pack = pack, L.mt = (int)((m + rows - 1) / rows), L.nt = (int)((n + cols - 1) / cols), L.steps = (int)((k + step - 1) / step);
    L.steps_per_slice = (L.steps + slices - 1) / slices;
    if (T.units == 4) L.steps_per_slice += L.steps_per_slice & 1;
    L.slices = L.steps ? (L.steps + L.steps_per_slice - 1) / L.steps_per_slice : 1;
    if (pack) L.pack_bytes = (size_t)whole_lines(k) * (m + (gated ? 2 : 1) * n);
    L.ws_bytes = L.pack_bytes + (L.slices > 1 ? (size_t)4 * L.slices * (gated ? 2 : 1) * m * n : 0) + vi::WS_SLACK;
    return L;
}
extern "C" size_t simt_workspace(int gated, int tile, int slices, int pack, int64_t m, int64_t k, int64_t n) { return forced(tile, slices, pack, m, k, n, gated).ws_bytes; }
extern "C" int simt_product(int gated, int tile, int slices, int pack, const int8_t *a, int64_t lda, const int8_t *b, int64_t ldb, const int8_t *b2, int64_t ldb2, int64_t m,
                            int64_t k, int64_t n, const float *a_scale, const float *b_scale, const float *b2_scale, const float *bias, int act, int dtype, void *out, void *ws) {
    Job J = {};
    J.a = (const signed char *)a, J.b = (const signed char *)b, J.b2 = (const signed char *)b2, J.lda = lda, J.ldb = ldb, J.ldb2 = ldb2, J.m = m, J.k = k, J.n = n;
    J.a_scale = a_scale, J.b_scale = b_scale, J.b2_scale = b2_scale, J.bias = bias, J.act = act, J.dtype = dtype, J.out = out, J.ldo = n;
    const bool aligned = aligned_rows(J.a, J.lda) && aligned_rows(J.b, J.ldb) && (!gated || aligned_rows(J.b2, J.ldb2));
    const Plan L = forced(tile, slices, pack, m, k, n, gated);
    const int rc = gated ? run<true>("simt", L, J, aligned, ws, nullptr) : run<false>("simt", L, J, aligned, ws, nullptr);
    simt::none_under_way();
    return rc;
}
