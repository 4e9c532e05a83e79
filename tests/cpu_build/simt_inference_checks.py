"""The kernels of the forward pass in 8-bit integers on the CPU (simt_inference.hpp), against 64-bit results, as a program of its own: the
test runs it under AddressSanitizer, where every numpy array is a heap block of exactly its size."""
import ctypes
import json
import math
import os
import sys

import numpy as np

I64, VP, SZ, INT, F32 = ctypes.c_int64, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_float
FLOATS = {0: "float32", 1: "bfloat16", 2: "float16"}
LOWEST = {0: float(np.finfo(np.float32).min), 1: -float(np.array(0x7F7F0000, dtype=np.uint32).view(np.float32)), 2: -65504.0}


def ptr(a):
    return a.ctypes.data if a is not None and a.size else None


def encode(x, kind):
    """float32 values as numbers of the type, which they fit or are rounded to, half to even"""
    x = np.ascontiguousarray(x, dtype=np.float32)
    if kind == 0:
        return x.copy()
    if kind == 2:
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    u = x.view(np.uint32)
    return np.where(np.isnan(x), 0x7FC0, (u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def decode(a, kind):
    if kind == 1:
        return (a.astype(np.uint32) << 16).view(np.float32)
    return a.astype(np.float32)


def strided(a, pad, shift=0):
    """The rows of a with `pad` elements of something else behind each, nothing behind the last; a view and how far they are apart."""
    m, k = a.shape
    n = shift + (m - 1) * (k + pad) + k
    others = []
    for lead in (0, 8) * 50:                                   # bytes: the first element is at a multiple of 16 bytes, but for the shift
        flat = np.full(n + lead // a.itemsize, 77, dtype=a.dtype)
        others.append(flat)
        if (flat.ctypes.data + lead) % 16 == 0:
            break
    flat = flat[lead // a.itemsize:]
    view = np.lib.stride_tricks.as_strided(flat[shift:], (m, k), ((k + pad) * a.itemsize, a.itemsize))
    view[:] = a
    return view, k + pad


def scratch(nbytes):
    """nbytes of garbage from an address that is a multiple of 8 only, nothing behind them."""
    return np.full(nbytes + 8, 0xA5, dtype=np.uint8)[8:]


# ---- quantize_rows ------------------------------------------------------------------------------------------------
def quantize(so):
    """Rows in 16 lanes, a wavefront and a workgroup, in one to eight chunks a thread and read twice; ends of one to seven entries; the definition's
    operations one by one in 32 bits."""
    L = ctypes.CDLL(so)
    L.vi_quantize_rows.argtypes = [INT, VP, I64, I64, I64, VP, I64, VP, VP]
    for kind in FLOATS:
        for m, k, pad, shift in ((1, 1, 0, 0), (3, 0, 2, 0), (3, 7, 1, 0), (2, 8, 0, 0), (5, 1000, 3, 0), (2, 2049, 0, 4), (2, 4100, 0, 0), (1, 8191, 0, 0), (2, 11008, 0, 0),
                                 (2, 12289, 1, 0), (1, 16384, 0, 0), (2, 16385, 3, 0), (1, 40001, 0, 4), (1025, 100, 0, 0), (1030, 130, 1, 0), (1024, 256, 0, 4), (2050, 300, 0, 0),
                                 (2048, 1000, 1, 0), (2049, 2047, 0, 0)):
            print("quantize", FLOATS[kind], m, k, pad, shift, flush=True)
            x = (np.random.default_rng(m + k).standard_normal((m, k)) * 5).astype(np.float32)
            if k > 6 and m > 4:
                x[0], x[1], x[2, 3], x[3, k - 1] = 0, -0.0, np.nan, -np.inf
                x[4] = 2.0 ** -118 if kind != 2 else 2.0 ** -24
            a, ldx = strided(encode(x, kind), pad, shift if kind else 0)
            f = decode(a, kind)
            q, scale = np.full((m - 1) * (k + pad) + max(k, 1), 99, np.int8), np.empty(m, np.float32)
            assert L.vi_quantize_rows(kind, a.ctypes.data, m, k, ldx, q.ctypes.data, k + pad, ptr(scale), None) == 0
            with np.errstate(all="ignore"):
                top, finite = np.abs(f).max(axis=1, initial=0), np.isfinite(f).all(axis=1)
                fine = finite & (top >= np.float32(127) * np.float32(2.0 ** -126))
                step = np.where(fine, np.float32(127) / top, np.float32(0)).astype(np.float32)
                want = np.where(fine[:, None], np.rint(f * step[:, None]), 0).astype(np.int8)
                want_scale = np.where(fine, top / np.float32(127), np.where(finite, np.float32(0), np.float32(np.nan)))
            got = np.lib.stride_tricks.as_strided(q, (m, k), (k + pad, 1))
            assert np.array_equal(got, want) and np.array_equal(scale, want_scale.astype(np.float32), equal_nan=True), (FLOATS[kind], m, k)
            for r in range(m - 1):
                assert (q[r * (k + pad) + k:(r + 1) * (k + pad)] == 99).all()


# ---- token_logprobs -----------------------------------------------------------------------------------------------
class Logprobs:
    def __init__(self, so):
        self.L = L = ctypes.CDLL(so)
        L.vi_token_logprobs_workspace_bytes.restype, L.vi_token_logprobs_workspace_bytes.argtypes = SZ, [INT, I64, I64, INT]
        L.vi_token_logprobs.argtypes = [INT, VP, I64, I64, I64, VP, F32, INT, VP, VP, VP, VP, VP, SZ, VP]
        L.simt_error.restype = ctypes.c_char_p
        L.simt_groups_met.restype = ctypes.c_long

    def run(self, x, kind, tokens, top, temperature=1.0, pad=0):
        m, v = x.shape
        rows, ld = strided(x, pad)
        out = [np.empty(m, np.float32), np.empty(m, np.float32), np.empty((m, top), np.float32), np.empty((m, top), np.int64)]
        need = self.L.vi_token_logprobs_workspace_bytes(kind, m, v, top)
        ws = scratch(need)
        before = self.L.simt_groups_met()
        rc = self.L.vi_token_logprobs(kind, rows.ctypes.data, m, v, ld, ptr(tokens), temperature, top, *map(ptr, out), ptr(ws), need, None)
        assert rc == 0, self.L.simt_error()
        self.met = self.L.simt_groups_met() - before
        return out

    def check(self, values, kind, tokens, top, temperature=1.0, pad=0):
        """A logit's distance to the largest is rounded twice (2^-23 of it), e^d with it; up to 128 terms are added one after another and
        their sums pairwise: 2^-24 * 160 of Z, so of log Z, and as much again of each exponential's and the logarithm's own units."""
        x = encode(values, kind)
        got = self.run(x, kind, tokens, top, temperature, pad)
        f = decode(x, kind).astype(np.float64)
        m, v = f.shape
        slack = 2.0 ** -24 * 200
        for i, r in enumerate(f):
            with np.errstate(all="ignore"):
                if np.isnan(r).any() or np.isposinf(r).any():
                    lp, h = np.full(v, np.nan), np.nan
                elif np.isneginf(r).all():
                    lp, h = r, 0.0
                else:
                    d = (r - r.max()) / temperature
                    lp = d - np.log(np.exp(d).sum())
                    h = -(np.exp(lp) * np.where(np.exp(lp) > 0, lp, 0)).sum()
            order = np.lexsort((np.arange(v), np.where(np.isnan(r), -np.inf, -np.where(np.isnan(r), 0, r)), ~np.isnan(r)))[:top]
            assert np.array_equal(got[3][i], order), (FLOATS[kind], m, v, top, i, got[3][i], order)
            t = tokens[i]
            pairs = [(got[0][i], 0.0 if t == -1 else lp[t] if 0 <= t < v else np.nan)] + list(zip(got[2][i], lp[order]))
            for a, b in pairs:
                with np.errstate(all="ignore"):
                    assert a == b or (np.isnan(a) and np.isnan(b)) or abs(a - b) <= slack + 2.0 ** -21 * abs(b), (FLOATS[kind], m, v, top, i, a, b)
            a = got[1][i]
            assert a == h or (np.isnan(a) and np.isnan(h)) or abs(a - h) <= slack * (2 + 2 * np.log(v)), (FLOATS[kind], m, v, top, i, a, h)


def widths(kind):
    """one slice in a workgroup of 256 threads; one in 1024; several, which a second launch joins"""
    return [70, 1000, 3000, 9001, 33001 if kind == 0 else 66001]


def zeros(so):
    """Entries of -0.0 are equal to those of 0.0 and go with them by the lowest index."""
    L = Logprobs(so)
    for kind in FLOATS:
        for v in widths(kind):
            print("zeros", FLOATS[kind], v, flush=True)
            rng = np.random.default_rng(v)
            x = -np.abs(rng.standard_normal((7, v))).astype(np.float32) - 1
            x[0] = -0.0
            x[1] = -0.0
            x[1, v // 2] = 5.0                                 # one positive entry
            x[2, :16], x[2, 64:70] = -0.0, 0.0                 # in front of 0.0
            x[3, 3::64] = -0.0                                 # far apart, among negative ones
            x[4] = -0.0
            x[4, v - 1] = 0.0
            x[5] = -np.inf
            x[5, 5:60:7] = -0.0
            x[6, v - 20:] = -0.0
            tokens = np.array([0, 1, 2, 3, 4, 5, v - 1])
            for top in (1, 3, 20, 64) if v < 3000 else (5,):
                L.check(x, kind, tokens, top)


def far(so):
    """Logits further apart than 32 bits hold, which a temperature brings together."""
    L = Logprobs(so)
    for kind in FLOATS:
        for v in widths(kind):
            print("far", FLOATS[kind], v, flush=True)
            x = np.full((3, v), LOWEST[kind], np.float32)
            x[0, v // 2] = x[1, :5] = -LOWEST[kind]
            x[2, v // 2], x[2, 0] = -LOWEST[kind], 1.0
            for temperature in (2.5, 50.0, 1000.0) if v < 2000 else (50.0,):
                L.check(x, kind, np.array([1, v - 1, 0]), 3, temperature)


def few(so):
    """Rows with fewer allowed entries than are asked for: the rest is filled up, no entries are counted for it.  A workgroup comes to as many
    barriers in every type."""
    L = Logprobs(so)
    for v in (300, 1000, 9001, 30000):
        for allowed in (0, 1, 2, 5):
            print("few", v, allowed, flush=True)
            x = np.full((1, v), -np.inf, np.float32)
            x[0, np.random.default_rng(v).choice(v, allowed, replace=False)] = np.arange(allowed) - 2
            met = []
            for kind in FLOATS:
                L.check(x, kind, np.array([v // 2]), 8)
                met.append(L.met)
            assert met[0] == met[1] == met[2], (v, allowed, met)


def rows(so):
    """Every form of the launch: threads to a row, loads to a thread, one slice and several; ragged ends, rows apart; what is no number."""
    L = Logprobs(so)
    for kind in FLOATS:
        unit = 1024 if kind == 0 else 2048                     # entries that 256 threads load at once
        for m, v, pad, top in ((1, 1, 0, 1), (3, 2, 1, 2), (2, 63, 0, 63), (2, unit, 3, 64), (2, unit + 1, 0, 5), (1, 4 * unit + 1, 0, 5), (1, 9 * unit, 0, 64),
                               (1, 32 * unit, 0, 8), (1, 32 * unit + 1, 1, 8), (2, 35 * unit, 0, 20), (257, unit + 1, 0, 2)) + \
                (((257, 2 * unit + 3, 0, 2), (300, 4 * unit - 5, 0, 3), (520, 6 * unit + 1, 0, 1), (520, 9 * unit, 0, 2)) if kind == 1 else ()):
            print("rows", FLOATS[kind], m, v, pad, top, flush=True)
            rng = np.random.default_rng(m + v)
            x = (rng.standard_normal((m, v)) * 4).astype(np.float32)
            if v > 2:
                x[m // 2, : v // 3] = -np.inf
            L.check(x, kind, rng.integers(-1, v, m), top, 0.7 if pad else 1.0, pad)
        for v in (70, 3 * unit, 33 * unit):
            print("no numbers", FLOATS[kind], v, flush=True)
            x = np.random.default_rng(v).standard_normal((8, v)).astype(np.float32)
            x[0] = -np.inf
            x[1] = LOWEST[kind]
            x[2] = 1.5
            x[3, 5] = np.nan
            x[4, [3, 60]], x[4, 61] = np.inf, np.nan
            x[5] = np.arange(v) % 3
            x[6], x[6, 9] = -np.inf, np.nan
            x[7, :40], x[7, 40:] = -np.inf, LOWEST[kind]
            L.check(x, kind, np.array([0, 1, v, -2, 3, -1, 6, 50]), 20)


# ---- products -----------------------------------------------------------------------------------------------------
I32, FIELD, SILU, GELU = 3, 4, 0, 1
P = (1 << 64) - (1 << 32) + 1
ROUND = {0: 2.0 ** -24, 1: 2.0 ** -8, 2: 2.0 ** -11}          # half a unit in the last place, relative
LEAST = {0: 2.0 ** -126, 1: 2.0 ** -126, 2: 2.0 ** -24}
OUT = {0: np.float32, 1: np.uint16, 2: np.float16, I32: np.int32, FIELD: np.uint64}


class Products:
    def __init__(self, so):
        self.L = L = ctypes.CDLL(so)
        L.simt_workspace.restype, L.simt_workspace.argtypes = SZ, [INT, INT, INT, INT, I64, I64, I64]
        L.simt_product.argtypes = [INT] * 4 + [VP, I64] * 3 + [I64] * 3 + [VP] * 4 + [INT, INT, VP, VP]
        L.simt_error.restype = ctypes.c_char_p
        self.tiles = L.simt_tiles()

    def check(self, gated, tile, m, k, n, kind, slices=1, pack=0, pad=None, shift=0, bias=False, act=SILU):
        """One product; pad: bytes behind each row, to 16-byte boundaries where there is none given."""
        rng = np.random.default_rng(m * 131 + k * 17 + n + tile)
        a, b, u = (rng.integers(-128, 128, (r, k)).astype(np.int8) for r in (m, n, n))
        pad = -k % 16 if pad is None else pad
        (ga, lda), (gb, ldb), (gu, ldu) = (strided(t, pad, shift) for t in (a, b, u))
        assert not k or all(t.ctypes.data % 16 == shift for t in (ga, gb, gu))
        sa, sb, su = (((rng.random(r) * 0.01 + 0.0001) * 9 / math.sqrt(k + 1) ** p).astype(np.float32) for r, p in ((m, 0), (n, 1), (n, 1)))
        add = rng.standard_normal(n).astype(np.float32) if bias else None
        out = np.empty((m, n), OUT[kind])
        ws = scratch(self.L.simt_workspace(gated, tile, slices, pack, m, k, n)) if tile < self.tiles else None
        rc = self.L.simt_product(gated, tile, slices, pack, ga.ctypes.data, lda, gb.ctypes.data, ldb, gu.ctypes.data if gated else None, ldu, m, k, n, ptr(sa), ptr(sb), ptr(su), ptr(add), act, kind, ptr(out), ptr(ws))
        what = ("gated" if gated else "plain", "tile", tile, m, k, n, "type", kind, "slices", slices, "copy", pack, "pad", pad, "shift", shift, "bias", bias, "act", act)
        assert rc == 0, (what, self.L.simt_error())
        S = a.astype(np.int64) @ b.astype(np.int64).T
        if kind == I32:
            assert np.array_equal(out, S), what
            return
        if kind == FIELD:
            assert np.array_equal(out, np.where(S < 0, S.astype(np.uint64) + np.uint64(P), S.astype(np.uint64))), what
            return
        got = decode(out, kind).astype(np.float64)
        G = S * sa.astype(np.float64)[:, None] * sb.astype(np.float64)
        if not gated:
            # the sum's conversion, two products and an addition in 32 bits, then one rounding to the type
            want = G if add is None else G + add
            most = np.abs(want) * (ROUND[kind] * 1.0001) + 2.0 ** -24 * 4 * (np.abs(G) + (0 if add is None else np.abs(add))) + LEAST[kind]
        else:
            U = (a.astype(np.int64) @ u.astype(np.int64).T) * sa.astype(np.float64)[:, None] * su.astype(np.float64)
            acted = G / (1 + np.exp(-G)) if act == SILU else G * 0.5 * np.vectorize(math.erfc)(-G * math.sqrt(0.5))
            want = acted * U
            # three roundings of 2^-24 in G and in U; silu's argument, exponential and reciprocal; gelu's relative derivative is below 1 + x^2, and its
            # exponential has no results below 2^-126, which U multiplies
            rel = 2.0 ** -24 * (8 + 8 * np.abs(G)) if act == SILU else 2.0 ** -24 * (16 + 8 * np.abs(G) ** 2)
            most = np.abs(want) * (ROUND[kind] * 1.0001 + rel) + LEAST[kind] + 2.0 ** -126 * np.abs(U)
        assert (np.abs(got - want) <= most).all(), (what, np.max(np.abs(got - want) - most))


SIZES = [(256, 256), (256, 192), (256, 128), (128, 128), (64, 128)]    # of the tiles; half as many channels gated
STEPS = [64, 64, 128, 128, 128]


def tiles(so, pick):
    """Every tile over one to nine steps, with and without a ragged end: operands straight into LDS, through registers, copied first; all types."""
    L = Products(so)
    assert L.tiles == len(SIZES)
    for tile in range(L.tiles):
        rows, cols = SIZES[tile]
        for gated in (0, 1):
            wide = cols // 2 if gated else cols
            kinds = (0, 1, 2) if gated else (0, 1, 2, I32, FIELD)
            at = 0
            for steps in range(1, 10):
                for end in (0, 1, 16, 37) if pick in ("direct", "staged") and not os.environ.get("SIMT_LATE") else (0, 37):
                    k = steps * STEPS[tile] - (STEPS[tile] - end if end else 0)
                    # whole tiles; a ragged one; a little more than one
                    m, n = ((rows, wide), (rows - 7, wide - 5), (33, wide), (1, 1))[(steps + end) % 4]
                    at += 1
                    kind = kinds[at % len(kinds)]
                    print(pick, gated, tile, m, k, n, kind, flush=True)
                    opts = {"bias": at % 2 == 0 and not gated, "act": at // 3 % 2}
                    if pick == "direct":
                        L.check(gated, tile, m, k, n, kind, **opts)
                    elif pick == "staged":
                        L.check(gated, tile, m, k, n, kind, pad=1 + at % 3, shift=at % 2, **opts)
                    elif pick == "copied" and steps % 2:
                        L.check(gated, tile, m, k, n, kind, pack=1, pad=1 + at % 3, shift=at % 2, **opts)
                    elif pick == "sliced" and steps > 2:
                        L.check(gated, tile, m, k, n, kind, slices=2 + at % 3, pad=at % 2 or None, pack=at % 2 * (at // 2 % 2), **opts)
            if pick in ("direct", "staged"):                   # no inner dimension: nothing is read
                L.check(gated, tile, rows + 1, 0, wide + 3, kinds[tile % len(kinds)], pad=0 if pick == "direct" else 3, bias=not gated)
            # several tiles, each way out to the end of a row
            for kind in kinds:
                print(pick, gated, tile, "several", kind, flush=True)
                more = {"pad": 3} if pick in ("staged", "copied") else {}
                L.check(gated, tile, rows + 1, 200, 2 * wide + 3, kind, slices=2 if pick == "sliced" else 1, pack=int(pick == "copied"), act=kind % 2, **more)
                L.check(gated, tile, rows + 40, 100, 2 * wide, kind, slices=2 if pick == "sliced" else 1, pack=int(pick == "copied"), act=kind % 2, bias=not gated, **more)


def direct(so):
    tiles(so, "direct")


def staged(so):
    tiles(so, "staged")


def copied(so):
    tiles(so, "copied")


def sliced(so):
    tiles(so, "sliced")


def few_rows(so):
    """Up to 32 rows: lengths about a block of 64 and the workgroup's eight parts, no channels or rows behind the last."""
    L = Products(so)
    for gated in (0, 1):
        for at, (m, k, n) in enumerate([(1, 1, 1), (1, 15, 3), (2, 16, 16), (3, 0, 5), (1, 63, 17), (16, 64, 33), (17, 65, 16), (5, 500, 40), (32, 513, 18),
                                        (31, 4200, 16), (1, 9000, 5), (16, 4096, 20)]):
            for kind in (0, 1, 2) if gated else (0, 1, 2, I32, FIELD):
                print("few rows", gated, m, k, n, kind, flush=True)
                L.check(gated, L.tiles, m, k, n, kind, pad=(None, 0, 1)[at % 3], shift=at % 2, bias=not gated and kind != 1, act=at % 2)


def overflow(so):
    """Products that overflow before the activation: +inf stays, -inf gives 0, a NaN shows."""
    L = Products(so)
    for tile in range(L.tiles + 1):
        for act in (SILU, GELU):
            for kind in (0, 1, 2):
                print("overflow", tile, act, kind, flush=True)
                m, n = (20, 37) if tile == L.tiles else (40, 128)
                a, g, u = np.ones((m, 16), np.int8), np.ones((n, 16), np.int8), np.ones((n, 16), np.int8)
                g[1::3] = -1
                sm, sn, su = np.full(m, 1e30, np.float32), np.full(n, 1e30, np.float32), np.full(n, 1e-30, np.float32)
                sn[2::3] = np.nan
                (a, _), (g, _), (u, _) = strided(a, 0), strided(g, 0), strided(u, 0)
                out = np.empty((m, n), OUT[kind])
                ws = scratch(L.L.simt_workspace(1, tile, 1, 0, m, 16, n))
                assert L.L.simt_product(1, tile, 1, 0, a.ctypes.data, 16, g.ctypes.data, 16, u.ctypes.data, 16, m, 16, n, ptr(sm), ptr(sn), ptr(su), None, act, kind, ptr(out), ptr(ws)) == 0
                out = decode(out, kind)
                assert (out[:, 0::3] == np.inf).all() and (out[:, 1::3] == 0).all() and np.isnan(out[:, 2::3]).all(), (tile, act, kind)


def plans(so):
    """The sizes of the tests on the GPU, which are in SHAPES: what they reach."""
    L = ctypes.CDLL(so)
    L.simt_plan.argtypes = [I64, I64, I64, INT, INT, VP]
    for gated, shapes in enumerate(json.loads(os.environ["SHAPES"])):
        reached = set()
        for m, k, n, aligned in shapes:
            plan = np.zeros(3, np.int32)
            L.simt_plan(m, k, n, gated, aligned, ptr(plan))
            tile, slices, copied = plan
            print("plan", gated, m, k, n, aligned, *plan, flush=True)
            reached |= {("tile", tile)} if aligned else {("copied" if copied else "through registers", "slices" if slices > 1 else "one slice")}
            reached |= {"slices"} if aligned and slices > 1 else set()
        want = {("tile", t) for t in range(L.simt_tiles())} | {(how, s) for how in ("copied", "through registers") for s in ("slices", "one slice")} | {"slices"}
        assert reached == want, want - reached


if __name__ == "__main__":
    globals()[sys.argv[1]](sys.argv[2])
    print("OK")
