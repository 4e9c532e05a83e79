"""The kernels of the forward pass in 8-bit integers on the CPU (simt_inference.hpp), against 64-bit results, as a program of its own: the
test runs it under AddressSanitizer, where every numpy array is a heap block of exactly its size."""
import ctypes
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
    flat = np.full(shift + (m - 1) * (k + pad) + k, 77, dtype=a.dtype)
    view = np.lib.stride_tricks.as_strided(flat[shift:], (m, k), ((k + pad) * a.itemsize, a.itemsize))
    view[:] = a
    return view, k + pad


def scratch(nbytes):
    """nbytes of garbage from an address that is a multiple of 8 only, nothing behind them."""
    return np.full(nbytes + 8, 0xA5, dtype=np.uint8)[8:]


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
            for top in (1, 3, 20, 64) if v < 10000 else (5, 64):
                L.check(x, kind, tokens, top)


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
                               (1, 32 * unit, 0, 8), (1, 32 * unit + 1, 1, 8), (2, 35 * unit, 0, 20), (257, unit + 1, 0, 2), (257, 2 * unit + 3, 0, 2),
                               (300, 4 * unit - 5, 0, 3), (300, 8 * unit + 1, 0, 2)) + (((520, 6 * unit + 1, 0, 1), (520, 9 * unit, 0, 2)) if kind == 1 else ()):
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


if __name__ == "__main__":
    globals()[sys.argv[1]](sys.argv[2])
    print("OK")
