"""Attention over the cache and drafts on the CPU where numbers are at the ends of their ranges: scores and scales far apart, probabilities of zero.  A program of its own, as
simt_generation_checks.py is, whose forms of the calls these are."""
import ctypes
import math
import sys

import numpy as np
from simt_generation_checks import F32, I8, I64, INT, ROUND, VP, Made
from simt_inference_checks import decode, encode, ptr


def attention(so):
    L = ctypes.CDLL(so)
    L.simt_attend.argtypes = [INT, INT, INT, VP, VP, INT, VP, I64, I64, I64, I64, VP, F32, VP, VP]
    L.simt_ws_floats.argtypes = [INT, INT, I64, I64, I64, I64, I64]
    L.simt_ws_floats.restype = I64
    return L


def attended(L, m, q, form, splits, per, scale):
    """Of queries (n, heads, dim) as stored, in 64 bits."""
    n, heads, dim = q.shape
    out, given = np.zeros_like(q), 2 if m.kind == 2 else 1
    ws = np.full(L.simt_ws_floats(form, splits, n, heads, m.heads, len(m.new), dim), np.nan, dtype=np.float32)
    assert L.simt_attend(form, splits, per, ctypes.byref(m.cache), ctypes.byref(m.batch), given, ptr(q), n, heads, heads * dim, dim, None, scale, ptr(out), ptr(ws)) == 0
    return decode(out, given).astype(np.float64)


FORMS = [(form, splits, per) for form in (0, 1) for splits, per in ((1, 128), (3, 128))]


def one_token(kind, scores, dim=128, key_scale=1.0):
    """A token whose query is one in the first column, over keys that have its scores there and nothing elsewhere."""
    m = Made(kind, [len(scores) - 1], [1], 1, dim, 64)
    q = encode(np.zeros((1, 1, dim)), 2 if kind == 2 else 1)
    q[0, 0, 0] = encode(np.ones(1), 2 if kind == 2 else 1)[0]
    m.data[0][:] = 0
    for j, s in enumerate(scores):
        p, r = m.place(0, j)
        m.data[0][p, 0, r, 0] = int(s) if kind == I8 else encode(np.array([s]), kind)[0]
    if kind == I8:
        m.scales[0][:] = key_scale
    return m, q


def places(m, count):
    return [m.place(0, j) for j in range(count)]


def late_keys(so):
    """Over 8-bit integers: a key far above those before it, behind value scales of any size."""
    L = attention(so)
    count = 301
    for value_scale in (0.02, 1.0, 3.0, 4.0, 100.0, 2.0 ** 60, 2.0 ** -60):
        for ahead in (20, 86, 88, 95, 110, 127):
            for late in (0, 40, 200, 300):
                scores = np.zeros(count)
                scores[late] = ahead
                m, q = one_token(I8, scores)
                m.scales[1][:] = value_scale
                v = np.stack([m.held(1, 0, j)[0] for j in range(count)])
                p = np.exp(scores - scores.max())
                p /= p.sum()
                want, size, weights = p @ v, p @ np.abs(v), value_scale
                # weights are fp16, half a step of them off or 2^-25 of the largest, times values up to 127; sums in 32 bits are of values up to 256; the result is bfloat16
                off = (2.0 ** -11 + 2.0 ** -20) * size + (count * 2.0 ** -25 * 127 + (count / 16 + 8) * 2.0 ** -24 * 256) * weights
                for form, splits, per in FORMS:
                    got = attended(L, m, q, form, splits, per, 1.0)[0, 0]
                    bad = ~(np.abs(got - want) <= off + ROUND[1] * (np.abs(want) + off))
                    assert not bad.any(), ("late", value_scale, ahead, late, form, splits, int(bad.sum()), got[:3], want[:3])


if __name__ == "__main__":
    globals()[sys.argv[1]](sys.argv[2])
    print("OK")
