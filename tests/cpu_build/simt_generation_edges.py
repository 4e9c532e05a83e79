"""Attention over the cache and drafts on the CPU where numbers are at the ends of their ranges: scores and scales far apart, probabilities of zero.  A program of its own, as
simt_generation_checks.py is, whose forms of the calls these are."""
import ctypes
import math
import sys

import numpy as np
from simt_generation_checks import F32, F64, I8, I64, INT, ROUND, SZ, VP, Made, walk
from simt_inference_checks import LOWEST, decode, encode, ptr


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


def small_weights(so, kinds):
    """A key far ahead whose value is nothing, and what all the others' weights come to: wherever it is, in keys of one part and of several."""
    L = attention(so)
    for kind in kinds:
        given = 2 if kind == 2 else 1
        for count, value in ((1024, 1.0), (301, 1000.0), (1024, 0.01)):
            for ahead in (10.0, 15.0, 18.5, 20.5, 22.5, 25.1):
                for strong in (0, 40, count // 2, count - 1):
                    key_scale, value_scale = np.float32(0.15), np.float32(value / 100)
                    number = round(ahead * math.log(2) / 0.15) if kind == I8 else ahead * math.log(2)
                    scores = np.zeros(count)
                    scores[strong] = number
                    m, q = one_token(kind, scores, key_scale=key_scale)
                    m.data[1][:] = 100 if kind == I8 else encode(np.array([value]), kind)[0]
                    if kind == I8:
                        m.scales[1][:] = value_scale
                    p_, r_ = m.place(0, strong)
                    m.data[1][p_, :, r_] = 0
                    exact = float(number * np.float64(key_scale)) if kind == I8 else float(decode(encode(np.array([number]), kind), kind)[0])
                    v = float(100 * np.float64(value_scale)) if kind == I8 else float(decode(encode(np.array([value]), kind), kind)[0])
                    others = (count - 1) * math.exp(-exact)
                    want = v * others / (1 + others)
                    # Weights are rounded to 16 bits, the other ones all alike: half a step of them, or fp16's 2^-25 where the largest is 2^7; scores and exponentials 2^-20; the result.
                    weight = math.exp(-exact)
                    rounding = ROUND[1 if kind == 1 else 2] * weight + (0 if kind == 1 else 2.0 ** -32)
                    off = want * (rounding / weight + 2.0 ** -20 * (1 + exact)) + (2.0 ** -25 if kind == 2 else 0)
                    for form, splits, per in FORMS:
                        got = attended(L, m, q, form, splits, per, 1.0)[0, 0]
                        assert (np.abs(got - want) <= off + ROUND[given] * (want + off)).all(), (kind, count, value, ahead, strong, form, splits, got[0], want, off)


def small_weights_16(so):
    small_weights(so, (1, 2))


def values_alike(so):
    """Values all alike come out as they are, whatever 16 bits make of their weights: of late keys that count for nearly all, too."""
    L = attention(so)
    for kind in (1, 2):
        for count in (60, 300):
            for dim in (64, 128):
                rng = np.random.default_rng(count + dim)
                late = [np.where(np.arange(count) == at, x, np.where(np.arange(count) == 0, 0.0, -30.0)) for x in (4.55, 4.9, 5.0, 5.5) for at in (29, 40, 129) if at < count]
                for scores in (rng.standard_normal(count), rng.standard_normal(count) * 4, np.linspace(0, 5, count), *late):
                    m, q = one_token(kind, scores, dim)
                    v = encode(rng.standard_normal(dim), kind)
                    m.data[1][:] = v
                    for form, splits, per in FORMS:
                        got = attended(L, m, q, form, splits, per, 1.0)[0, 0]
                        assert np.array_equal(got, decode(v, kind).astype(np.float64)), (kind, count, dim, form, splits)


def small_scales(so):
    """Queries and scales so small that all scores are nothing: each key counts alike, and none that is hidden."""
    L = attention(so)
    for kind in (1, 2, I8):
        for scale in (1e-10, 1e-30, 1e-45):
            for size in (0.0, 1e-30, 1.0):
                for count in (40, 300):
                    m = Made(kind, [count - 3], [3], 1, 64, 64)
                    q = encode(np.full((3, 1, 64), size), 2 if kind == 2 else 1)
                    v = np.stack([m.held(1, 0, j)[0] for j in range(count)])
                    for form, splits, per in FORMS:
                        got = attended(L, m, q, form, splits, per, scale)[:, 0]
                        for i in range(3):
                            seen = v[:count - 2 + i]
                            want, size_ = seen.mean(0), np.abs(seen).mean(0)
                            # weights all alike are right, but times scales over integers, where they are fp16 and 32-bit sums of values up to 256; the result
                            off = 2.0 ** -20 * size_ + (2.0 ** -11 * size_ + (count / 16 + 8) * 2.0 ** -24 * 256 * 0.03 if kind == I8 else 0) + (2.0 ** -25 if kind == 2 else 0)
                            assert (np.abs(got[i] - want) <= off + ROUND[2 if kind == 2 else 1] * (np.abs(want) + off)).all(), (kind, scale, size, count, form, splits, i, got[i][:3], want[:3])


# ---- drafts -------------------------------------------------------------------------------------------------------
def drafts(so):
    L = ctypes.CDLL(so)
    L.vi_verify_drafts_workspace_bytes.restype = SZ
    L.vi_verify_drafts_workspace_bytes.argtypes = [INT, I64, I64, I64, INT]
    L.vi_verify_drafts.argtypes = [INT, VP, I64, I64, I64, VP, I64, VP, VP, I64, VP, VP, F64, I64, VP, VP, VP, VP, SZ, VP]
    return L


def verified(L, kind, logits, draft, tokens, parents, u, depth, t=1.0):
    """One sequence; what comes out, and what walk() says."""
    n, v = logits.shape
    tokens, parents, u = np.array(tokens, np.int64), np.array(parents, np.int32), np.array(u, np.float64)
    starts = np.array([0, n], np.int32)
    count, nodes, out = np.zeros(1, np.int64), np.full((1, depth), 9, np.int64), np.full((1, depth + 1), 9, np.int64)
    need = L.vi_verify_drafts_workspace_bytes(kind, n, v, 1, int(draft is not None))
    ws = np.full(need + 8, 0xA5, dtype=np.uint8)[8:]
    assert L.vi_verify_drafts(kind, ptr(logits), n, v, v, ptr(draft), v, ptr(tokens), ptr(starts), 1, ptr(parents), ptr(u), t, depth, ptr(count), ptr(nodes), ptr(out), ptr(ws), need, None) == 0
    (c, wn, wo), = walk(decode(logits, kind), tokens, starts, parents, u, depth, None if draft is None else decode(draft, kind), t)
    return (int(count[0]), nodes[0].tolist(), out[0].tolist()), (c, wn, wo)


ALMOST_ONE = 1.0 - 2.0 ** -53


def masked_drafts(so):
    """Drafts whose token the target, the draft model or both mask, with -inf or far down, behind refusals of others or of none."""
    L = drafts(so)
    for kind in (0, 1, 2):
        for v in (50, 2100):
            rng = np.random.default_rng(v + kind)
            for mask in (-np.inf, -1e9, LOWEST[kind]):
                logits, draft = (rng.standard_normal((5, v)).astype(np.float32) * 3 for _ in range(2))
                likelier = np.argsort(logits[0] - draft[0])            # by the draft model, and so refused by numbers close to one
                masked = int(likelier[v // 2])
                for where in ("target", "draft", "both"):
                    x, y = logits.copy(), draft.copy()
                    if where != "draft":
                        x[0, masked] = mask
                    if where != "target":
                        y[0, masked] = mask
                    x, y = encode(x, kind), encode(y, kind)
                    for refused in (0, 1, 2):
                        for u in (0.0, 0.3, ALMOST_ONE):
                            for root in (0.0, 0.6):
                                tokens = [0] + likelier[:refused].tolist() + [masked] + [int(likelier[-1])] * (3 - refused)
                                numbers = [root] + [ALMOST_ONE] * refused + [u] + [0.5] * (3 - refused)
                                for given in (None, y):
                                    got, want = verified(L, kind, x, given, tokens, [-1] + [0] * 4, numbers, 2)
                                    assert got == want, (kind, v, mask, where, refused, u, root, given is not None, got, want)


def first_tokens(so):
    """The token of a root's number zero is the first that has a probability, and where nothing is left behind refusals, too."""
    L = drafts(so)
    for kind in (0, 1, 2):
        for v in (40, 1100, 9000):
            for mask in (-np.inf, -1e9, LOWEST[kind]):
                rng = np.random.default_rng(v)
                x = rng.standard_normal((3, v)).astype(np.float32)
                x[:, :v // 2] = mask
                x[:, v - 3:] = mask
                x = encode(x, kind)
                for given in (None, x):
                    for u in (0.0, 0.5, ALMOST_ONE):
                        # p - p is nothing, where p / sum(p) - p in 64 bits may leave 1e-17: of p itself, which refused tokens without a probability change as little without a draft model
                        args = [0, 1, 2], [-1, 0, 0], [u, ALMOST_ONE, ALMOST_ONE], 2
                        got, want = verified(L, kind, x, given, *args)[0], verified(L, kind, x, None, *args)[1]
                        assert got == want, (kind, v, mask, u, given is not None, got, want)
                one = np.full((2, v), mask, np.float32)        # all of it refused
                one[:, v // 2] = 1.0
                one = encode(one, kind)
                for given in (None, one):
                    got, _ = verified(L, kind, one, given, [0, v // 2], [-1, 0], [0.0, 1.0], 1)
                    assert got == (0, [-1], [v // 2, -1]), (kind, v, mask, given is not None, got)


def far_logits(so):
    """Rows all of whose entries are the type's lowest, or as large, or near to each other and far from nothing."""
    L = drafts(so)
    for kind in (0, 1, 2):
        for v in (7, 1300):
            rng = np.random.default_rng(v)
            for far in (LOWEST[kind], LOWEST[kind] / 2, -LOWEST[kind], 3e4, -1.7e4, 1e6, -1e12, 1e20):
                if kind == 2 and abs(far) > 65504:
                    continue
                for near in (False, True):
                    x = np.full((4, v), far, np.float32)
                    if near:                   # neighbouring numbers of the type, or equal ones
                        x *= (1 - rng.integers(0, 3, x.shape) * {0: 2.0 ** -23, 1: 2.0 ** -7, 2: 2.0 ** -10}[kind]).astype(np.float32)
                    x = encode(x, kind)
                    y = encode(rng.standard_normal((4, v)), kind)
                    for t in (1.0, 0.7, 0.3, 1e-3, 1e3, 17.0):
                        for given in (None, y):
                            got, want = verified(L, kind, x, given, [0] + rng.integers(0, v, 3).tolist(), [-1, 0, 0, 1], rng.random(4), 2, t)
                            assert got == want, (kind, v, far, near, t, given is not None, got, want)


def few_tokens_left(so):
    """Without a draft model, refusals that leave little or one token, or nothing: what is left is summed, not taken for what the refused ones lack to one."""
    L = drafts(so)
    for kind in (0, 1, 2):
        for v in (3, 60, 1500):
            for allowed in (2, 3, 5):
                for seed in range(6):
                    rng = np.random.default_rng(seed)
                    allowed = min(allowed, v)
                    x = np.full((allowed + 3, v), -np.inf, np.float32)
                    tokens = rng.permutation(v)[:allowed]
                    # one after the other 10 to 40 nats apart, or near each other
                    x[0, tokens] = rng.standard_normal(allowed) if seed < 3 else -rng.uniform(5, 45, allowed).cumsum().astype(np.float32) / (1 if allowed < 5 else 3)
                    x[1:, 0] = 0
                    x = encode(x, kind)
                    for u in ([ALMOST_ONE] * (allowed - 1) + [0.5], [ALMOST_ONE] * allowed, [ALMOST_ONE] * (allowed - 1) + [0.999]):
                        # the same token twice; in the end the one that is left, again, and any
                        children = tokens.tolist()[:-1] + [int(tokens[0]), int(tokens[-1])] + [int(tokens[-1])]
                        got, want = verified(L, kind, x, None, [0] + children, [-1] + [0] * (allowed + 2), [0.4] + u[:-1] + [0.7, u[-1], 0.0], 2)
                        assert got == want, (kind, v, allowed, seed, u, got, want)


def next_to_the_border(so):
    """Drafts whose number is 3 10^-14 of it above or below p / q.  Entries are at most 32 below their row's largest: differences of them are 32 2^-53 off, their exponentials
    4 10^-16, sums and quotients 10 2^-53 - of p and q together 10^-14."""
    L = drafts(so)
    for kind in (0, 1, 2):
        rng = np.random.default_rng(kind)
        x, y = (encode(np.clip(rng.standard_normal((2, 300)) * 3, -16, 16), kind) for _ in range(2))
        p, q = (np.exp(z - z.max()) for z in (decode(x[0], kind).astype(np.longdouble), decode(y[0], kind).astype(np.longdouble)))
        share = (p / p.sum()) / (q / q.sum())
        for token in np.argsort(share)[:40].tolist():
            for above in (0, 1):
                (count, _, _), _ = verified(L, kind, x, y, [0, token], [-1, 0], [0.5, float(share[token] * (1 + (2 * above - 1) * np.longdouble(3e-14)))], 1)
                assert count == 1 - above, (kind, token, above)


if __name__ == "__main__":
    globals()[sys.argv[1]](sys.argv[2])
    print("OK")
