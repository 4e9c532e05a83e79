"""The kernels of the cache, of attention over it and of drafts on the CPU (simt_generation.hpp), against 64-bit results, as a program of its own: the test runs it
under AddressSanitizer, where every numpy array is a heap block of exactly its size."""
import ctypes
import math
import sys

import numpy as np
from simt_inference_checks import decode, encode, ptr

I64, VP, SZ, INT, F32, F64 = ctypes.c_int64, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_float, ctypes.c_double
ROUND = {0: 2.0 ** -24, 1: 2.0 ** -8, 2: 2.0 ** -11}
I8 = 5


class CacheArgs(ctypes.Structure):
    _fields_ = [("keys", VP), ("values", VP), ("key_scales", VP), ("value_scales", VP), ("key_strides", I64 * 3), ("value_strides", I64 * 3), ("key_scale_strides", I64 * 2),
                ("value_scale_strides", I64 * 2), ("pages", I64), ("heads", I64), ("page_size", I64), ("dim", I64), ("dtype", I64)]


class BatchArgs(ctypes.Structure):
    _fields_ = [("starts", VP), ("lengths", VP), ("pages", VP), ("sequences", I64), ("width", I64), ("stride", I64)]


def aligned(a):
    """The array at a multiple of 16 bytes, in a block that ends with it."""
    for lead in (0, 8) * 50:
        flat = np.full(a.nbytes + lead, 0xA5, dtype=np.uint8)
        if (flat.ctypes.data + lead) % 16 == 0:
            break
        aligned.kept.append(flat)
    view = flat[lead:].view(a.dtype).reshape(a.shape)
    view[:] = a
    return view


aligned.kept = []


class Made:
    """Sequences with `before` entries and `new` more in a cache of pages in no order, rows by rows or heads by heads."""

    def __init__(self, kind, before, new, heads, dim, page, layout=0, gap=0, bad=()):
        rng = np.random.default_rng(len(before) * 1000 + heads * 100 + dim + page)
        self.kind, self.before, self.new, self.page, self.heads, self.dim = kind, before, new, page, heads, dim
        lengths = [b + n for b, n in zip(before, new)]
        need = [-(-x // page) for x in lengths]
        self.pages = sum(need) + 1
        shape = (self.pages, heads, page, dim) if layout == 0 else (self.pages, page, heads, dim)
        self.data, self.scales, self.values = [], [], []
        for _ in range(2):
            x = rng.integers(-127, 128, shape).astype(np.int8) if kind == I8 else encode(rng.standard_normal(shape), kind)
            self.data.append(aligned(x))
            self.scales.append((rng.random((self.pages, heads, page)) * 0.02 + 0.01).astype(np.float32) if kind == I8 else None)
        self.layout = layout
        step = [heads * page * dim, page * dim, dim] if layout == 0 else [heads * page * dim, dim, heads * dim]
        scale_step = [heads * page, page]
        order = rng.permutation(self.pages)[:sum(need)].tolist()
        width = max(need + [0])
        self.table = np.full((len(before), width), -1, dtype=np.int32)
        for b, k in enumerate(need):
            self.table[b, :k] = [order.pop() for _ in range(k)]
        for b, i, number in bad:
            self.table[b, i] = number
        self.starts = np.array([gap + sum(new[:b]) for b in range(len(new) + 1)], dtype=np.int32)
        self.lengths = np.array(lengths, dtype=np.int32)
        self.n = int(self.starts[-1]) + gap
        self.cache = CacheArgs(ptr(self.data[0]), ptr(self.data[1]), ptr(self.scales[0]), ptr(self.scales[1]), (I64 * 3)(*step), (I64 * 3)(*step), (I64 * 2)(*scale_step),
                               (I64 * 2)(*scale_step), self.pages, heads, page, dim, kind)
        self.batch = BatchArgs(ptr(self.starts), ptr(self.lengths), ptr(self.table), len(before), width, max(width, 1))

    def place(self, b, j):
        """Page and row of an entry, None where no page holds it."""
        p = int(self.table[b, j // self.page])
        return (p, j % self.page) if 0 <= p < self.pages else None

    def entry(self, h, p, r):
        """(heads, dim) as stored."""
        return self.data[h][p, :, r] if self.layout == 0 else self.data[h][p, r]

    def held(self, h, b, j):
        at = self.place(b, j)
        if at is None:
            return None
        x = self.entry(h, *at)
        return x.astype(np.float64) * self.scales[h][at[0], :, at[1]][:, None] if self.kind == I8 else decode(x, self.kind).astype(np.float64)


def steps_of(dim):
    f = [10000.0 ** (-2 * i / dim) for i in range(dim // 2)]
    return f, np.array([round(x / (2 * math.pi) * 2.0 ** 64) % (1 << 64) for x in f], dtype=np.uint64)


def turn(x, positions, dim, interleaved):
    x = x.astype(np.float64).copy()
    f, _ = steps_of(dim)
    a = np.outer(positions.astype(np.float64), f)[:, None]
    c, s = np.cos(a), np.sin(a)
    u, w = (x[..., 0:dim:2].copy(), x[..., 1:dim:2].copy()) if interleaved else (x[..., :dim // 2].copy(), x[..., dim // 2:dim].copy())
    y = (u * c - w * s, u * s + w * c)
    if interleaved:
        x[..., 0:dim:2], x[..., 1:dim:2] = y
    else:
        x[..., :dim // 2], x[..., dim // 2:dim] = y
    return x


# ---- positions ----------------------------------------------------------------------------------------------------
def rotate(so):
    L = ctypes.CDLL(so)
    L.vi_rotate_heads.argtypes = [INT, VP, I64, I64, I64, I64, I64, VP, VP, I64, INT, F64, VP, I64, I64, VP]
    for kind in (0, 1, 2):
        for n, heads, d, dim, interleaved in ((1, 1, 2, 2, 0), (1, 32, 128, 128, 0), (3, 5, 64, 32, 1), (2, 3, 80, 20, 0), (5, 17, 30, 6, 1), (40, 1, 256, 256, 0), (33, 2, 16, 16, 1), (3, 20, 112, 48, 0)):
            print("rotate", kind, n, heads, d, dim, flush=True)
            rng = np.random.default_rng(n + heads + d)
            x = encode(rng.standard_normal((n, heads, d)), kind)
            out, positions, steps = np.zeros_like(x), rng.integers(0, 1000, n), steps_of(dim)[1]
            assert L.vi_rotate_heads(kind, ptr(x), n, heads, d, heads * d, d, ptr(positions), ptr(steps), dim, interleaved, 1.0, ptr(out), heads * d, d, None) == 0
            want = turn(decode(x, kind), positions, dim, interleaved)
            assert (np.abs(decode(out, kind) - want) <= ROUND[kind] * np.abs(want) + 1e-5).all()


def append(so):
    L = ctypes.CDLL(so)
    L.vi_append_tokens.argtypes = [VP, VP, INT, VP, I64, I64, VP, I64, I64, I64, VP, VP, I64, INT, F64, VP]
    for kind in (1, 2, I8):
        for number, (before, new, heads, dim, page, rotated, layout, bad) in enumerate((
                ([0], [1], 1, 16, 16, 16, 0, ()), ([5, 15, 0], [3, 1, 20], 3, 64, 16, 64, 1, ()), ([30, 16, 7], [2, 0, 33], 8, 128, 32, 64, 0, ()), ([0], [50], 2, 80, 16, 20, 0, ()),
                ([3, 9], [40, 30], 1, 256, 16, 256, 1, [(0, 1, -1), (1, 2, 1 << 30)]), ([100] * 70, [1] * 70, 1, 32, 64, 0, 0, ()))):
            print("append", kind, before[:3], new[:3], heads, dim, page, flush=True)
            m = Made(kind, before, new, heads, dim, page, layout, 2, bad)
            rng = np.random.default_rng(number)
            for given in (0, 1, 2):
                k, v = (encode(rng.standard_normal((m.n, heads, dim)), given) for _ in range(2))
                was = [a.copy() for a in m.data] + [a.copy() for a in m.scales if a is not None]
                steps = steps_of(rotated)[1] if rotated else None
                assert L.vi_append_tokens(ctypes.byref(m.cache), ctypes.byref(m.batch), given, ptr(k), heads * dim, dim, ptr(v), heads * dim, dim, m.n, None, ptr(steps), rotated, number & 1,
                                          1.0, None) == 0
                touched = np.zeros((m.pages, page), dtype=bool)
                for b, count in enumerate(new):
                    for i in range(count):
                        at = m.place(b, before[b] + i)
                        if at is None:
                            continue
                        touched[at] = True
                        row = int(m.starts[b]) + i
                        key = decode(k[row:row + 1], given).astype(np.float64)
                        if rotated:
                            key = turn(key, np.array([before[b] + i]), rotated, number & 1)
                        for h, want in ((0, key[0]), (1, decode(v[row], given).astype(np.float64))):
                            got, most = m.held(h, b, before[b] + i), np.abs(want).max(axis=1, keepdims=True)
                            off = most / 127 * 0.5001 if kind == I8 else ROUND[kind] * np.abs(want) + (0 if h else 1e-5)
                            assert (np.abs(got - want) <= off + 1e-6).all()
                now = m.data + [a for a in m.scales if a is not None]
                for i, (a, b) in enumerate(zip(was, now)):
                    if layout and i < 2:
                        a, b = a.swapaxes(1, 2), b.swapaxes(1, 2)
                    assert np.array_equal(a.swapaxes(1, 2)[~touched], b.swapaxes(1, 2)[~touched])


# ---- attention ----------------------------------------------------------------------------------------------------
def wanted(m, q, group, parents):
    out, size = np.zeros(q.shape), np.zeros(q.shape)
    for b, count in enumerate(m.new):
        above = []
        for i in range(count):
            p = i - 1 if parents is None else int(parents[m.starts[b] + i])
            above.append({i} | (above[p] if 0 <= p < i else set()))
        held = [[m.held(h, b, j) for j in range(m.before[b] + count)] for h in range(2)]
        for i in range(count):
            keys = [j for j in list(range(m.before[b])) + [m.before[b] + a for a in sorted(above[i])] if held[0][j] is not None]
            if not keys:
                continue
            k, v = (np.stack([held[h][j] for j in keys]) for h in range(2))
            for head in range(q.shape[1]):
                s = k[:, head // group] @ q[m.starts[b] + i, head] / math.sqrt(m.dim)
                p = np.exp(s - s.max())
                p /= p.sum()
                out[m.starts[b] + i, head], size[m.starts[b] + i, head] = p @ v[:, head // group], p @ np.abs(v[:, head // group])
    return out, size


CASES = [  # before, new, heads of the cache, group, dim, page, layout, tree, pages that are none
    ([0], [1], 1, 1, 16, 16, 0, False, ()), ([70, 0, 33], [1, 1, 1], 2, 3, 64, 16, 1, False, ()), ([200], [3], 1, 4, 128, 64, 0, False, ()), ([40, 300], [9, 20], 1, 2, 80, 32, 0, True, [(1, 2, -1)]),
    ([5], [70], 1, 2, 64, 16, 1, False, [(0, 1, 1 << 20)]), ([150], [40], 1, 4, 128, 128, 0, True, ()), ([33], [2], 1, 16, 256, 16, 0, False, ()), ([0, 100], [130, 1], 1, 1, 96, 64, 0, True, ()),
    ([100], [33], 1, 4, 256, 64, 1, True, ())]


def attend(so, kinds=(1, 2, I8), whole=False):
    """Both forms, keys in one part and in several; `whole`: where all loads of a stage are made alike, arriving late."""
    L = ctypes.CDLL(so)
    L.simt_attend.argtypes = [INT, INT, INT, VP, VP, INT, VP, I64, I64, I64, I64, VP, F32, VP, VP]
    L.simt_ws_floats.argtypes = [INT, INT, I64, I64, I64, I64, I64]
    L.simt_ws_floats.restype = I64
    for kind in kinds:
        given = 2 if kind == 2 else 1
        for before, new, heads, group, dim, page, layout, tree, bad in CASES:
            if whole and dim not in (64, 128, 256):
                continue
            m = Made(kind, before, new, heads, dim, page, layout, 1, bad)
            rng = np.random.default_rng(dim + sum(new))
            q = encode(rng.standard_normal((m.n, heads * group, dim)), given)
            parents = None
            if tree:
                parents = np.concatenate([[0]] + [np.array([-1] + [int(rng.integers(max(0, (i - 1) // 3), i)) for i in range(1, c)]) for c in new] + [[0]]).astype(np.int32)
                parents[m.starts[0]] = 7       # none that is lower: a root all the same
            want, size = wanted(m, decode(q, given).astype(np.float64), group, parents)
            for form in (0, 1):
                for splits, per in ((1, 128), (3, 128)):
                    print("attend", kind, before, new, heads, group, dim, page, "form", form, "parts", splits, flush=True)
                    out = np.full_like(q, 0x4242 if given == 1 else 7)
                    ws = np.full(L.simt_ws_floats(form, splits, m.n, heads * group, heads, len(new), dim), np.nan, dtype=np.float32)
                    assert L.simt_attend(form, splits, per, ctypes.byref(m.cache), ctypes.byref(m.batch), given, ptr(q), m.n, heads * group, heads * group * dim, dim, ptr(parents),
                                         dim ** -0.5, ptr(out), ptr(ws)) == 0
                    got = decode(out, given).astype(np.float64)
                    off = ROUND[given] * (1.02 * size + np.abs(want)) + 1e-3 * size + 1e-30
                    assert (np.abs(got - want) <= off).all(), (np.abs(got - want) - off).max()


def late(so):
    attend(so, (1, 2), True)


# ---- drafts -------------------------------------------------------------------------------------------------------
def softmax(x, t):
    z = x.astype(np.float64) / t
    if not (z < np.inf).all() or not (z > -np.inf).any():
        return None
    e = np.exp(z - z.max())
    return e / e.sum()


def walk(logits, tokens, starts, parents, u, depth, draft, t):
    result = []
    for s0, s1 in zip(starts, starts[1:]):
        path, out = [0], [-1] * (depth + 1)
        nodes = [-1] * depth
        if s1 > s0:
            p = first = softmax(logits[s0], t)
            for i in range(1, s1 - s0):
                up, x, cur = parents[s0 + i], tokens[s0 + i], path[-1]
                q = None if draft is None else softmax(draft[s0 + cur], t)
                if up != cur or len(path) > depth or not 0 <= x < logits.shape[1] or p is None or (draft is not None and q is None):
                    continue
                if u[s0 + i] * (1.0 if q is None else q[x]) * p.sum() < p[x]:
                    nodes[len(path) - 1], out[len(path) - 1] = i, x
                    path.append(i)
                    p = first = softmax(logits[s0 + i], t)
                elif q is None:
                    p = p.copy()
                    p[x] = 0
                elif p.sum() > 0:
                    p = np.maximum(p / p.sum() - q, 0)
            if p is not None:
                c = np.cumsum(p if p.sum() > 0 else first)
                out[len(path) - 1] = int((c <= u[s0] * c[-1]).sum())
        result.append((len(path) - 1, nodes, out))
    return result


def drafts(so):
    L = ctypes.CDLL(so)
    L.vi_verify_drafts_workspace_bytes.restype = SZ
    L.vi_verify_drafts_workspace_bytes.argtypes = [INT, I64, I64, I64, INT]
    L.vi_verify_drafts.argtypes = [INT, VP, I64, I64, I64, VP, I64, VP, VP, I64, VP, VP, F64, I64, VP, VP, VP, VP, SZ, VP]
    for kind in (0, 1, 2):
        for counts, v, depth, t, drafted in (([1], 1, 2, 1.0, False), ([3, 2], 2, 1, 1.0, True), ([6, 0, 9], 77, 4, 0.7, True), ([8, 5], 700, 3, 1.0, False), ([12], 2100, 6, 1.3, True),
                                             ([4], 9000, 2, 1.0, True), ([7, 7, 7], 33, 0, 1.0, False)):
            print("drafts", kind, counts, v, depth, drafted, flush=True)
            rng = np.random.default_rng(v + depth)
            starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
            n = int(starts[-1])
            logits, draft = (encode(rng.standard_normal((n, v)) * 3, kind) for _ in range(2))
            parents = np.concatenate([np.array([-1] + [int(rng.integers(0, i)) for i in range(1, c)][:max(c - 1, 0)])[:c] for c in counts]).astype(np.int32)
            tokens, u = rng.integers(0, v, n), rng.random(n)
            tokens[0:n:5] = rng.integers(-2, v + 2, len(tokens[0:n:5]))
            for chain in (False, True):
                pa = np.concatenate([np.arange(c) - 1 for c in counts]).astype(np.int32) if chain else parents
                rc, rn, ro = np.full(len(counts), 9, np.int64), np.full((len(counts), depth), 9, np.int64), np.full((len(counts), depth + 1), 9, np.int64)
                need = L.vi_verify_drafts_workspace_bytes(kind, n, v, len(counts), int(drafted))
                ws = np.full(need + 8, 0xA5, dtype=np.uint8)[8:]
                assert L.vi_verify_drafts(kind, ptr(logits), n, v, v, ptr(draft) if drafted else None, v, ptr(tokens), ptr(starts), len(counts), None if chain else ptr(parents), ptr(u), t,
                                          depth, ptr(rc), ptr(rn), ptr(ro), ptr(ws), need, None) == 0
                for b, (c, nodes, out) in enumerate(walk(decode(logits, kind), tokens, starts, pa, u, depth, decode(draft, kind) if drafted else None, t)):
                    assert rc[b] == c and rn[b].tolist() == nodes and ro[b].tolist() == out, (b, rc[b], c, rn[b], nodes, ro[b], out)

    # one sibling refused after the other: more entries left than the lists of them hold, and fewer
    for kind, v, n in ((0, 36000, 5), (2, 3000, 9)):
        print("siblings", kind, v, flush=True)
        rng = np.random.default_rng(v)
        logits, draft = (encode(rng.standard_normal((n, v)) * 3, kind) for _ in range(2))
        likelier = np.argsort(decode(logits, kind)[0] - decode(draft, kind)[0])          # by the draft model, and so refused
        tokens, starts, parents, u = likelier[:n].astype(np.int64), np.array([0, n], np.int32), np.array([-1] + [0] * (n - 1), np.int32), rng.random(n)
        tokens[-1] = likelier[-1]
        rc, rn, ro = np.zeros(1, np.int64), np.zeros((1, 2), np.int64), np.zeros((1, 3), np.int64)
        need = L.vi_verify_drafts_workspace_bytes(kind, n, v, 1, 1)
        ws = np.full(need + 8, 0xA5, dtype=np.uint8)[8:]
        assert L.vi_verify_drafts(kind, ptr(logits), n, v, v, ptr(draft), v, ptr(tokens), ptr(starts), 1, ptr(parents), ptr(u), 1.0, 2, ptr(rc), ptr(rn), ptr(ro), ptr(ws), need, None) == 0
        (c, nodes, out), = walk(decode(logits, kind), tokens, starts, parents, u, 2, decode(draft, kind), 1.0)
        assert c == 1 and rc[0] == c and rn[0].tolist() == nodes and ro[0].tolist() == out, (rc, c, rn, nodes, ro, out)


def keep(so):
    L = ctypes.CDLL(so)
    L.vi_keep_drafts.argtypes = [VP, VP, VP, I64, VP, VP, VP]
    for kind in (1, I8):
        for before, new, depth, heads, dim, page, layout, bad in (([0], [1], 1, 1, 16, 16, 0, ()), ([100, 3, 7], [25, 0, 9], 5, 3, 128, 16, 1, ()), ([15] * 6, [40] * 6, 20, 2, 80, 32, 0, [(2, 1, -5)])):
            print("keep", kind, before, new, flush=True)
            m = Made(kind, before, new, heads, dim, page, layout, 0, bad)
            rng = np.random.default_rng(depth)
            nodes, counts = np.full((len(new), depth), -1, np.int64), np.zeros(len(new), np.int64)
            for b, x in enumerate(new):
                path = sorted(rng.choice(np.arange(1, max(x, 2)), min(depth, max(x - 1, 0)), replace=False).tolist())
                nodes[b, :len(path)], counts[b] = path, rng.integers(0, len(path) + 1)
            counts[0] += 3                     # more than there are
            want = [a.copy() for a in m.data] + [a.copy() for a in m.scales if a is not None]
            lengths = np.zeros(len(new), np.int32)
            expected = []
            for b, x in enumerate(new):
                d, last = 0, 0
                while d < min(counts[b], depth) and last < nodes[b, d] < x:
                    src, dst = m.place(b, before[b] + int(nodes[b, d])), m.place(b, before[b] + d + 1)
                    if src and dst:
                        for a in want[:2]:
                            if layout:
                                a[dst[0], dst[1]] = a[src[0], src[1]]
                            else:
                                a[dst[0], :, dst[1]] = a[src[0], :, src[1]]
                        for a in want[2:]:
                            a[dst[0], :, dst[1]] = a[src[0], :, src[1]]
                    last, d = nodes[b, d], d + 1
                expected.append(before[b] + 1 + d if x else before[b])
            assert L.vi_keep_drafts(ctypes.byref(m.cache), ctypes.byref(m.batch), ptr(nodes), depth, ptr(counts), ptr(lengths), None) == 0
            assert lengths.tolist() == expected
            assert all(np.array_equal(a, b) for a, b in zip(want, m.data + [a for a in m.scales if a is not None]))


if __name__ == "__main__":
    {"rotate": rotate, "append": append, "attend": attend, "late": late, "drafts": drafts, "keep": keep}[sys.argv[1]](sys.argv[2])
    print("OK")
