"""Positions, the paged cache, attention over it, drafts: against plain implementations in 64 bits."""
import math
import random

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from verinf_amd.prover import generation as gen  # noqa: E402
from verinf_amd.prover import inference as inf  # noqa: E402

FLOATS = [torch.float32, torch.bfloat16, torch.float16]
CACHED = [torch.bfloat16, torch.float16, torch.int8]
# half a unit in the last place, relative, of one rounding to the type; the spacing of its smallest numbers
ROUND = {t: torch.finfo(t).eps / 2 for t in FLOATS}
LEAST = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}


def seeded(*key):
    return torch.Generator().manual_seed(hash(key) % (1 << 31))


def normal(shape, g, dtype=torch.float32):
    return torch.randn(shape, generator=g).to(dtype).cuda()


# ---- positions ----------------------------------------------------------------------------------------------------
def radians(dim, base=10000.0, scaling=None):
    """The definition, written apart."""
    i = torch.arange(dim // 2, dtype=torch.float64)
    f = torch.exp(-2 * i / dim * math.log(base))
    if scaling is None:
        return f, 1.0
    kind, factor = scaling[:2]
    if kind == "linear":
        return f / factor, 1.0
    if kind == "base":
        return f * torch.exp(-2 * i / max(dim - 2, 1) * math.log(factor)), 1.0
    low, high = scaling[3:] or (1.0, 32.0)
    part = ((scaling[2] * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
    return f * part + f / factor * (1 - part), 0.1 * math.log(factor) + 1


def turn64(x, positions, dim, interleaved, base=10000.0, scaling=None):
    """x (n, heads, d) on the CPU in 64 bits, the first dim columns turned."""
    f, amplitude = radians(dim, base, scaling)
    a = positions.double()[:, None] * f
    c, s = amplitude * torch.cos(a)[:, None], amplitude * torch.sin(a)[:, None]
    x = x.double().clone()
    u, w = (x[..., 0:dim:2], x[..., 1:dim:2]) if interleaved else (x[..., :dim // 2], x[..., dim // 2:dim])
    u, w = u * c - w * s, u * s + w * c
    x[..., :dim] = torch.stack((u, w), dim=-1).flatten(-2) if interleaved else torch.cat((u, w), dim=-1)
    return x


def turn_error(x, dim, interleaved, amplitude, far):
    """How far 32 bits may be: cosine and sine 6 units of 2^-24 each (series, reduction, amplitude), two products and a sum 2; and the angles of
    this test, which has 53 bits of them."""
    big = x.double().abs().clone()
    u, w = (big[..., 0:dim:2], big[..., 1:dim:2]) if interleaved else (big[..., :dim // 2], big[..., dim // 2:dim])
    t = (u + w) * amplitude * (8 * 2.0 ** -24 + far * 2.0 ** -50)
    big[..., :dim] = torch.stack((t, t), dim=-1).flatten(-2) if interleaved else torch.cat((t, t), dim=-1)
    big[..., dim:] = 0
    return big


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("n,heads,d,dim,interleaved,far,scaling", [
    (1, 1, 2, 2, False, 5, None), (1, 32, 128, 128, False, 4096, None), (3, 5, 64, 64, True, 4096, None), (7, 8, 128, 64, True, 1 << 20, ("parts", 16.0, 4096)),
    (5, 3, 80, 20, False, 100000, ("linear", 4.0)), (5, 3, 80, 20, True, 100000, ("base", 4.0)), (33, 2, 96, 96, False, 1 << 30, ("base", 8.0)), (2, 1, 256, 256, False, 4096, None),
    (17, 1, 256, 248, True, 4096, None), (1200, 12, 112, 16, False, 4096, ("parts", 8.0, 2048, 2.0, 20.0)), (1030, 40, 64, 64, True, 8192, None), (9, 20, 30, 6, True, 300, None), (4, 17, 128, 0, False, 10, None)])
def test_heads_are_turned(dtype, n, heads, d, dim, interleaved, far, scaling):
    g = seeded(n, heads, d, dim)
    x = normal((n, heads, d), g, dtype)
    positions = torch.randint(0, far, (n,), generator=g)
    positions[-1] = far - 1
    if dim == 0:
        plan = gen.RotaryPlan(gen.rotary_plan(2).steps[:0], 0, False, 1.0)
        got, want, off = gen.rotate_heads(x, positions.cuda(), plan), x.cpu().double(), 0.0
    else:
        plan = gen.rotary_plan(dim, interleaved=interleaved, scaling=scaling)
        got = gen.rotate_heads(x, positions.cuda(), plan)
        want = turn64(x.cpu(), positions, dim, interleaved, scaling=scaling)
        off = turn_error(x.cpu(), dim, interleaved, plan.amplitude, far)
    assert got.shape == x.shape and got.dtype == dtype and got.is_contiguous()
    assert ((got.cpu().double() - want).abs() <= off + ROUND[dtype] * (want.abs() + off) + LEAST[dtype]).all()


def test_heads_of_views_and_in_place():
    g = seeded(3)
    plan = gen.rotary_plan(64)
    positions = torch.arange(50).cuda() * 77
    x = normal((50, 3, 8, 96), g, torch.bfloat16)            # queries, keys and values of a projection beside each other
    want = gen.rotate_heads(x[:, 1, :, 16:].contiguous(), positions, plan)
    keep = x.clone()
    q = x[:, 1, :, 16:]
    assert torch.equal(gen.rotate_heads(q, positions, plan), want)
    assert gen.rotate_heads(q, positions, plan, out=q) is q and torch.equal(q, want)
    keep[:, 1, :, 16:] = want
    assert torch.equal(x, keep)                # nothing else
    heads_first = x[:, 1].transpose(0, 1).contiguous().transpose(0, 1)[:, :, :80]       # (tokens, heads, d), tokens next to each other; unaligned rows below
    odd = torch.zeros(50, 8, 81, dtype=torch.bfloat16, device="cuda")[:, :, 1:]
    odd.copy_(heads_first)
    assert torch.equal(gen.rotate_heads(odd, positions, plan), gen.rotate_heads(heads_first, positions, plan))
    one = normal((50, 1, 80), g).expand(50, 6, 80)
    assert torch.equal(gen.rotate_heads(one, positions, plan), gen.rotate_heads(one.contiguous(), positions, plan))


def test_positions_far_below_and_above():
    """The angle is exact mod a turn for any 64-bit position, and -p turns back."""
    plan = gen.rotary_plan(128)
    x = normal((4, 2, 128), seeded(1))
    p = torch.tensor([0, 1 << 40, -(1 << 40), (1 << 62) + 12345]).cuda()
    there = gen.rotate_heads(x, p, plan)
    assert torch.equal(there[0], x[0])
    back = gen.rotate_heads(there, -p, plan)
    assert (back - x).abs().max() <= 4 * 16 * 2.0 ** -24 * 6        # two turns of 16 units at entries up to 6
    steps = [int(w) % (1 << 64) for w in plan.steps.tolist()]
    turns = [(int(p[3]) * w % (1 << 64)) / 2.0 ** 64 for w in steps]
    a = torch.tensor(turns, dtype=torch.float64) * 2 * math.pi
    u, w = x[3, :, :64].cpu().double(), x[3, :, 64:].cpu().double()
    want = torch.cat((u * a.cos() - w * a.sin(), u * a.sin() + w * a.cos()), dim=1)
    assert ((there[3].cpu().double() - want).abs() <= 12 * 2.0 ** -24 * 8).all()


# ---- the cache ----------------------------------------------------------------------------------------------------
class Made:
    """Sequences with `before` entries each and `new` more, their pages in no order, and two pages that nobody has; entries are random."""

    def __init__(self, dtype, before, new, heads, dim, page, seed=0, layout=0, gap=0, spare=0):
        g = seeded(dtype.itemsize, len(before), heads, dim, page, seed)
        self.before, self.new, self.page = before, new, page
        lengths = [b + n for b, n in zip(before, new)]
        width = max([-(-x // page) for x in lengths] + [0]) + spare
        need = sum(-(-x // page) for x in lengths)
        self.pages = need + 2
        shape = (self.pages, heads, page, dim)
        made = []
        for _ in range(2):
            x = torch.randint(-127, 128, shape, generator=g).to(torch.int8) if dtype == torch.int8 else torch.randn(shape, generator=g).to(dtype)
            made.append(x.cuda())
        if layout == 1:                        # entries of all heads beside each other, as (pages, rows, heads, dim)
            made = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in made]
        if layout == 2:                        # keys and values of an entry beside each other
            both = torch.cat(made, dim=3)
            made = [both[..., :dim], both[..., dim:]]
        scales = [None, None]
        if dtype == torch.int8:
            scales = [(torch.rand(shape[:3], generator=g) * 0.02 + 0.01).cuda() for _ in range(2)]
        self.cache = gen.Cache(made[0], made[1], *scales)
        order = torch.randperm(self.pages, generator=g)[:need].tolist()
        table = torch.full((len(before), width), -1, dtype=torch.int32)
        for b, x in enumerate(lengths):
            for i in range(-(-x // page)):
                table[b, i] = order.pop()
        self.table = table
        self.starts = [gap + sum(new[:b]) for b in range(len(new) + 1)]
        self.n = self.starts[-1] + gap
        self.batch = gen.Batch(torch.tensor(self.starts, dtype=torch.int32).cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), table.cuda())

    def places(self, b, numbers):
        """Page and row of entries of sequence b."""
        j = torch.as_tensor(numbers)
        return self.table[b][j // self.page].long(), j % self.page

    def held(self, b, name, count):
        """(count, heads, dim) of the cache in 64 bits."""
        page, row = self.places(b, torch.arange(count))
        x = getattr(self.cache, name)[page.cuda(), :, row.cuda()].cpu().double()
        s = getattr(self.cache, name[:-1] + "_scales")
        return x if s is None else x * s[page.cuda(), :, row.cuda()].cpu().double()[..., None]


def held_bits(cache):
    """All that a cache holds, to compare."""
    return [t.clone() for t in (cache.keys, cache.values, cache.key_scales, cache.value_scales) if t is not None]


APPENDS = [([0], [1], 1, 128, 16, 0), ([5], [3], 8, 128, 16, 0), ([0, 15, 16, 31], [1, 1, 1, 1], 4, 64, 16, 1), ([100, 0, 7], [0, 40, 17], 3, 80, 32, 2), ([3], [700], 2, 256, 64, 0),
           ([1000] * 70, [1] * 70, 1, 48, 128, 0), ([0, 0], [129, 500], 32, 128, 16, 0)]


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("cached", CACHED)
@pytest.mark.parametrize("before,new,heads,dim,page,layout", APPENDS)
def test_tokens_are_appended(dtype, cached, before, new, heads, dim, page, layout):
    m = Made(cached, before, new, heads, dim, page, layout=layout, gap=2)
    g = seeded(9, len(new), dim)
    k, v = normal((m.n, heads, dim), g, dtype), normal((m.n, heads, dim), g, dtype)
    rotated = {128: 128, 64: 32, 80: 20, 256: 256, 48: 48}[dim]
    plan = gen.rotary_plan(rotated, interleaved=dim == 64)
    # what should be there, by the definition, over what is
    want = held_bits(m.cache)
    number = torch.cat([torch.zeros(2, dtype=torch.long)] + [torch.arange(b, b + x) for b, x in zip(before, new)] + [torch.zeros(2, dtype=torch.long)])
    turned = turn64(k.cpu(), number, rotated, dim == 64)
    off = turn_error(k.cpu(), rotated, dim == 64, 1.0, 4096) if cached != torch.int8 else torch.zeros(1, dtype=torch.float64)
    gen.append_tokens(m.cache, k, v, m.batch, plan=plan)
    got = held_bits(m.cache)
    for b, count in enumerate(new):
        if not count:
            continue
        rows = slice(m.starts[b], m.starts[b + 1])
        page_, row = (t.cuda() for t in m.places(b, torch.arange(before[b], before[b] + count)))
        if cached == torch.int8:
            for i, x in enumerate((turned[rows].float(), v[rows].cpu().float())):
                q, s = inf.quantize_rows(x.reshape(-1, dim).cuda())
                here, scale = got[i][page_, :, row], got[2 + i][page_, :, row]
                # 64 bits of an angle decide the same integers, but where they round to another 32 bits: 2^-27 of the keys
                assert (here.int() - q.view(count, heads, dim).int()).abs().max() <= (0 if i else 1)
                assert (here != q.view(count, heads, dim)).sum() <= (0 if i else 2)
                s = s.view(count, heads)
                assert torch.equal(scale, s) if i else ((scale - s).abs() <= s * 2.0 ** -23).all()
                want[i][page_, :, row], want[2 + i][page_, :, row] = here, scale
        else:
            here = got[0][page_, :, row]
            assert ((here.cpu().double() - turned[rows]).abs() <= off[rows] + ROUND[cached] * (turned[rows].abs() + off[rows]) + LEAST[cached]).all()
            want[0][page_, :, row] = here
            want[1][page_, :, row] = v[rows].to(cached)
    for a, b in zip(got, want):
        assert torch.equal(a, b)               # nothing else was written


def test_appended_positions_and_none():
    m, other = (Made(torch.bfloat16, [3, 20], [5, 9], 2, 64, 16) for _ in range(2))
    k, v = normal((m.n, 2, 64), seeded(4), torch.bfloat16), normal((m.n, 2, 64), seeded(5), torch.bfloat16)
    positions = torch.tensor([3, 4, 4, 5, 5] + [20 + i // 3 for i in range(9)]).cuda()
    plan = gen.rotary_plan(64)
    gen.append_tokens(m.cache, k, v, m.batch, positions=positions, plan=plan)
    gen.append_tokens(other.cache, gen.rotate_heads(k, positions, plan), v, other.batch)
    assert all(torch.equal(a, b) for a, b in zip(held_bits(m.cache), held_bits(other.cache)))


def test_appending_skips_pages_that_are_none():
    m = Made(torch.float16, [0, 30], [40, 20], 2, 64, 16)
    for bad in (-1, m.pages, m.pages + 1000, -(1 << 31)):
        table = m.table.clone()
        table[0, 1], table[1, 2] = bad, bad
        batch = gen.Batch(m.batch.starts, m.batch.lengths, table.cuda())
        was = held_bits(m.cache)
        k, v = normal((60, 2, 64), seeded(bad & 255), torch.float16), normal((60, 2, 64), seeded(5), torch.float16)
        gen.append_tokens(m.cache, k, v, batch)
        now = held_bits(m.cache)
        gone = 0
        for b, (first, count) in enumerate(((0, 40), (30, 20))):
            for i in range(count):
                j = first + i
                page, row = int(table[b, j // 16]), j % 16
                if page == bad:
                    gone += 1
                    continue
                was[0][page, :, row], was[1][page, :, row] = k[m.starts[b] + i], v[m.starts[b] + i]
        assert gone == 16 + 16 and all(torch.equal(a, b) for a, b in zip(was, now))


def test_rows_that_are_hard_to_cache():
    """Zeros, infinities, NaN and the smallest numbers in 8 bits, as quantize_rows has them."""
    m = Made(torch.int8, [0], [8], 1, 64, 16)
    v = normal((8, 1, 64), seeded(1))
    v[0], v[1, 0, 5], v[2, 0, 63], v[3], v[4, 0, 1] = 0, math.inf, math.nan, 1e-39, -math.inf
    v[5] = torch.arange(64) / 2 - 16
    v[5, 0, 0] = 127
    gen.append_tokens(m.cache, v, v, m.batch)
    q, s = inf.quantize_rows(v[:, 0])
    page, row = m.places(0, torch.arange(8))
    for name in ("key", "value"):
        assert torch.equal(getattr(m.cache, name + "s")[page.cuda(), 0, row.cuda()], q)
        assert torch.equal(getattr(m.cache, name + "_scales")[page.cuda(), 0, row.cuda()].nan_to_num(-7.0), s.nan_to_num(-7.0))


# ---- attention ----------------------------------------------------------------------------------------------------
def ancestors(parents):
    """(n, n): whether j is i or above it."""
    n = len(parents)
    seen = torch.eye(n, dtype=torch.bool)
    for i, p in enumerate(parents):
        if 0 <= p < i:
            seen[i] |= seen[p]
    return seen


def attend64(m, q, group, parents=None, scale=None, missing=()):
    """In 64 bits; also sum of p |v|, which errors are relative to, and how far 32-bit sums may take a score."""
    n, heads, dim = q.shape
    scale = dim ** -0.5 if scale is None else scale
    out, size, far = torch.zeros(n, heads, dim, dtype=torch.float64), torch.zeros(n, heads, dim, dtype=torch.float64), 0.0
    for b, count in enumerate(m.new):
        if not count:
            continue
        rows, length = slice(m.starts[b], m.starts[b + 1]), m.before[b] + count
        k, v = m.held(b, "keys", length).cuda(), m.held(b, "values", length).cuda()
        allowed = torch.ones(count, length, dtype=torch.bool)
        allowed[:, m.before[b]:] = torch.ones(count, count, dtype=torch.bool).tril() if parents is None or count > 256 else ancestors(parents[rows])
        for j in missing:
            if j[0] == b:
                allowed[:, j[1]:j[2]] = False
        x = q[rows].double().view(count, heads // group, group, dim)
        for h in range(heads // group):
            xx = x[:, h].reshape(-1, dim)
            s = (xx @ k[:, h].T.contiguous()) * scale
            far = max(far, float((xx.abs() @ k[:, h].abs().T.contiguous()).nan_to_num(0.0, 0.0, 0.0).max()) * scale * dim * 2.0 ** -24)
            mask = allowed.cuda().repeat_interleave(group, dim=0)
            s = torch.where(mask, s, -math.inf)
            p = torch.exp(s - torch.where(mask.any(1), s.amax(1), 0.0)[:, None])
            p = torch.where(mask, p, 0.0)
            p = p / torch.where(mask.any(1), p.sum(1), 1.0)[:, None]
            for o, w in ((out, v[:, h]), (size, v[:, h].abs())):
                y = p @ w.nan_to_num(0.0, 0.0, 0.0)
                for bad in (math.inf, -math.inf, math.nan):          # what no mask hides shows
                    here = w == bad if bad == bad else w != w
                    if here.any():
                        y = torch.where((mask.double() @ here.double()) > 0, y + bad, y)
                o[rows, h * group:(h + 1) * group] = y.view(count, group, dim).cpu()
    return out, size, far


def check_attention(m, q, group, parents=None, scale=None, missing=(), **more):
    got = gen.attend_cache(q, m.cache, m.batch, parents=None if parents is None else torch.tensor(parents, dtype=torch.int32).cuda(), scale=scale, **more)
    want, size, far = attend64(m, q, group, parents, scale, missing)
    r = ROUND[q.dtype]
    # P rounded once (with the value's scale, for 8 bits), exponentials and their sums 2^-20 off with scores `far` off, the result rounded
    off = (r * (1 + 2.0 ** -6) + 4 * far + 2.0 ** -20) * size + LEAST[q.dtype] * 256
    got = got.cpu().double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
    bad = ((got - want).abs() > off + r * (want.abs() + off)) & fine
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:5].tolist(), got[bad][:5].tolist(), want[bad][:5].tolist())
    return got


def tree(count, g, wide=1):
    return [-1] + [int(torch.randint(max(0, (i - 1) // 4), i, (1,), generator=g)) if i > wide else 0 for i in range(1, count)]


# before, new, heads of the cache, group, dim, page
ATTENDS = [([0], [1], 1, 1, 128, 16), ([6], [1], 2, 4, 128, 16), ([1000], [1], 8, 4, 128, 16), ([31, 32, 33, 500, 0], [1] * 5, 2, 7, 64, 32), ([4095, 17, 2047], [1] * 3, 1, 8, 80, 64),
           ([100], [17], 2, 3, 96, 16), ([0], [64], 1, 1, 128, 64), ([3, 2000], [25, 9], 2, 4, 128, 128), ([0, 0, 5], [33, 1, 0], 3, 2, 256, 16), ([63], [5], 1, 16, 256, 1024),
           ([0], [300], 2, 1, 128, 16), ([77, 0], [200, 129], 1, 5, 64, 32), ([1000], [257], 1, 2, 112, 64), ([3000], [1], 1, 40, 128, 16), ([0, 10], [130, 100], 2, 3, 256, 32),
           ([0], [1000], 1, 4, 16, 16), ([900], [65], 2, 1, 240, 16)]


@pytest.mark.parametrize("cached", CACHED)
@pytest.mark.parametrize("before,new,heads,group,dim,page", ATTENDS)
def test_attention_over_the_cache(cached, before, new, heads, group, dim, page):
    dtype = torch.float16 if cached == torch.float16 else torch.bfloat16
    m = Made(cached, before, new, heads, dim, page, layout=len(before) % 3, gap=1)
    q = normal((m.n, heads * group, dim), seeded(2, dim, len(new)), dtype)
    got = check_attention(m, q, group)
    assert (got[0] == 0).all() and (got[-1] == 0).all()                # of no sequence
    check_attention(m, q, group, longest=0)    # a hint that is wrong costs time, nothing else


@pytest.mark.parametrize("cached", CACHED)
@pytest.mark.parametrize("dim", [48, 64, 128, 208, 256])
@pytest.mark.parametrize("new,group", [([1, 3], 2), ([100, 1], 1)])
def test_attention_in_many_parts(cached, dim, new, group):
    """Few heads over long sequences, cut as the longest that there may be says, which may be wrong."""
    m = Made(cached, [5000, 1100], new, 1, dim, 64)
    q = normal((m.n, group, dim), seeded(dim, group), torch.float16 if cached == torch.float16 else torch.bfloat16)
    for longest in (None, 0, 700, 1 << 30):
        check_attention(m, q, group, longest=longest)


@pytest.mark.parametrize("cached", CACHED)
@pytest.mark.parametrize("before,new,heads,group,dim,page", [([100], [17], 2, 3, 96, 16), ([3, 2000], [25, 9], 2, 4, 128, 128), ([0, 37, 5], [33, 1, 64], 3, 1, 64, 16),
                                                             ([15, 700], [256, 100], 1, 2, 128, 16), ([40, 0], [100, 300], 2, 1, 128, 32), ([9], [20], 1, 8, 256, 16)])
def test_attention_of_trees(cached, before, new, heads, group, dim, page):
    dtype = torch.float16 if cached == torch.float16 else torch.bfloat16
    m = Made(cached, before, new, heads, dim, page)
    g = seeded(8, dim, len(new))
    q = normal((m.n, heads * group, dim), g, dtype)
    check_attention(m, q, group, parents=sum((tree(x, g) for x in new), []))
    wild = torch.randint(-3, 300, (m.n,), generator=g).tolist()        # numbers that are no parents make roots
    check_attention(m, q, group, parents=wild)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,group", [(40, 1), (40, 2), (200, 1)])
def test_what_a_mask_hides_does_not_show(dtype, tokens, group):
    """Infinities and NaN in keys and values that a token does not attend to, on pages behind the end too."""
    m = Made(dtype, [21], [tokens], 2, 128, 16)
    page, row = m.places(0, [21 + 7, 21 + 8, 21 + 30, 21 + 31])
    page, row = page.cuda(), row.cuda()
    m.cache.values[page[0], 0, row[0], 3] = math.inf
    m.cache.values[page[1], 0, row[1], 3] = -math.inf
    m.cache.values[page[1], 0, row[1], 9] = -math.inf
    m.cache.values[page[2], 1, row[2], 100] = math.nan
    m.cache.keys[page[3], 1, row[3], 5] = math.nan
    length = 21 + tokens
    if length % 16:
        p = int(m.table[0, length // 16])
        m.cache.values[p, :, length % 16:] = math.nan
        m.cache.keys[p, :, length % 16:] = math.inf
    q = normal((m.n, 2 * group, 128), seeded(6), dtype)
    # a NaN key makes the scores of those that see it NaN, and all they get
    want, _, _ = attend64(m, q, group)
    got = gen.attend_cache(q, m.cache, m.batch).cpu().double()
    sees = torch.arange(tokens) >= 31
    for h in range(2 * group):
        second = h >= group
        for cols in (3, 9, 100, 50):
            a, b = got[:, h, cols], want[:, h, cols]
            if second:
                assert torch.isnan(a[sees]).all()
                a, b = a[~sees], b[~sees]
            assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.isinf(a), torch.isinf(b)), (h, cols)
            f = torch.isfinite(b)
            assert ((a - b).abs()[f] < 0.05).all()


def test_scales_that_are_nan_show_where_they_count():
    m = Made(torch.int8, [10], [30], 1, 64, 16)
    page, row = m.places(0, [10 + 12])
    m.cache.value_scales[page.cuda(), 0, row.cuda()] = math.nan
    q = normal((30, 1, 64), seeded(7), torch.bfloat16)
    got = gen.attend_cache(q, m.cache, m.batch)
    assert torch.isnan(got[12:]).all() and torch.isfinite(got[:12]).all()


@pytest.mark.parametrize("cached", CACHED)
def test_attention_skips_pages_that_are_none(cached):
    dtype = torch.float16 if cached == torch.float16 else torch.bfloat16
    m = Made(cached, [200, 1500], [1, 40], 2, 128, 16)
    good = m.table.clone()
    for bad in (-1, m.pages, 1 << 30):
        m.batch = gen.Batch(m.batch.starts, m.batch.lengths, torch.where(torch.isin(torch.arange(good.shape[1]), torch.tensor([3, 7, 90])), bad, good).int().cuda())
        q = normal((41, 4, 128), seeded(bad & 63), dtype)
        check_attention(m, q, 2, missing=[(b, 16 * p, 16 * p + 16) for b in (0, 1) for p in (3, 7, 90)])


def test_tokens_that_attend_to_nothing():
    m = Made(torch.bfloat16, [0, 0], [5, 40], 1, 64, 16)
    q = normal((45, 3, 64), seeded(1), torch.bfloat16)
    none = torch.full_like(m.table, -1).cuda()
    assert (gen.attend_cache(q, m.cache, gen.Batch(m.batch.starts, m.batch.lengths, none)) == 0).all()
    zero = torch.zeros(2, dtype=torch.int32, device="cuda")
    assert (gen.attend_cache(q, m.cache, gen.Batch(m.batch.starts, zero, m.batch.pages)) == 0).all()
    empty = gen.attend_cache(q, m.cache, gen.Batch(m.batch.starts, m.batch.lengths, torch.empty((2, 0), dtype=torch.int32, device="cuda")))
    assert (empty == 0).all()
    # fewer entries than new tokens: the first ones have none, the others what is there
    few = gen.attend_cache(q, m.cache, gen.Batch(m.batch.starts, torch.tensor([2, 40], dtype=torch.int32, device="cuda"), m.batch.pages))
    assert (few[:3] == 0).all() and (few[3:5] != 0).any()


def test_attention_writes_where_it_should():
    m = Made(torch.bfloat16, [50, 3], [2, 30], 2, 64, 16, gap=3)
    q = normal((m.n, 4, 64), seeded(1), torch.bfloat16)
    want = gen.attend_cache(q, m.cache, m.batch)
    out = torch.full((m.n, 2, 4, 70), 7.0, dtype=torch.bfloat16, device="cuda")
    view = out[:, 1, :, 3:67]
    assert gen.attend_cache(q, m.cache, m.batch, out=view) is view
    assert torch.equal(view[3:-3], want[3:-3])
    out[3:-3, 1, :, 3:67] = 7.0
    assert (out == 7.0).all()
    wide = torch.zeros((m.n, 4, 192), dtype=torch.bfloat16, device="cuda")[:, :, 64:128]
    wide.copy_(q)
    assert torch.equal(gen.attend_cache(wide, m.cache, m.batch), want)


@pytest.mark.parametrize("new", [[3, 1], [40, 70]])
@pytest.mark.parametrize("low,high", [(-110, -90), (-60, 60), (60, 90), (-2, 2)])
def test_value_scales_of_any_size(new, low, high):
    """Scales that differ by 2^(high - low) from entry to entry, some of them 0; a token does not see those behind it, however large."""
    m = Made(torch.int8, [300, 20], new, 2, 128, 16)
    g = seeded(low, high)
    power = torch.randint(low, high + 1, m.cache.value_scales.shape, generator=g)
    scales = torch.ldexp(torch.rand(power.shape, generator=g) + 1, power)
    scales[torch.rand(power.shape, generator=g) < 0.1] = 0.0
    m.cache.value_scales.copy_(scales)
    q = normal((m.n, 4, 128), g, torch.bfloat16)
    got, (want, size, far) = gen.attend_cache(q, m.cache, m.batch, scale=0.3).cpu().double(), attend64(m, q, 2, scale=0.3)
    # Where a column's values of the largest weights are 0 or small, `size` is small beside what these weights are rounded with.  The weights p f are fp16, the largest of
    # a row 1 or more: each is 2^-12 of itself off, or 2^-25 of the largest where that is more, times values up to 128.  Their sums in 32 bits, a rounding a product of
    # 16 keys and eight for those of partial sums, are of values up to 256: with W the sum of the weights, count 2^-25 128 W + (count / 16 + 8) 2^-24 256 W.
    m.cache.values.fill_(1)
    whole, count = attend64(m, q, 2, scale=0.3)[0], 300 + new[0]
    r = ROUND[torch.bfloat16]
    off = (r + 4 * far + 2.0 ** -20) * size + (count * 2.0 ** -18 + (count / 16 + 8) * 2.0 ** -16) * whole + LEAST[torch.bfloat16]
    assert ((got - want).abs() <= off + r * (want.abs() + off)).all()


@pytest.mark.parametrize("power", [-120, -30, 30, 110])
def test_queries_of_any_size(power):
    """Rows whose queries differ in size, with scales of keys that bring their scores back."""
    m = Made(torch.int8, [100], [40], 1, 96, 16)
    q = normal((40, 2, 96), seeded(power), torch.bfloat16)
    q[::3] *= 2.0 ** -20
    far = torch.ldexp(q.double(), torch.tensor(power).cuda()).to(torch.bfloat16)
    q = torch.ldexp(far.double(), torch.tensor(-power).cuda()).to(torch.bfloat16)      # without the digits that bfloat16 has not down there
    want = gen.attend_cache(q, m.cache, m.batch)
    m.cache.key_scales.copy_(torch.ldexp(m.cache.key_scales, torch.tensor(-power).cuda()))
    got = gen.attend_cache(far, m.cache, m.batch)
    assert torch.equal(got[1::3], want[1::3]) and torch.equal(got[2::3], want[2::3])
    assert ((got - want).abs().float() <= 2.0 ** -8 * 2 * 4).all()     # two roundings of values up to 4; the small queries may have lost digits


def test_large_scores():
    """Scores up to 10^4, one far above the rest, and equal ones."""
    m = Made(torch.bfloat16, [700], [1], 1, 128, 16)
    m.cache.keys.mul_(30.0)
    q = normal((1, 2, 128), seeded(1), torch.bfloat16) * 30
    got = gen.attend_cache(q, m.cache, m.batch, scale=0.1).cpu().double()
    want, size, far = attend64(m, q, 2, scale=0.1)
    assert ((got - want).abs() <= ROUND[torch.bfloat16] * 2.1 * size + 8 * far * size).all()
    m.cache.keys.zero_()
    check_attention(m, q, 2)


def test_offsets_beyond_32_bits():
    """A cache of 9 GB, the sequence on its last pages."""
    pages, heads, size, dim = 4400, 16, 256, 128
    keys = torch.empty((pages, 2, heads, size, dim), dtype=torch.bfloat16, device="cuda")
    cache = gen.Cache(keys[:, 0], keys[:, 1])
    table = torch.tensor([[pages - 1, pages - 3, 0, pages - 2]], dtype=torch.int32).cuda()
    k, v = normal((1000, heads, dim), seeded(1), torch.bfloat16), normal((1000, heads, dim), seeded(2), torch.bfloat16)
    batch = gen.Batch(torch.tensor([0, 1000], dtype=torch.int32).cuda(), torch.tensor([1000], dtype=torch.int32).cuda(), table)
    gen.append_tokens(cache, k, v, batch)
    small = gen.new_cache(4, heads, size, dim)
    alike = gen.Batch(batch.starts, batch.lengths, torch.arange(4, dtype=torch.int32, device="cuda")[None])
    gen.append_tokens(small, k, v, alike)
    q = normal((1000, heads, dim), seeded(3), torch.bfloat16)
    assert torch.equal(gen.attend_cache(q, cache, batch), gen.attend_cache(q, small, alike))
    assert torch.equal(cache.keys[pages - 2, :, :232], k[768:].transpose(0, 1))


# ---- drafts -------------------------------------------------------------------------------------------------------
def verify64(logits, tokens, starts, parents, u, depth, draft, temperature):
    """One node after the other, in 64 bits."""
    v = logits.shape[1]
    counts, nodes, out = [], [], []
    for s0, s1 in zip(starts, starts[1:]):
        if s1 <= s0:
            counts.append(0), nodes.append([-1] * depth), out.append([-1] * (depth + 1))
            continue

        def p_of(x, i):
            z = x[s0 + i].double() / temperature
            good = (z < math.inf).all() and (z > -math.inf).any()
            e = torch.exp(z - z.max())             # torch.softmax on the GPU has no probabilities below 2^-126
            return e / e.sum() if good else None

        path, p = [0], p_of(logits, 0)
        first = p
        q = None if draft is None else p_of(draft, 0)
        for i in range(1, min(s1 - s0, 1024)):
            up, x = parents[s0 + i], tokens[s0 + i]
            if up != path[-1] or len(path) > depth or not 0 <= x < v or p is None or (draft is not None and q is None):
                continue
            said = 1.0 if draft is None else float(q[x])
            if u[s0 + i] * said * float(p.sum()) < float(p[x]):
                path.append(i)
                first = p = p_of(logits, i)
                q = None if draft is None else p_of(draft, i)
            elif draft is None:
                p = p.clone()
                p[x] = 0
            else:
                p = (p / p.sum() - q).clamp(min=0) if p.sum() > 0 else p
        last = -1
        if p is not None:
            p = p if p.sum() > 0 else first
            c = p.cumsum(0)
            last = int((c <= u[s0] * c[-1]).sum())
            if last == v:
                last = int(p.nonzero()[-1])
        counts.append(len(path) - 1)
        nodes.append((path[1:] + [-1] * depth)[:depth])
        out.append(([tokens[s0 + i] for i in path[1:]] + [last] + [-1] * depth)[:depth + 1])
    return counts, nodes, out


def draft_case(sequences, count, v, dtype, drafted, seed, near=1.0, chain=False, temperature=1.0):
    g = seeded(sequences, count, v, drafted, seed)
    starts = [i * count for i in range(sequences + 1)]
    n = starts[-1]
    logits = (torch.randn(n, v, generator=g) * 3).to(dtype)
    draft = (logits.float() + torch.randn(n, v, generator=g) * near).to(dtype)
    parents = sum(([i - 1 for i in range(count)] if chain else tree(count, g) for _ in range(sequences)), [])
    at = torch.tensor([max(p, 0) + i // count * count for i, p in enumerate(parents)])
    noise = -torch.log(-torch.log(torch.rand(n, v, generator=g).clamp(min=1e-12)))
    tokens = (draft[at].float() / temperature + noise).argmax(1).tolist()
    u = torch.rand(n, generator=g, dtype=torch.float64)
    return logits, tokens, starts, parents, u, draft if drafted else None


def check_drafts(logits, tokens, starts, parents, u, draft, depth, temperature=1.0, chain=False, pad=0):
    def rows(t):
        if t is None or not pad:
            return None if t is None else t.cuda()
        wide = torch.full((t.shape[0], t.shape[1] + pad), 50.0, dtype=t.dtype, device="cuda")
        wide[:, :t.shape[1]] = t.cuda()
        return wide[:, :t.shape[1]]

    counts, nodes, out = gen.verify_drafts(rows(logits), torch.tensor(tokens, dtype=torch.int64).cuda(), torch.tensor(starts, dtype=torch.int32).cuda(),
                                           None if chain else torch.tensor(parents, dtype=torch.int32).cuda(), u.cuda(), depth, draft_logits=rows(draft), temperature=temperature)
    wc, wn, wo = verify64(logits.cuda(), tokens, starts, parents, u.tolist(), depth, None if draft is None else draft.cuda(), temperature)
    assert counts.tolist() == wc and nodes.tolist() == wn and out.tolist() == wo
    return wc


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("drafted", [False, True])
@pytest.mark.parametrize("sequences,count,v,depth,temperature,pad", [(1, 1, 1, 3, 1.0, 0), (2, 2, 3, 2, 1.0, 1), (3, 5, 100, 4, 0.7, 0), (1, 5, 32000, 4, 1.0, 0), (20, 9, 511, 3, 1.3, 3),
                                                                     (7, 16, 5003, 8, 1.0, 5), (2, 60, 513, 256, 1.0, 0), (2, 8, 100000, 2, 1.0, 0), (5, 4, 2049, 0, 1.0, 0)])
def test_drafts_are_verified(dtype, drafted, sequences, count, v, depth, temperature, pad):
    for chain in (False, True):
        case = draft_case(sequences, count, v, dtype, drafted, depth, chain=chain, temperature=temperature)
        check_drafts(*case, depth, temperature, chain, pad)


def test_many_siblings_are_refused_one_after_the_other():
    """All drafts hang on the root, drawn from a draft model that is far off."""
    accepted = set()
    for drafted in (False, True):
        logits, tokens, starts, _, u, draft = draft_case(30, 12, 300, torch.float32, drafted, 1, near=6.0)
        parents = ([-1] + [0] * 11) * 30
        root = torch.tensor([i // 12 * 12 for i in range(360)])
        noise = -torch.log(-torch.log(torch.rand(360, 300, generator=seeded(5))))
        tokens = ((logits * 0.2 if draft is None else draft)[root] + noise).argmax(1).tolist()
        tokens[3], tokens[14] = tokens[2], tokens[13]                  # the same twice
        accepted.add(tuple(check_drafts(logits, tokens, starts, parents, u, draft, 5)))
    assert len(accepted) == 2 and all(0 in a and 1 in a for a in accepted)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("v", [5000, 33000, 150001])
def test_refusals_leave_less_and_less(dtype, v):
    """Siblings that the draft model thinks likelier than the target does are refused; what is left of long rows does not fit into one place."""
    g = seeded(v)
    logits, draft = ((torch.randn(20, v, generator=g) * 3).to(dtype) for _ in range(2))
    tokens, parents = [], []
    for s0 in (0, 10):
        likelier = (torch.softmax(logits[s0].double(), 0) / torch.softmax(draft[s0].double(), 0)).argsort()
        tokens += likelier[:5].tolist() + likelier[v // 2 - 2:v // 2 + 2].tolist() + [int(likelier[-1])]
        parents += [-1] + [0] * 9
    u = torch.rand(20, generator=g, dtype=torch.float64) * 0.5 + 0.5
    check_drafts(logits, tokens, [0, 10, 20], parents, u, draft, 4)
    u[9] = u[19] = 1.0 - 2.0 ** -53            # the last ones refused as well, it may be: the token from what is left
    check_drafts(logits, tokens, [0, 10, 20], parents, u, draft, 4, temperature=0.7)


def test_drafts_that_are_hard_to_verify():
    inf_, v = math.inf, 70
    logits, tokens, starts, parents, u, draft = draft_case(12, 6, v, torch.float32, True, 3)
    logits[0] = -inf_                          # a root without probabilities
    logits[6, 5], logits[12, 5] = math.nan, inf_
    draft[18, 3] = math.nan                    # the draft's
    logits[24, 1:] = -inf_                     # one token
    logits[30] = torch.finfo(torch.float32).min
    logits[30, 7:9] = 0                        # masked with the type's lowest
    tokens[37], tokens[38] = -1, v             # tokens that are none
    parents[43], parents[44], parents[45] = 1, 5, -2                   # parents that are none
    u[48], u[49] = 0.0, 0.0
    u[54], u[55:60] = 1.0 - 2.0 ** -53, 1.0 - 2.0 ** -53
    draft[60:66] = logits[60:66]               # the same probabilities: always accepted
    for d in (draft, None):
        check_drafts(logits, tokens, starts, parents, u, d, 4)
    check_drafts(logits, tokens, [0, 0, 6, 6, 40, 72], parents, u, draft, 3)           # sequences of nothing, and of other lengths
    check_drafts(logits, tokens, [5, 9], parents, u, draft, 3)                         # rows of no sequence


def test_rows_that_rise_and_fall():
    """Logits over many powers of two, in an order in which the largest come last, first or anywhere, in long rows."""
    for v in (5000, 200001):
        up = torch.linspace(-300, 300, v)
        logits = torch.stack((up, up.flip(0), up[torch.randperm(v, generator=seeded(v))], up * 0.01))
        draft = logits + torch.randn(4, v, generator=seeded(v, 1))
        draft[1, :v // 2] = -math.inf
        u = torch.rand(4, generator=seeded(v, 2), dtype=torch.float64)
        for tokens in ([0, v - 1, 0, 5], [0, 3, int(logits[2].argmax()), 7]):
            for d in (draft, None):
                check_drafts(logits, tokens, [0, 4], [-1, 0, 0, 0], u, d, 3)
                check_drafts(logits, tokens, [0, 4], [-1, 0, 1, 2], u, d, 3, temperature=30.0)


def test_a_refused_token_of_everything():
    """Nothing is left behind the refusal of all that there is: the target's own probabilities."""
    logits = torch.full((2, 9), -math.inf)
    logits[:, 4] = 1.0
    u = torch.tensor([0.5, 1.0], dtype=torch.float64)
    for draft in (None, logits):
        c, n, o = gen.verify_drafts(logits.cuda(), torch.tensor([0, 4]).cuda(), torch.tensor([0, 2], dtype=torch.int32).cuda(), None, u.cuda(), 1,
                                    draft_logits=None if draft is None else draft.cuda())
        assert c.tolist() == [0] and n.tolist() == [[-1]] and o.tolist() == [[4, -1]]


def test_tokens_come_as_often_as_the_target_says():
    """10^5 sequences of one draft: the token behind the root, accepted or not, is distributed as p, whatever q is."""
    n, v = 100000, 8
    g = seeded(11)
    logits, draft = (torch.randn(v, generator=g) * 1.5 for _ in range(2))
    p, q = torch.softmax(logits.double(), 0), torch.softmax(draft.double(), 0)
    x = torch.multinomial(q, n, replacement=True, generator=g)
    tokens = torch.stack((torch.zeros(n, dtype=torch.long), x), dim=1).flatten()
    u = torch.rand(2 * n, generator=g, dtype=torch.float64)
    _, _, out = gen.verify_drafts(logits.expand(2 * n, v).contiguous().cuda(), tokens.cuda(), (torch.arange(n + 1) * 2).int().cuda(), None, u.cuda(), 1,
                                  draft_logits=draft.expand(2 * n, v).contiguous().cuda())
    got = torch.bincount(out[:, 0].cpu(), minlength=v).double() / n
    assert ((got - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all()     # five standard deviations


# ---- the path's entries -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("cached", CACHED)
@pytest.mark.parametrize("before,new,depth,heads,dim,page", [([0], [1], 1, 1, 16, 16), ([1000], [25], 5, 8, 128, 16), ([15, 0, 100, 7], [20, 2, 0, 64], 9, 3, 80, 32), ([40] * 50, [9] * 50, 4, 2, 64, 64),
                                                             ([5], [400], 200, 1, 256, 16), ([3, 4], [30, 30], 0, 2, 64, 16)])
def test_accepted_entries_move_to_the_front(cached, before, new, depth, heads, dim, page):
    m = Made(cached, before, new, heads, dim, page, layout=len(before) % 3)
    rng = random.Random(len(before) * 100 + depth)
    nodes, counts = [], []
    for x in new:
        path = sorted(rng.sample(range(1, x), min(depth, x - 1))) if x > 1 else []
        nodes.append(path + [-1] * (depth - len(path)))
        counts.append(rng.choice([len(path), len(path), rng.randint(0, len(path))]))
    want = held_bits(m.cache)
    lengths = []
    for b, x in enumerate(new):
        for d in range(counts[b]):
            (p0, r0), (p1, r1) = m.places(b, before[b] + nodes[b][d]), m.places(b, before[b] + d + 1)
            for t in want:
                t[p1, :, r1] = t[p0, :, r0].clone()
        lengths.append(before[b] + 1 + counts[b] if x else before[b])
    got = gen.keep_drafts(m.cache, m.batch, torch.tensor(nodes, dtype=torch.int64).view(len(new), depth).cuda(), torch.tensor(counts).cuda())
    assert got.dtype == torch.int32 and got.tolist() == lengths
    assert all(torch.equal(a, b) for a, b in zip(held_bits(m.cache), want))


def test_paths_that_are_none_end():
    m = Made(torch.bfloat16, [7] * 6, [12] * 6, 2, 64, 16)
    nodes = torch.tensor([[3, 5, 4, 9], [12, 1, 2, 3], [-1, 2, 3, 4], [2, 2, 5, 6], [5, 8, 1 << 40, 9], [2, 4, 6, 8]]).cuda()
    counts = torch.tensor([4, 4, 3, 4, 4, 1 << 40]).cuda()
    want = held_bits(m.cache)
    taken = [2, 0, 0, 1, 2, 4]
    for b, k in enumerate(taken):
        for d in range(k):
            (p0, r0), (p1, r1) = m.places(b, 7 + int(nodes[b, d])), m.places(b, 8 + d)
            for t in want:
                t[p1, :, r1] = t[p0, :, r0].clone()
    assert gen.keep_drafts(m.cache, m.batch, nodes, counts).tolist() == [8 + k for k in taken]
    assert all(torch.equal(a, b) for a, b in zip(held_bits(m.cache), want))
    assert gen.keep_drafts(m.cache, m.batch, nodes, torch.full((6,), -5).cuda()).tolist() == [8] * 6
