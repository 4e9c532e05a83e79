"""Attention over the cache and drafts at the ends of numbers' ranges, against 64 bits."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from test_gpu_generation import CACHED, FLOATS, ROUND, Made, check_drafts, seeded  # noqa: E402
from verinf_amd.prover import generation as gen  # noqa: E402


# ---- attention ----------------------------------------------------------------------------------------------------
def with_scores(kind, scores, tokens=1, dim=128, seed=0):
    """Tokens whose queries are one in the first column, over keys that have `scores` there and nothing elsewhere; what comes before the tokens, and theirs."""
    m = Made(kind, [len(scores) - tokens], [tokens], 1, dim, 64, seed=seed)
    q = torch.zeros((tokens, 1, dim), dtype=torch.float16 if kind == torch.float16 else torch.bfloat16, device="cuda")
    q[:, :, 0] = 1
    page, row = (t.cuda() for t in m.places(0, torch.arange(len(scores))))
    m.cache.keys.zero_()
    m.cache.keys[page, 0, row, 0] = scores.to(kind).cuda()
    if kind == torch.int8:
        m.cache.key_scales.fill_(1.0)
    return m, q, page, row


def seen64(m, scores, tokens):
    """What each of the tokens sees: probabilities (tokens, entries) and values (entries, dim)."""
    count = len(scores)
    seen = torch.ones(tokens, count, dtype=torch.bool).tril(count - tokens)
    return torch.softmax(torch.where(seen, scores.double(), -math.inf), dim=1), m.held(0, "values", count)[:, 0]


@pytest.mark.parametrize("tokens", [1, 100])
@pytest.mark.parametrize("count", [301, 5000])
@pytest.mark.parametrize("value_scale", [0.02, 1.0, 3.0, 4.0, 100.0, 2.0 ** 60, 2.0 ** -60])
def test_keys_far_above_those_before_them(tokens, count, value_scale):
    """Over 8-bit integers, whose weights have a power of two of their own: with keys in one part and in several."""
    for ahead in (20, 86, 88, 95, 110, 127):
        for late in (0, 40, 190):
            scores = torch.zeros(count)
            scores[late] = ahead
            m, q, _, _ = with_scores(torch.int8, scores, tokens)
            m.cache.value_scales.fill_(value_scale)
            p, v = seen64(m, scores, tokens)
            want, size = p @ v, p @ v.abs()
            # Weights are fp16, half a step of them off or 2^-25 of the largest, times values up to 127; sums in 32 bits are of values up to 256; the result is bfloat16.
            off = (2.0 ** -11 + 2.0 ** -20) * size + (count * 2.0 ** -25 * 127 + (count / 16 + 8) * 2.0 ** -24 * 256) * value_scale
            r = ROUND[torch.bfloat16]
            for longest in (None, 0):
                got = gen.attend_cache(q, m.cache, m.batch, scale=1.0, longest=longest)[:, 0].cpu().double()
                assert ((got - want).abs() <= off + r * (want.abs() + off)).all(), (ahead, late, longest)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens", [1, 100])
@pytest.mark.parametrize("count,value", [(1024, 1.0), (301, 1000.0), (6000, 0.01)])
def test_weights_that_are_small_together(kind, tokens, count, value):
    """A key far ahead whose value is nothing, and what all the others' weights come to: wherever it is, in keys of one part and of several."""
    key_scale, value_scale = (0.15, value / 100) if kind == torch.int8 else (1.0, value)
    for ahead in (10.0, 15.0, 18.5, 20.5, 22.5, 25.1):
        for strong in (0, 40, count // 2, count - tokens):
            scores = torch.zeros(count)
            scores[strong] = round(ahead * math.log(2) / key_scale) if kind == torch.int8 else ahead * math.log(2)
            m, q, page, row = with_scores(kind, scores, tokens)
            m.cache.values.fill_(100 if kind == torch.int8 else value)
            m.cache.values[page[strong], 0, row[strong]] = 0
            if kind == torch.int8:
                m.cache.key_scales.fill_(key_scale)
                m.cache.value_scales.fill_(value_scale)
            exact = m.held(0, "keys", count)[strong, 0, 0]             # ahead by so much
            weight, v = torch.exp(-exact), m.held(0, "values", count)[(strong + 1) % count, 0, 0]
            others = (torch.arange(count - tokens, count) * weight)[:, None]
            want = v * others / (1 + others)
            # Weights are rounded to 16 bits, the other ones all alike: half a step of them, or fp16's 2^-25 where the largest is 2^7; scores and exponentials 2^-20; the result.
            bf16 = kind == torch.bfloat16
            rounding = ROUND[kind if bf16 else torch.float16] * weight + (0 if bf16 else 2.0 ** -32)
            off = want * (rounding / weight + 2.0 ** -20 * (1 + exact)) + (2.0 ** -25 if kind == torch.float16 else 0)
            for longest in (None, 0):
                got = gen.attend_cache(q, m.cache, m.batch, scale=1.0, longest=longest)
                assert ((got[:, 0].cpu().double() - want).abs() <= off + ROUND[got.dtype] * (want + off)).all(), (ahead, strong, longest)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [48, 64, 128, 256])
@pytest.mark.parametrize("tokens", [1, 100])
def test_values_all_alike_come_out_as_they_are(kind, dim, tokens):
    """What is added up of weights is what is multiplied: sums are 2^-20 off, which does not move a number of 16 bits."""
    g = seeded(dim, tokens, 45)
    for count in (230, 4000):
        # one late key that counts for nearly all, its weight relative to the first
        late = [torch.tensor([0.0] + [-30.0] * (at - 1) + [x] + [-30.0] * (count - at - 1)) for x in (4.55, 4.9, 5.0, 5.5) for at in (29, 129)]
        for scores in (torch.randn(count, generator=g), torch.randn(count, generator=g) * 4, torch.linspace(0, 5, count), *late):
            m, q, page, row = with_scores(kind, scores, tokens, dim)
            v = torch.randn(dim, generator=g).to(kind).cuda()
            m.cache.values[:] = v
            for longest in (None, 0):
                got = gen.attend_cache(q, m.cache, m.batch, scale=1.0, longest=longest)
                assert torch.equal(got, v.expand_as(got)), (count, longest)


@pytest.mark.parametrize("kind", CACHED)
@pytest.mark.parametrize("scale", [1e-10, 1e-30, 1e-45])
@pytest.mark.parametrize("tokens", [3, 100])
def test_scores_that_are_all_nothing(kind, scale, tokens):
    """Queries and scales so small that all scores are nothing: each key counts alike, and none that is hidden."""
    for size in (0.0, 1e-30, 1.0):
        for count in (140, 3000):
            m = Made(kind, [count - tokens], [tokens], 1, 64, 64)
            q = torch.full((tokens, 1, 64), size, dtype=torch.float16 if kind == torch.float16 else torch.bfloat16, device="cuda")
            v, seen = m.held(0, "values", count)[:, 0], torch.arange(count - tokens + 1, count + 1)[:, None]
            want, size_ = v.cumsum(0)[count - tokens:] / seen, v.abs().cumsum(0)[count - tokens:] / seen
            # Weights all alike are right, but times scales over integers, where they are fp16 and 32-bit sums of values up to 256; sums; the result.
            off = 2.0 ** -20 * size_ + (2.0 ** -11 * size_ + (count / 16 + 8) * 2.0 ** -24 * 256 * 0.03 if kind == torch.int8 else 0) + (2.0 ** -25 if kind == torch.float16 else 0)
            got = gen.attend_cache(q, m.cache, m.batch, scale=scale)
            assert ((got[:, 0].cpu().double() - want).abs() <= off + ROUND[got.dtype] * (want.abs() + off)).all(), (size, count)


# ---- drafts -------------------------------------------------------------------------------------------------------
ALMOST_ONE = 1.0 - 2.0 ** -53


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("v", [50, 33000])
@pytest.mark.parametrize("mask", [-math.inf, -1e9, None])
def test_drafts_of_masked_tokens(dtype, v, mask):
    """Tokens that the target, the draft model or both mask, with -inf or far down, behind refusals of others or of none: a sequence for each."""
    g = seeded(v, 41)
    mask = torch.finfo(dtype).min if mask is None else mask
    first = [(torch.randn(v, generator=g) * 3) for _ in range(2)]
    likelier = (first[0] - first[1]).argsort().tolist()                # by the draft model, and so refused by numbers close to one
    masked = likelier[v // 2]
    logits, draft, tokens, parents, u = [], [], [], [], []
    for where in ("target", "draft", "both"):
        for refused in (0, 1, 2):
            for number in (0.0, 0.3, ALMOST_ONE):
                for root in (0.0, 0.6):
                    x, y = (torch.randn(5, v, generator=g) * 3 for _ in range(2))
                    x[0], y[0] = first
                    if where != "draft":
                        x[0, masked] = mask
                    if where != "target":
                        y[0, masked] = mask
                    logits.append(x.to(dtype)), draft.append(y.to(dtype))
                    tokens += [0] + likelier[:refused] + [masked] + [likelier[-1]] * (3 - refused)
                    parents += [-1] + [0] * 4
                    u += [root] + [ALMOST_ONE] * refused + [number] + [0.5] * (3 - refused)
    starts = list(range(0, len(tokens) + 1, 5))
    for given in (torch.cat(draft), None):
        check_drafts(torch.cat(logits), tokens, starts, parents, torch.tensor(u, dtype=torch.float64), given, 2)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("v", [40, 9000, 40001])
@pytest.mark.parametrize("mask", [-math.inf, -1e9, None])
def test_first_tokens_that_have_a_probability(dtype, v, mask):
    """The token of a root's number zero is the first that has a probability, and where nothing is left behind refusals, too."""
    mask = torch.finfo(dtype).min if mask is None else mask
    x = torch.randn(3, v, generator=seeded(v, 42))
    x[:, :v // 2] = mask
    x[:, v - 3:] = mask
    x = x.to(dtype)
    for root in (0.0, 0.5, ALMOST_ONE):
        u = torch.tensor([root, ALMOST_ONE, ALMOST_ONE], dtype=torch.float64)
        check_drafts(x, [0, 1, 2], [0, 3], [-1, 0, 0], u, None, 2)
        args = x.cuda(), torch.tensor([0, 1, 2]).cuda(), torch.tensor([0, 3], dtype=torch.int32).cuda(), torch.tensor([-1, 0, 0], dtype=torch.int32).cuda(), u.cuda(), 2
        # p - p is nothing: of p itself, which refused tokens without a probability change as little without a draft model
        assert all(torch.equal(a, b) for a, b in zip(gen.verify_drafts(*args, draft_logits=args[0]), gen.verify_drafts(*args)))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("v", [7, 40000])
def test_logits_far_from_nothing(dtype, v):
    """Rows all of whose entries are the type's lowest, or as large, or near to each other and far from nothing."""
    g = seeded(v, 43)
    lowest = torch.finfo(dtype).min
    for far in (lowest, lowest / 2, -lowest, 3e4, 1e6, -1e12, 1e20):
        if abs(far) > -lowest:
            continue
        for near in (0, 3):                    # equal, or neighbouring numbers of the type
            x = (far * (1 - torch.randint(0, max(near, 1), (4, v), generator=g) * torch.finfo(dtype).eps).double()).to(dtype)
            y = torch.randn(4, v, generator=g).to(dtype)
            for t in (1.0, 0.7, 1e-3, 1e3):
                tokens, u = [0] + torch.randint(0, v, (3,), generator=g).tolist(), torch.rand(4, generator=g, dtype=torch.float64)
                for given in (None, y):
                    check_drafts(x, tokens, [0, 4], [-1, 0, 0, 1], u, given, 2, t)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("v,allowed", [(3, 2), (60, 3), (60, 5), (33000, 2), (33000, 3)])
def test_few_tokens_left(dtype, v, allowed):
    """Without a draft model, refusals that leave little, one token or nothing: what is left is summed, not taken for what the refused ones lack to one."""
    g = seeded(v, allowed, 44)
    logits, tokens, u, parents = [], [], [], []
    for seed in range(10):
        for numbers in ([ALMOST_ONE] * (allowed - 1) + [0.5], [ALMOST_ONE] * allowed, [ALMOST_ONE] * (allowed - 1) + [0.999]):
            x = torch.full((allowed + 3, v), -math.inf)
            few = torch.randperm(v, generator=g)[:allowed]
            # near each other, or one after the other 5 to 40 nats apart
            x[0, few] = torch.randn(allowed, generator=g) if seed < 5 else -(torch.rand(allowed, generator=g) * 35 + 5).cumsum(0) / (1 if allowed < 5 else 3)
            x[1:, 0] = 0
            few = few.tolist()
            logits.append(x.to(dtype))
            tokens += [0] + few[:-1] + [few[0], few[-1], few[-1]]      # the same token twice; in the end the one that is left, and again
            u += [0.4] + numbers[:-1] + [0.7, numbers[-1], 0.0]
            parents += [-1] + [0] * (allowed + 2)
    check_drafts(torch.cat(logits), tokens, list(range(0, len(tokens) + 1, allowed + 3)), parents, torch.tensor(u, dtype=torch.float64), None, 2)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("v", [300, 20000])
def test_numbers_next_to_the_border(dtype, v):
    """Drafts whose number is 3 10^-14 of it above or below p / q.  Entries are at most 32 below their row's largest: differences of them, times log2(e), are 32 2^-53 off, their
    exponentials 4 10^-16, sums and quotients 10 2^-53 - of p and q together 10^-14."""
    g = seeded(v, 46)
    n = 300
    logits, draft = ((torch.randn(2 * n, v, generator=g) * 3).clamp(-16, 16).to(dtype) for _ in range(2))
    p, q = (torch.softmax(x[::2].double(), dim=1) for x in (logits, draft))
    x = (q / p).topk(20, dim=1).indices.gather(1, torch.randint(0, 20, (n, 1), generator=g))
    share = (p.gather(1, x) / q.gather(1, x))[:, 0]
    above = torch.arange(n) % 2
    u = torch.stack((torch.full((n,), 0.5, dtype=torch.float64), share * (1 + (2 * above - 1).double() * 3e-14)), dim=1)
    assert (u < 1).all()
    tokens = torch.stack((torch.zeros_like(x[:, 0]), x[:, 0]), dim=1)
    counts, _, _ = gen.verify_drafts(logits.cuda(), tokens.flatten().cuda(), (torch.arange(n + 1) * 2).int().cuda(), None, u.flatten().cuda(), 1, draft_logits=draft.cuda())
    assert torch.equal(counts.cpu(), 1 - above)
