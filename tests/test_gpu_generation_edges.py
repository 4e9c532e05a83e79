"""Attention over the cache and drafts at the ends of numbers' ranges, against 64 bits."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from test_gpu_generation import ROUND, Made  # noqa: E402
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
    return torch.softmax(torch.where(seen, scores.double(), float("-inf")), dim=1), m.held(0, "values", count)[:, 0]


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
