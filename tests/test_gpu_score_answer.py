"""The example that takes an answer's hidden states to its log probabilities, against the same in 64 bits."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

SPEC = importlib.util.spec_from_file_location("score_answer", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "score_answer.py"))


@pytest.fixture(scope="module")
def ex():
    module = importlib.util.module_from_spec(SPEC)
    SPEC.loader.exec_module(module)
    return module


def dequantized(pair):
    q, s = pair
    return q.double() * s.double()[:, None]


def rounded(x):
    """rows to 8 bits and back, by the definition's 32-bit operations"""
    x = x.float()
    top = x.abs().amax(dim=1, keepdim=True)
    return torch.round(x * (torch.full_like(top, 127.0) / top)).double() * (top.double() / 127)


@pytest.mark.parametrize("tokens,hidden,ffn,vocab", [(1, 64, 160, 500), (37, 128, 343, 1009), (150, 256, 700, 3001)])
def test_an_answer_is_scored(ex, tokens, hidden, ffn, vocab):
    weights = ex.make_weights(hidden, ffn, vocab, 3)
    x = torch.randn((tokens, hidden), generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").to(torch.bfloat16)
    logits = ex.forward(x, weights)
    # the same steps in 64 bits, rounded to 8 bits and to bfloat16 where the pass is
    xq = rounded(x)
    g, u = xq @ dequantized(weights["gate"]).T, xq @ dequantized(weights["up"]).T
    h = rounded((g * torch.sigmoid(g) * u).to(torch.bfloat16))
    y = x + (h @ dequantized(weights["down"]).T).to(torch.bfloat16)
    want = rounded(y) @ dequantized(weights["head"]).T
    # where the products' 32-bit roundings fall on the other side of a rounding to bfloat16 (2^-8 of an entry) or to 8 bits (a
    # step of 1/127 of the row's largest), single entries of a row differ by that: of sums of `hidden` terms of size one a part in 127
    assert (logits.double() - want).norm() <= 0.01 * want.norm()
    t = want.argmax(dim=1)
    t[::2] = torch.arange(tokens, device="cuda")[::2] % vocab
    s = ex.score(logits, t, 4)
    lp = torch.log_softmax(logits.double(), dim=1)
    assert torch.allclose(s["bits"].double(), -lp[torch.arange(tokens), t] / 0.6931471805599453, rtol=1e-5, atol=1e-5)
    assert torch.allclose(s["entropy"].double(), -(lp.exp() * lp).sum(dim=1), rtol=1e-5, atol=1e-4)
    assert torch.equal(s["top_tokens"], torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :4])
    assert abs(s["agreed"] - float((logits.argmax(dim=1) == t).double().mean())) < 1e-9
    assert abs(s["total_bits"] - float(s["bits"].double().sum())) < 1e-6


def test_its_words_are_the_field_product(ex):
    from verinf_amd.prover import cuda_primitives as cp
    from verinf_amd.prover import inference as inf
    q, _ = inf.quantize_rows(torch.randn((50, 300), generator=torch.Generator(device="cuda").manual_seed(5), device="cuda"))
    w = ex.make_weights(300, 128, 64, 6)["gate"][0]
    assert torch.equal(ex.words(q, w).view(torch.int64), cp.gl_matmul(ex.lift(q), ex.lift(w.T)).view(torch.int64))
