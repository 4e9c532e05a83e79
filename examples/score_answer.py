"""How likely was the answer?  The end of a forward pass in 8-bit integers, and the exact sums of a projection in the field.

    python examples/score_answer.py [--tokens 1000] [--hidden 4096] [--ffn 11008] [--vocab 32000] [--top 5]

Random weights and activations of a layer's sizes go through a gated feed-forward block and the projection to the vocabulary, all
products in 8-bit integers with a scale for each token and channel (`verinf_amd.prover.inference`); the logits then say how likely given
tokens were, how uncertain the model was, and what it would rather have said.  The sums of the block's first projection are also taken as
field elements and compared with the field product of the lifted operands; nothing is committed to or proved here.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from verinf_amd.prover import cuda_primitives as cp  # noqa: E402
from verinf_amd.prover import inference as inf  # noqa: E402

P = cp.P


def make_weights(hidden, ffn, vocab, seed, device="cuda"):
    """8-bit weights, (channels, inputs) with a scale a channel: gate, up, down and the vocabulary's."""
    gen = torch.Generator(device=device).manual_seed(seed)
    shapes = {"gate": (ffn, hidden), "up": (ffn, hidden), "down": (hidden, ffn), "head": (vocab, hidden)}
    return {name: inf.quantize_rows(torch.randn(s, generator=gen, device=device) / s[1] ** 0.5) for name, s in shapes.items()}


def forward(x, weights):
    """Logits (tokens, vocab) float32 of hidden states x (tokens, hidden) behind a gated feed-forward block and the vocabulary's projection."""
    q, scale = inf.quantize_rows(x)
    (gate, gate_scale), (up, up_scale) = weights["gate"], weights["up"]
    h, h_scale = inf.quantize_rows(inf.int8_gated(q, gate, up, scale, gate_scale, up_scale))
    x = x + inf.int8_matmul(h, weights["down"][0], h_scale, weights["down"][1], dtype=x.dtype)
    q, scale = inf.quantize_rows(x)
    return inf.int8_matmul(q, weights["head"][0], scale, weights["head"][1], dtype=torch.float32)


def score(logits, tokens, top):
    """What the answer says of itself: bits that the model leaves unexplained, by token and in all, its uncertainty, and how often it would
    have said the same."""
    logprob, entropy, top_logprobs, top_tokens = inf.token_logprobs(logits, tokens, top=top)
    bits = -logprob / 0.6931471805599453
    return {"bits": bits, "entropy": entropy, "top_logprobs": top_logprobs, "top_tokens": top_tokens, "total_bits": float(bits.double().sum()),
            "agreed": float((top_tokens[:, 0] == tokens).double().mean()) if top else None}


def words(q, w):
    """The sums of a projection as field elements."""
    return inf.int8_matmul(q, w, dtype=torch.uint64)


def lift(t):
    """8-bit integers as field elements."""
    v = t.to(torch.int64)
    return torch.where(v < 0, v + (P - (1 << 64)), v).contiguous().view(torch.uint64)


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("tokens", 1000), ("hidden", 4096), ("ffn", 11008), ("vocab", 32000), ("top", 5), ("seed", 0)):
        ap.add_argument("--" + name, type=int, default=value)
    a = ap.parse_args()
    weights = make_weights(a.hidden, a.ffn, a.vocab, a.seed)
    gen = torch.Generator(device="cuda").manual_seed(a.seed + 1)
    x = torch.randn((a.tokens, a.hidden), generator=gen, device="cuda").to(torch.bfloat16)
    logits = forward(x, weights)
    # an answer sampled from the model itself
    tokens = torch.multinomial(torch.softmax(logits, dim=1), 1, generator=gen)[:, 0]
    score(logits, tokens, a.top)                 # every kernel has been loaded before the time is taken
    torch.cuda.synchronize()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    logits = forward(x, weights)
    s = score(logits, tokens, a.top)
    end.record()
    torch.cuda.synchronize()
    print(f"{a.tokens} tokens: {s['total_bits'] / a.tokens:.3f} bits a token unexplained, entropy {float(s['entropy'].mean()) / 0.6931471805599453:.3f} bits, "
          f"{100 * s['agreed']:.1f} % were the likeliest token, {start.elapsed_time(end):.3f} ms")
    some = min(a.tokens, 64)
    q, _ = inf.quantize_rows(x[:some])
    w = weights["gate"][0][:256]
    same = torch.equal(words(q, w).view(torch.int64), cp.gl_matmul(lift(q), lift(w.T)).view(torch.int64))
    print(f"sums of the first projection as field elements {'equal' if same else 'DIFFER FROM'} the field product of the lifted operands")
    return 0 if same else 1


if __name__ == "__main__":
    sys.exit(main())
