"""The operators of a forward pass in 8-bit integers, over the sizes a prover runs it at.

What a proof is about is a pass that has been run: rows of activations are rounded to 8-bit integers with a scale a token
(`quantize`), multiplied with weights that have a scale a channel (`matmul`; its exact sums are the words that are proved),
taken through the gated feed-forward block (`gated`), and at the end the logits say how likely the tokens of the answer
were (`logprobs`).  4096, 11008 and 1000 are the sizes of the layer workload of the benchmark.
"""
import math

import torch

own = False             # whether run() makes the framework's calls, or computes the plain form

P = (1 << 64) - (1 << 32) + 1
CHUNK = 1024            # products of this many 8-bit pairs sum to 2^24 at most: exact in 32-bit floats in any order
MOST_OPS = 2 * 4096 * 4096 * 11008      # of a drawn product, as of the largest listed
MOST_ELEMENTS = 32000 * 4096            # of a drawn matrix of rows or logits, as of the largest listed

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "int32": torch.int32, "field": torch.uint64}


def listed():
    return [
        # one token's activations in front of a projection: a call that is all latency
        {"name": "quantize_token", "kind": "quantize", "m": 1, "k": 4096, "pad": 0, "type": "bf16"},
        # the activations of 1000 tokens in front of the feed-forward block's last projection
        {"name": "quantize_layer", "kind": "quantize", "m": 1000, "k": 11008, "pad": 0, "type": "bf16"},
        # a vocabulary's projection, a scale for each channel, done once when the weights are loaded
        {"name": "quantize_weights", "kind": "quantize", "m": 32000, "k": 4096, "pad": 0, "type": "f32"},
        # one token through the widest projection: the weights are read and hardly used
        {"name": "matmul_token", "kind": "matmul", "m": 1, "k": 4096, "n": 11008, "pad": 0, "bias": False, "type": "bf16"},
        # the words of a square projection of 1000 tokens, as field elements for the proof
        {"name": "matmul_words", "kind": "matmul", "m": 1000, "k": 4096, "n": 4096, "pad": 0, "bias": False, "type": "field"},
        # sizes that divide by nothing, rows apart from each other, a bias
        {"name": "matmul_ragged", "kind": "matmul", "m": 333, "k": 1411, "n": 5003, "pad": 13, "bias": True, "type": "f16"},
        # a long prompt's tokens through the widest projection
        {"name": "matmul_long", "kind": "matmul", "m": 4096, "k": 4096, "n": 11008, "pad": 0, "bias": False, "type": "bf16"},
        # the feed-forward block for a handful of sequences, a token each
        {"name": "gated_tokens", "kind": "gated", "m": 7, "k": 4096, "n": 11008, "pad": 0, "act": "silu", "type": "bf16"},
        # the same for the benchmark's 1000 tokens
        {"name": "gated_layer", "kind": "gated", "m": 1000, "k": 4096, "n": 11008, "pad": 0, "act": "silu", "type": "bf16"},
        # one answered token with the alternatives that an interface shows
        {"name": "logprobs_token", "kind": "logprobs", "m": 1, "v": 32000, "pad": 0, "top": 20, "temperature": 1.0, "masked": 0.0, "type": "f32"},
        # the answer of 1000 tokens
        {"name": "logprobs_answer", "kind": "logprobs", "m": 1000, "v": 32000, "pad": 0, "top": 5, "temperature": 1.0, "masked": 0.0, "type": "bf16"},
        # an odd vocabulary most of which a grammar forbids, sampled below temperature one
        {"name": "logprobs_grammar", "kind": "logprobs", "m": 37, "v": 50257, "pad": 7, "top": 8, "temperature": 0.7, "masked": 0.99, "type": "f16"},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi, multiple):
    """The same, every other one a multiple of `multiple`, as the widths of models are."""
    n = _log(rng, lo, hi)
    n = max(multiple, n // multiple * multiple) if rng.random() < 0.5 else n
    return n if n != 3072 else n + multiple


def draw(rng):
    kind = rng.choice(["quantize", "matmul", "gated", "logprobs"])
    pad = rng.choice([0, 0, 0, 5, 16])
    if kind == "quantize":
        k = _size(rng, 64, 16384, 128)
        return {"kind": kind, "m": _log(rng, 1, min(32000, MOST_ELEMENTS // k)), "k": k, "pad": pad, "type": rng.choice(["f32", "bf16", "f16"])}
    if kind == "logprobs":
        v = _size(rng, 1000, 160000, 64)
        return {"kind": kind, "m": _log(rng, 1, min(4096, MOST_ELEMENTS // v)), "v": v, "pad": pad, "top": rng.choice([0, 1, 2, 5, 8, 20, 33, 64]),
                "temperature": rng.choice([1.0, 1.0, 0.7, 1.3]), "masked": rng.choice([0.0, 0.0, 0.5, 0.99]), "type": rng.choice(["f32", "bf16", "f16"])}
    k, n = _size(rng, 64, 16384, 128), _size(rng, 64, 16384, 128)
    m = _log(rng, 1, max(1, min(4096, MOST_OPS // (4 * k * n))))
    case = {"kind": kind, "m": m, "k": k, "n": n, "pad": pad}
    if kind == "gated":
        return {**case, "act": rng.choice(["silu", "silu", "gelu"]), "type": rng.choice(["f32", "bf16", "f16"])}
    return {**case, "bias": rng.random() < 0.3, "type": rng.choice(["f32", "bf16", "f16", "int32", "field"])}


# ---- inputs -------------------------------------------------------------------------------------------------------
def _normal(gen, rows, width, pad, dtype):
    """Rows of a normal distribution, `pad` columns of other data behind each."""
    return torch.randn((rows, width + pad), generator=gen, device="cuda").to(dtype)[:, :width]


def _eighths(gen, rows, width, pad, outliers):
    """8-bit rows as rounding a normal distribution gives them, with their scales; `outliers`: a few channels ten times the
    rest, as activations have them."""
    x = torch.randn((rows, width + pad), generator=gen, device="cuda")
    if outliers:
        x = x * torch.where(torch.rand((width + pad,), generator=gen, device="cuda") < 0.003, 10.0, 1.0)
    most = x.abs().amax(dim=1, keepdim=True)
    q = torch.round(x * (127.0 / most)).to(torch.int8)
    return q[:, :width], (most[:, 0] / 127.0).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, m, pad = case["kind"], case["m"], case["pad"]
    state = {"case": case}
    if kind == "quantize":
        state["x"] = _normal(gen, m, case["k"], pad, TYPES[case["type"]])
    elif kind == "logprobs":
        x = torch.randn((m, case["v"] + pad), generator=gen, device="cuda") * 3.0
        if case["masked"]:
            x = x.masked_fill(torch.rand(x.shape, generator=gen, device="cuda") < case["masked"], -math.inf)
        state["logits"] = x.to(TYPES[case["type"]])[:, :case["v"]]
        # mostly tokens that the model finds likely
        noise = torch.rand((m, case["v"]), generator=gen, device="cuda").log_().neg_().log_().neg_()
        state["tokens"] = torch.argmax(state["logits"].float() + noise, dim=1)
    else:
        state["a"], state["a_scale"] = _eighths(gen, m, case["k"], pad, True)
        state["b"], state["b_scale"] = _eighths(gen, case["n"], case["k"], pad, False)
        state["b_scale"] *= 0.02
        if kind == "gated":
            state["u"], state["u_scale"] = _eighths(gen, case["n"], case["k"], pad, False)
            state["u_scale"] *= 0.02
        elif case["bias"]:
            state["bias"] = torch.randn((case["n"],), generator=gen, device="cuda")
    return state


# ---- one pass -----------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    return _framework(case, state) if own else _plain(case, state)


def _framework(case, state):
    from verinf_amd.prover import inference
    kind = case["kind"]
    if kind == "quantize":
        q, scale = inference.quantize_rows(state["x"])
        return {"values": q * scale[:, None], "scale": scale}
    if kind == "matmul":
        dtype = TYPES[case["type"]]
        if not dtype.is_floating_point:
            out = inference.int8_matmul(state["a"], state["b"], dtype=dtype)
            return {"out": out if dtype == torch.int32 else out.view(torch.int64)}
        return {"out": inference.int8_matmul(state["a"], state["b"], state["a_scale"], state["b_scale"], bias=state.get("bias"), dtype=dtype)}
    if kind == "gated":
        return {"out": inference.int8_gated(state["a"], state["b"], state["u"], state["a_scale"], state["b_scale"], state["u_scale"],
                                            activation=case["act"], dtype=TYPES[case["type"]])}
    logprob, entropy, top_logprobs, top_tokens = inference.token_logprobs(state["logits"], state["tokens"], top=case["top"],
                                                                          temperature=case["temperature"])
    return {"logprob": logprob, "entropy": entropy, "top_logprobs": top_logprobs, "top_tokens": top_tokens}


def _plain(case, state):
    kind = case["kind"]
    if kind == "quantize":
        x = state["x"].float()
        most = x.abs().amax(dim=1)
        scale = most / 127.0
        steps = torch.div(torch.full_like(most, 127.0), most)
        return {"values": torch.round(x * steps[:, None]) * scale[:, None], "scale": scale}
    if kind == "matmul":
        dtype = TYPES[case["type"]]
        if not dtype.is_floating_point:
            s = _exact_sums(state["a"], state["b"])
            if dtype == torch.int32:
                return {"out": s.to(torch.int32)}
            return {"out": torch.where(s < 0, s - ((1 << 32) - 1), s)}         # p - |s| as a signed 64-bit word
        s = _scaled(state, "b")
        if "bias" in state:
            s = s + state["bias"]
        return {"out": s.to(dtype)}
    if kind == "gated":
        g, u = _scaled(state, "b"), _scaled(state, "u")
        if case["act"] == "silu":
            g = g / (1.0 + torch.exp(-g))
        else:
            g = g * 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return {"out": (g * u).to(TYPES[case["type"]])}
    x = state["logits"].float()
    forbidden = x == -math.inf
    d = torch.where(forbidden, -math.inf, (x - x.amax(dim=1, keepdim=True)) * (1.0 / case["temperature"]))
    e = torch.exp(d)
    z = e.sum(dim=1)
    log_z = torch.log(z)
    entropy = torch.where(z == 0, 0.0, log_z - torch.where(e > 0, e * d, 0.0).sum(dim=1) / z)
    lp = torch.where(forbidden, -math.inf, d - log_z[:, None])
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["top"]]
    return {"logprob": lp.gather(1, state["tokens"][:, None])[:, 0], "entropy": entropy, "top_logprobs": lp.gather(1, order), "top_tokens": order}


def _scaled(state, name):
    return (state["a"].float() @ state[name].float().T) * state["a_scale"][:, None] * state[name + "_scale"]


def _exact_sums(a, b):
    """a b^T as 64-bit integers: products of CHUNK inner indices at a time are whole numbers up to 2^24."""
    k = a.shape[1]
    a, b = (torch.nn.functional.pad(t.float(), (0, -k % CHUNK)).view(t.shape[0], -1, CHUNK).transpose(0, 1).contiguous() for t in (a, b))
    return torch.bmm(a, b.transpose(1, 2).contiguous()).to(torch.int64).sum(dim=0)


# ---- what it costs, what is right ---------------------------------------------------------------------------------
def work(case):
    kind, m = case["kind"], case["m"]
    size = {"f32": 4, "int32": 4, "field": 8}.get(case["type"], 2)
    if kind == "quantize":
        return {"bytes": m * case["k"] * (size + 1) + 4 * m, "flops": 3 * m * case["k"]}
    if kind == "logprobs":
        return {"bytes": m * case["v"] * size + 16 * m + 12 * m * case["top"], "flops": 6 * m * case["v"]}
    k, n = case["k"], case["n"]
    weights = 2 if kind == "gated" else 1
    return {"bytes": (m + weights * n) * k + m * n * size + 4 * (m + weights * n), "flops": 2 * weights * m * k * n}


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        x = state["x"].double()
        top = x.abs().max(dim=1).values
        steps = (127.0 / top).float().double()          # held in 32 bits by the definition
        return {"values": (x * steps[:, None]).round() * (top / 127.0)[:, None], "scale": top / 127.0}
    if kind == "logprobs":
        z = state["logits"].double() / case["temperature"]
        lp = torch.where(torch.isneginf(z), z, z - torch.logsumexp(z, dim=1, keepdim=True))
        p = lp.exp()
        # equal logits in the order of their indexes
        order = torch.argsort(z, dim=1, descending=True, stable=True)[:, :case["top"]]
        return {"logprob": lp[torch.arange(case["m"], device="cuda"), state["tokens"]], "entropy": torch.special.entr(p).sum(dim=1),
                "top_logprobs": torch.take_along_dim(lp, order, dim=1), "top_tokens": order}
    s = state["a"].double() @ state["b"].double().T      # whole numbers below 2^53
    if kind == "matmul":
        if case["type"] == "int32":
            return {"out": s.to(torch.int32)}
        if case["type"] == "field":
            s = s.to(torch.int64)
            return {"out": s + torch.where(s < 0, P - (1 << 64), 0)}
        s = s * torch.outer(state["a_scale"].double(), state["b_scale"].double())
        return {"out": s + state["bias"].double() if case["bias"] else s}
    g = s * torch.outer(state["a_scale"].double(), state["b_scale"].double())
    u = state["a"].double() @ state["u"].double().T * torch.outer(state["a_scale"].double(), state["u_scale"].double())
    act = g * torch.sigmoid(g) if case["act"] == "silu" else g * torch.special.ndtr(g)
    return {"out": act * u}
