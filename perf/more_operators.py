"""The operators that answer with a cache and drafted tokens, over the sizes of serving.

A model's queries and keys are turned by their positions (`rotate`), keys and values go into a paged cache (`append`), the new
tokens - one a sequence, a prompt's, or a tree of drafts - attend over it (`attend`), the drafts are held against the target's
probabilities (`verify`), and the accepted ones' entries move to the front of the cache (`keep`).  32 heads of 128, 32000 tokens
and 4096 positions are the sizes of the benchmark's layer workload; 8 heads of keys shared by 32 are common beside them.
"""
import math

import torch

own = False             # whether run() makes the framework's calls, or computes the plain form

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "int8": torch.int8}
MOST_ELEMENTS = 4096 * 32 * 128                 # of a drawn matrix of heads, as of the largest listed
MOST_CACHED = 64 * 4600 * 8 * 128               # of a drawn cache's keys, as of the largest listed
MOST_PAIRS = 32 * 4096 * 4096 // 2              # of query heads and keys, the same
MOST_LOGITS = 1024 * 32000


def listed():
    return [
        # one token's queries: a call that is all latency
        {"name": "rotate_token", "kind": "rotate", "n": 1, "heads": 32, "dim": 128, "rotated": 128, "interleaved": False, "far": 4096, "scaling": "none", "pad": 0, "type": "bf16"},
        # a long prompt's, half of each head turned, frequencies scaled for a context far longer than the model was trained on
        {"name": "rotate_prompt", "kind": "rotate", "n": 4096, "heads": 32, "dim": 128, "rotated": 64, "interleaved": True, "far": 1000000, "scaling": "parts", "pad": 0, "type": "f16"},
        # a token for each of 64 sequences into the cache
        {"name": "append_tokens", "kind": "append", "batch": 64, "tokens": 1, "context": 4000, "heads": 8, "dim": 128, "page": 16, "rotated": 128, "interleaved": False, "cache": "bf16", "type": "bf16"},
        # a long prompt into an empty cache of 8-bit integers
        {"name": "append_prompt", "kind": "append", "batch": 1, "tokens": 4096, "context": 0, "heads": 8, "dim": 128, "page": 64, "rotated": 128, "interleaved": False, "cache": "int8", "type": "bf16"},
        # the next token of one conversation
        {"name": "attend_token", "kind": "attend", "batch": 1, "tokens": 1, "context": 1000, "ragged": False, "tree": False, "heads": 8, "group": 4, "dim": 128, "page": 16, "cache": "bf16", "type": "bf16"},
        # the next token of 64, which are of all lengths
        {"name": "attend_batch", "kind": "attend", "batch": 64, "tokens": 1, "context": 8192, "ragged": True, "tree": False, "heads": 8, "group": 4, "dim": 128, "page": 64, "cache": "bf16", "type": "bf16"},
        # trees of 24 drafts over caches of 8-bit integers
        {"name": "attend_trees", "kind": "attend", "batch": 16, "tokens": 25, "context": 4100, "ragged": False, "tree": True, "heads": 8, "group": 4, "dim": 128, "page": 64, "cache": "int8", "type": "bf16"},
        # a long prompt, every head with keys of its own
        {"name": "attend_prompt", "kind": "attend", "batch": 1, "tokens": 4096, "context": 0, "ragged": False, "tree": False, "heads": 32, "group": 1, "dim": 128, "page": 64, "cache": "f16", "type": "f16"},
        # four drafted tokens of one conversation, drafted without probabilities
        {"name": "verify_chain", "kind": "verify", "batch": 1, "nodes": 5, "v": 32000, "tree": False, "drafted": False, "depth": 4, "temperature": 1.0, "type": "f32"},
        # trees of 15 drafts for 64 sequences, each drawn from the draft model's probabilities
        {"name": "verify_trees", "kind": "verify", "batch": 64, "nodes": 16, "v": 32000, "tree": True, "drafted": True, "depth": 6, "temperature": 1.0, "type": "bf16"},
        # one conversation's accepted drafts in one layer's cache
        {"name": "keep_one", "kind": "keep", "batch": 1, "nodes": 25, "context": 1000, "depth": 5, "heads": 8, "dim": 128, "page": 16, "cache": "bf16"},
        # 64 sequences' in the caches of 32 layers, which lie together page by page
        {"name": "keep_layers", "kind": "keep", "batch": 64, "nodes": 32, "context": 400, "depth": 8, "heads": 256, "dim": 128, "page": 16, "cache": "int8"},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotate", "append", "attend", "attend", "verify", "keep"])
    dim = rng.choice([64, 128, 128, 128, 256, 80, 96, 112])
    page = rng.choice([16, 32, 64, 128])
    if kind == "rotate":
        heads = rng.choice([1, 5, 8, 12, 32, 40])
        kept = rng.choice(["f32", "bf16", "f16"])
        return {"kind": kind, "n": _log(rng, 1, MOST_ELEMENTS // (heads * dim * (2 if kept == "f32" else 1))), "heads": heads, "dim": dim, "rotated": rng.choice([dim, dim, dim // 2, 16 * rng.randint(1, dim // 16)]),
                "interleaved": rng.random() < 0.5, "far": _log(rng, 4096, 1000000), "scaling": rng.choice(["none", "linear", "base", "parts"]), "pad": rng.choice([0, 0, 8, 24]),
                "type": kept}
    heads = rng.choice([1, 2, 4, 8, 8, 16, 32])
    if kind == "append":
        tokens = rng.choice([1, 1, _log(rng, 2, min(4096, MOST_ELEMENTS // (10 * heads * dim)))])
        batch = _log(rng, 1, max(1, min(256, MOST_ELEMENTS // (10 * tokens * heads * dim))))
        cache = rng.choice(["bf16", "f16", "int8"])
        return {"kind": kind, "batch": batch, "tokens": tokens, "context": rng.choice([0, _log(rng, 1, 200)]), "heads": heads, "dim": dim, "page": page,
                "rotated": rng.choice([0, dim, dim, dim // 2]), "interleaved": rng.random() < 0.5, "cache": cache, "type": rng.choice(["f32", "bf16", "f16"])}
    if kind == "attend":
        cache = rng.choice(["bf16", "f16", "int8"])
        group, tree = rng.choice([1, 2, 4, 4, 7, 8]), False
        tokens = rng.choice([1, 1, 1, rng.randint(2, 64), rng.randint(2, 64), _log(rng, 65, 4096)])
        if 2 <= tokens <= 64:
            tree = rng.random() < 0.7
        batch = _log(rng, 1, 64) if tokens <= 64 else rng.randint(1, 3)
        pairs = MOST_PAIRS * 100 // dim
        tokens = min(tokens, int((pairs / (batch * heads * group)) ** 0.5))
        most = max(tokens, min(32768, MOST_CACHED * 3 // 4 // (batch * heads * dim), pairs // (batch * tokens * heads * group)))
        context = _log(rng, 1, max(1, most - tokens)) if tokens <= 64 else rng.choice([0, _log(rng, 1, max(1, most - tokens))])
        return {"kind": kind, "batch": batch, "tokens": tokens, "context": context, "ragged": rng.random() < 0.5, "tree": tree, "heads": heads, "group": group, "dim": dim,
                "page": page, "cache": cache, "type": "bf16" if cache == "int8" else cache}
    if kind == "verify":
        v = _log(rng, 1000, 160000)
        v = v // 64 * 64 if rng.random() < 0.5 else v
        nodes = rng.choice([1, 2, 5, 8, rng.randint(9, 64)])
        drafted = rng.random() < 0.5
        return {"kind": kind, "batch": _log(rng, 1, max(1, min(128, MOST_LOGITS // (nodes * v * (2 if drafted else 1))))), "nodes": nodes, "v": v, "tree": rng.random() < 0.5,
                "drafted": drafted, "depth": rng.randint(1, 10), "temperature": rng.choice([1.0, 1.0, 0.7, 1.3]), "type": rng.choice(["f32", "bf16", "f16"])}
    depth = rng.randint(1, 8)
    heads = heads * rng.choice([1, 1, 8, 32])
    return {"kind": kind, "batch": _log(rng, 1, max(1, min(64, MOST_ELEMENTS * 8 // (heads * dim * 600)))), "nodes": 2 * depth + rng.randint(2, 40), "context": _log(rng, 1, 400), "depth": depth,
            "heads": heads, "dim": dim, "page": page, "cache": rng.choice(["bf16", "f16", "int8"])}


# ---- inputs -------------------------------------------------------------------------------------------------------
def _frequencies(case):
    """Radians a position, of each pair of the `rotated` first columns, and what the turned columns are multiplied by; in 64 bits."""
    half = case["rotated"] // 2
    base, scaling = 10000.0, case.get("scaling", "none")
    if scaling == "base":
        base *= 16.0 ** (2 * half / (2 * half - 2)) if half > 1 else 1.0
    f = [base ** (-i / half) for i in range(half)]
    if scaling == "linear":
        f = [x / 16.0 for x in f]
    if scaling == "parts":          # fast ones as they are, slow ones divided by 16, by how often they turn in 4096 positions
        keep = [min(1.0, max(0.0, (4096 * x / (2 * math.pi) - 1.0) / 31.0)) for x in f]
        f = [x * k + x / 16.0 * (1.0 - k) for x, k in zip(f, keep)]
    return f, 0.1 * math.log(16.0) + 1.0 if scaling == "parts" else 1.0


SCALINGS = {"none": None, "linear": ("linear", 16.0), "base": ("base", 16.0), "parts": ("parts", 16.0, 4096)}


def _plan(state, case):
    """The frequencies in hand; the framework's plan of them where its calls are made."""
    f, state["amplitude"] = _frequencies(case)
    state["frequencies"] = torch.tensor(f, dtype=torch.float64, device="cuda")
    if own:
        from verinf_amd.prover import generation
        state["plan"] = generation.rotary_plan(case["rotated"], interleaved=case["interleaved"], scaling=SCALINGS[case.get("scaling", "none")])


def _parents(gen, batch, nodes, tree, wide=1):
    """Each sequence's tree: nodes by level, the root first; a chain where it is none.  The first `wide` nodes hang on the root."""
    i = torch.arange(nodes, device="cuda")
    if not tree:
        return (i - 1).expand(batch, nodes).contiguous()
    p = (torch.rand((batch, nodes), generator=gen, device="cuda") * 0.6 * i).long()
    p = torch.where(i <= wide, 0, torch.maximum(p, (i - 1) // 4))
    p = torch.cummax(p, dim=1).values
    p[:, 0] = -1
    return p


def _pages(gen, case, longest):
    """A table of pages in no order, (batch, pages a sequence)."""
    each = -(-longest // case["page"])
    return torch.randperm(case["batch"] * each, generator=gen, device="cuda").view(case["batch"], each).int()


def _cache(gen, case, pages):
    """Keys, values and for 8-bit integers their scales, full of entries."""
    shape = (pages, case["heads"], case["page"], case["dim"])
    out = []
    for _ in range(2):
        if case["cache"] == "int8":
            x = torch.randint(-127, 128, shape, generator=gen, device="cuda", dtype=torch.int8)
            out.append((x, torch.rand(shape[:3], generator=gen, device="cuda") * 0.02 + 0.01))
        else:
            out.append((torch.randn(shape, generator=gen, device="cuda").to(TYPES[case["cache"]]), None))
    return {"keys": out[0][0], "values": out[1][0], "key_scales": out[0][1], "value_scales": out[1][1]}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, state = case["kind"], {"case": case}
    if kind == "rotate":
        x = torch.randn((case["n"], case["heads"], case["dim"] + case["pad"]), generator=gen, device="cuda")
        state["x"] = x.to(TYPES[case["type"]])[:, :, :case["dim"]]
        state["positions"] = torch.randint(0, case["far"], (case["n"],), generator=gen, device="cuda")
        _plan(state, case)
        return state
    batch = case["batch"]
    if kind == "verify":
        n, v = batch * case["nodes"], case["v"]
        t = TYPES[case["type"]]
        logits = torch.randn((n, v), generator=gen, device="cuda") * 3.0
        draft = logits + torch.randn((n, v), generator=gen, device="cuda")          # a draft model that is mostly right
        parents = _parents(gen, batch, case["nodes"], case["tree"])
        state["logits"], state["parents"] = logits.to(t), parents.flatten().int()
        # a node's token is drawn from what the draft model says behind its parent
        noise = torch.rand((n, v), generator=gen, device="cuda").clamp_(min=1e-12).log_().neg_().log_().neg_()
        at = (parents.clamp(min=0) + torch.arange(batch, device="cuda")[:, None] * case["nodes"]).flatten()
        state["tokens"] = torch.argmax(draft.to(t).float()[at] / case["temperature"] + noise, dim=1)
        state["draft"] = draft.to(t) if case["drafted"] else None
        state["uniforms"] = torch.rand((n,), generator=gen, device="cuda", dtype=torch.float64)
        state["starts"] = (torch.arange(batch + 1, device="cuda") * case["nodes"]).int()
        return state
    new = case["nodes"] if kind == "keep" else case["tokens"]
    lengths = torch.full((batch,), case["context"], device="cuda")
    if case.get("ragged"):
        lengths = torch.randint(case["context"] // 16, case["context"] + 1, (batch,), generator=gen, device="cuda")
    state["lengths"] = (lengths + new).int()
    state["longest"] = case["context"] + new
    state["pages"] = _pages(gen, case, state["longest"])
    state["starts"] = (torch.arange(batch + 1, device="cuda") * new).int()
    cache = _cache(gen, case, state["pages"].numel())
    state.update(cache)
    if kind == "append":
        for name in ("k", "v"):
            state[name] = torch.randn((batch * new, case["heads"], case["dim"]), generator=gen, device="cuda").to(TYPES[case["type"]])
        if case["rotated"]:
            _plan(state, case)
    elif kind == "attend":
        state["q"] = torch.randn((batch * new, case["heads"] * case["group"], case["dim"]), generator=gen, device="cuda").to(TYPES[case["type"]])
        if case["tree"]:
            state["parents"] = _parents(gen, batch, new, True, 3).flatten().int()
    else:
        # a path whose entries all lie behind the places they go to, some of it accepted
        step = torch.randint(1, max(1, (new - 1 - case["depth"]) // case["depth"]) + 1, (batch, case["depth"]), generator=gen, device="cuda")
        nodes = case["depth"] + torch.cumsum(step, dim=1)
        counts = torch.randint(0, case["depth"] + 1, (batch,), generator=gen, device="cuda")
        counts[0] = case["depth"]
        state["nodes"] = torch.where(torch.arange(case["depth"], device="cuda") < counts[:, None], nodes, -1)
        state["counts"] = counts
    if own:
        from verinf_amd.prover import generation
        state["cache"] = generation.Cache(**cache)
        state["batch"] = generation.Batch(state["starts"], state["lengths"], state["pages"])
    return state


# ---- one pass -----------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    return _framework(case, state) if own else _plain(case, state)


def _held(state):
    """A cache's entries as the values that they stand for."""
    if state["key_scales"] is None:
        return {"keys": state["keys"], "values": state["values"]}
    return {"keys": state["keys"] * state["key_scales"][..., None], "values": state["values"] * state["value_scales"][..., None]}


def _framework(case, state):
    from verinf_amd.prover import generation
    kind = case["kind"]
    if kind == "rotate":
        return {"out": generation.rotate_heads(state["x"], state["positions"], state["plan"])}
    if kind == "append":
        generation.append_tokens(state["cache"], state["k"], state["v"], state["batch"], plan=state.get("plan"))
        return _held(state)
    if kind == "attend":
        return {"out": generation.attend_cache(state["q"], state["cache"], state["batch"], parents=state.get("parents"), longest=state["longest"])}
    if kind == "verify":
        counts, nodes, tokens = generation.verify_drafts(state["logits"], state["tokens"], state["starts"], state["parents"], state["uniforms"], case["depth"],
                                                         draft_logits=state["draft"], temperature=case["temperature"])
        return {"counts": counts, "nodes": nodes, "tokens": tokens}
    lengths = generation.keep_drafts(state["cache"], state["batch"], state["nodes"], state["counts"])
    if case["cache"] == "int8":     # moved as they are, integers and scales
        return {"keys": state["keys"], "values": state["values"], "key_scales": state["key_scales"], "value_scales": state["value_scales"], "lengths": lengths}
    return {"keys": state["keys"], "values": state["values"], "lengths": lengths}


def _turn(x, positions, state, case, wide=torch.float32):
    """x (n, heads, dim) with its first columns turned, in `wide`; the angles in 64 bits."""
    r = case["rotated"]
    a = positions[:, None].double() * state["frequencies"]
    c, s = ((t * state["amplitude"]).to(wide)[:, None, :] for t in (torch.cos(a), torch.sin(a)))
    x = x.to(wide)
    if case["interleaved"]:
        u, w = x[..., 0:r:2], x[..., 1:r:2]
    else:
        u, w = x[..., :r // 2], x[..., r // 2:r]
    turned = (u * c - w * s, u * s + w * c)
    turned = torch.stack(turned, dim=-1).flatten(-2) if case["interleaved"] else torch.cat(turned, dim=-1)
    return torch.cat((turned, x[..., r:]), dim=-1)


def _places(state, new):
    """Page and row of each new token's entry, (batch * new) each."""
    at = state["lengths"].long()[:, None] - new + torch.arange(new, device="cuda")
    size = state["keys"].shape[2]
    return state["pages"].long().gather(1, at // size).flatten(), (at % size).flatten(), at.flatten()


def _plain(case, state):
    kind = case["kind"]
    if kind == "rotate":
        return {"out": _turn(state["x"], state["positions"], state, case).to(state["x"].dtype)}
    if kind == "verify":
        return _walk(case, state)
    if kind == "attend":
        return {"out": _attention(case, state)}
    if kind == "append":
        page, row, at = _places(state, case["tokens"])
        # which integer an entry becomes is decided next to a border: turned in 64 bits there
        wide = torch.float64 if case["cache"] == "int8" else torch.float32
        rows = _turn(state["k"], at, state, case, wide).float() if case["rotated"] else state["k"].float()
        for name, x in (("key", rows), ("value", state["v"].float())):
            if case["cache"] == "int8":
                most = x.abs().amax(dim=2)
                x = torch.round(x * torch.div(torch.full_like(most, 127.0), most)[..., None])
                state[name + "_scales"][page, :, row] = most / 127.0
            state[name + "s"][page, :, row] = x.to(state[name + "s"].dtype)
        return _held(state)
    n, size = case["nodes"], case["page"]
    first = state["lengths"].long() - n
    order = torch.arange(case["depth"], device="cuda")
    use = order < state["counts"][:, None]
    src, dst = first[:, None] + torch.where(use, state["nodes"], 0), first[:, None] + torch.where(use, order + 1, 0)
    page = [state["pages"].long().gather(1, t // size).flatten() for t in (src, dst)]
    row = [(t % size).flatten() for t in (src, dst)]
    out = {}
    for name in ("keys", "values", "key_scales", "value_scales"):
        if state[name] is not None:
            state[name][page[1], :, row[1]] = state[name][page[0], :, row[0]]
            out[name] = state[name]
    return {**out, "lengths": (first + 1 + state["counts"]).int()}


def _allowed(case, state, longest):
    """(batch, tokens, longest): which keys a token attends to."""
    batch, n = case["batch"], case["tokens"]
    node = torch.arange(longest, device="cuda") - (state["lengths"].long()[:, None, None] - n)              # a key's place among the new tokens
    i = torch.arange(n, device="cuda")[:, None]
    if not case["tree"]:
        return node <= i
    above = (state["parents"].view(batch, n, 1) == torch.arange(n, device="cuda")) | torch.eye(n, dtype=torch.bool, device="cuda")
    for _ in range(n.bit_length()):         # paths of twice as many steps
        above = torch.bmm(above.float(), above.float()) > 0
    return (node < 0) | (above.gather(2, node.clamp(0, n - 1).expand(batch, n, longest)) & (node < n))


def _attention(case, state):
    """All sequences at once, each as if it were as long as the longest: what lies behind its end is masked."""
    batch, n, heads, group, dim = case["batch"], case["tokens"], case["heads"], case["group"], case["dim"]
    longest = state["pages"].shape[1] * case["page"]

    def entries(name, scales):
        pages = state["pages"].long()
        x = state[name][pages].float()
        if case["cache"] == "int8":
            x = x * state[scales][pages][..., None]
        return x.transpose(1, 2).reshape(batch * heads, longest, dim)

    q = state["q"].float().view(batch, n, heads, group, dim).transpose(1, 2).reshape(batch * heads, n * group, dim)
    s = torch.bmm(q, entries("keys", "key_scales").transpose(1, 2).contiguous()).view(batch, heads, n, group, longest)
    s = (s * dim ** -0.5).masked_fill_(~_allowed(case, state, longest)[:, None, :, None], -math.inf)
    p = torch.exp(s - s.amax(dim=4, keepdim=True))
    p = p / p.sum(dim=4, keepdim=True)
    o = torch.bmm(p.view(batch * heads, n * group, longest), entries("values", "value_scales"))
    return o.view(batch, heads, n, group, dim).transpose(1, 2).reshape(batch * n, heads * group, dim).to(state["q"].dtype)


def _softmax64(x, temperature):
    x = x.double() / temperature
    e = torch.exp(x - x.amax(dim=-1, keepdim=True))
    return e / e.sum(dim=-1, keepdim=True)


def _walk(case, state):
    """Every sequence's tree at once, a node after the other in the order of the nodes: a child comes behind its parent."""
    batch, n, depth, t = case["batch"], case["nodes"], case["depth"], case["temperature"]
    seq = torch.arange(batch, device="cuda")
    logits = state["logits"].view(batch, n, -1)
    draft = None if state["draft"] is None else state["draft"].view(batch, n, -1)
    parents, tokens, u = (state[name].view(batch, n).long() if name != "uniforms" else state[name].view(batch, n) for name in ("parents", "tokens", "uniforms"))
    cur, count = torch.zeros(batch, dtype=torch.long, device="cuda"), torch.zeros(batch, dtype=torch.long, device="cuda")
    left = _softmax64(logits[:, 0], t)                   # what is left of the target's probabilities behind the path
    q = None if draft is None else _softmax64(draft[:, 0], t)
    nodes = torch.full((batch, depth), -1, dtype=torch.long, device="cuda")
    out = torch.full((batch, depth + 1), -1, dtype=torch.long, device="cuda")
    for i in range(1, n):
        asked = (parents[:, i] == cur) & (count < depth)
        x = tokens[:, i]
        have = left[seq, x]
        said = torch.ones_like(have) if q is None else q[seq, x]
        took = asked & (u[:, i] * said * left.sum(dim=1) < have)
        place = torch.where(took, count, 0)
        nodes[seq, place] = torch.where(took, i, nodes[seq, place])
        out[seq, place] = torch.where(took, x, out[seq, place])
        cur, count = torch.where(took, i, cur), count + took.long()
        if q is None:
            less = left.scatter(1, x[:, None], 0.0)
        else:
            less = (left / left.sum(dim=1, keepdim=True) - q).clamp(min=0.0)
        left = torch.where(took[:, None], _softmax64(logits[:, i], t), torch.where(asked[:, None], less, left))
        if q is not None:
            q = torch.where(took[:, None], _softmax64(draft[:, i], t), q)
    c = torch.cumsum(left, dim=1)
    last = (c <= u[:, :1] * c[:, -1:]).sum(dim=1)
    out[seq, count] = last
    return {"counts": count, "nodes": nodes, "tokens": out}


# ---- what it costs, what is right ---------------------------------------------------------------------------------
def _size(name):
    return {"f32": 4, "int8": 1}.get(name, 2)


def work(case):
    kind = case["kind"]
    if kind == "rotate":
        n = case["n"] * case["heads"]
        return {"bytes": 2 * n * case["dim"] * _size(case["type"]) + 8 * case["n"], "flops": 3 * n * case["rotated"]}
    if kind == "verify":
        rows = case["batch"] * case["nodes"] * (2 if case["drafted"] else 1)
        return {"bytes": rows * case["v"] * _size(case["type"]) + 20 * case["batch"] * case["nodes"], "flops": 3 * rows * case["v"]}
    entry = case["dim"] * _size(case["cache"]) + (4 if case["cache"] == "int8" else 0)
    if kind == "append":
        n = case["batch"] * case["tokens"] * case["heads"]
        return {"bytes": 2 * n * (case["dim"] * _size(case["type"]) + entry), "flops": 3 * n * case["rotated"] + 2 * n * case["dim"]}
    if kind == "keep":
        return {"bytes": 4 * case["batch"] * case["depth"] / 2 * case["heads"] * entry, "flops": 0}
    context = case["context"] * (17 / 32 if case["ragged"] else 1)
    n = case["batch"] * case["tokens"]
    pairs = n * case["heads"] * case["group"] * (context + (case["tokens"] + 1) / 2)
    return {"bytes": 2 * case["batch"] * (context + case["tokens"]) * case["heads"] * entry + 2 * n * case["heads"] * case["group"] * case["dim"] * _size(case["type"]),
            "flops": 4 * pairs * case["dim"]}


def _turned64(x, positions, case):
    """The turned heads by complex products, in 64 bits."""
    f, amplitude = _frequencies(case)
    r = case["rotated"]
    w = torch.polar(torch.full((1,), amplitude, dtype=torch.float64, device="cuda"), torch.outer(positions.double(), torch.tensor(f, dtype=torch.float64, device="cuda")))[:, None]
    x = x.double().clone()
    pairs = x[..., :r].unflatten(-1, (r // 2, 2)) if case["interleaved"] else x[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2)
    y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * w)
    x[..., :r] = (y if case["interleaved"] else y.transpose(-1, -2)).flatten(-2)
    return x


def exact(case, seed):
    state = prepare(case, seed)
    kind, many = case["kind"], case.get("tokens", 0)
    if kind == "rotate":
        return {"out": _turned64(state["x"], state["positions"], case)}
    if kind == "append":
        held = {k: v.double() for k, v in _held(state).items()}
        for b in range(case["batch"]):
            at = torch.arange(many, device="cuda") + int(state["lengths"][b]) - many
            page, row = state["pages"][b].long()[at // case["page"]], at % case["page"]
            k, v = (state[name][b * many:(b + 1) * many] for name in ("k", "v"))
            for name, x in (("keys", _turned64(k, at, case) if case["rotated"] else k.double()), ("values", v.double())):
                if case["cache"] == "int8":
                    x = x.float().double()                  # what is rounded to integers is held in 32 bits by the definition, and so are
                    top = x.abs().amax(dim=-1, keepdim=True)
                    steps = (127 / top).float().double()    # the steps and the product with them
                    x = (x * steps).float().double().round() * (top / 127)
                held[name][page, :, row] = x
        return held
    if kind == "attend":
        if 4 * case["batch"] * many * case["heads"] * case["group"] * state["longest"] * case["dim"] > 2e13:
            return None
        out, group = [], case["group"]
        for b in range(case["batch"]):
            n = int(state["lengths"][b])
            hidden = torch.ones((many, many), dtype=torch.bool, device="cuda").triu(1)
            if case["tree"]:
                parents = state["parents"][b * many:(b + 1) * many].tolist()
                hidden[:] = True
                for i, p in enumerate(parents):
                    hidden[i, i] = False
                    if p >= 0:
                        hidden[i] &= hidden[p]
                        hidden[i, i] = False
            heads = []
            for h in range(case["heads"]):
                k, v = (state[name][state["pages"][b].long(), h].flatten(0, 1)[:n].double() for name in ("keys", "values"))
                if case["cache"] == "int8":
                    k, v = (t * state[name][state["pages"][b].long(), h].flatten()[:n, None].double() for t, name in ((k, "key_scales"), (v, "value_scales")))
                for g in range(group):
                    s = state["q"][b * many:(b + 1) * many, h * group + g].double() @ k.T / math.sqrt(case["dim"])
                    s[:, n - many:][hidden] = -math.inf
                    heads.append(torch.softmax(s, dim=1) @ v)
            out.append(torch.stack(heads, dim=1))
        return {"out": torch.cat(out)}
    if kind == "keep":
        out = {name: state[name].clone() for name in ("keys", "values", "key_scales", "value_scales") if state[name] is not None}
        lengths = []
        for b in range(case["batch"]):
            first, took = int(state["lengths"][b]) - case["nodes"], int(state["counts"][b])
            for d, node in enumerate(state["nodes"][b, :took].tolist()):
                (p, r), (s, t) = (divmod(first + at, case["page"]) for at in (node, d + 1))
                for x in out.values():
                    x[state["pages"][b, s], :, t] = x[state["pages"][b, p], :, r]
            lengths.append(first + 1 + took)
        return {**out, "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda")}
    counts, paths, said = [], [], []
    for b in range(case["batch"]):
        rows = slice(b * case["nodes"], (b + 1) * case["nodes"])
        parents, tokens, u = (state[name][rows].tolist() for name in ("parents", "tokens", "uniforms"))
        p = torch.softmax(state["logits"][rows].double() / case["temperature"], dim=1)
        q = None if state["draft"] is None else torch.softmax(state["draft"][rows].double() / case["temperature"], dim=1)
        path, left = [0], p[0].clone()
        for i in range(1, case["nodes"]):
            if parents[i] != path[-1] or len(path) > case["depth"]:
                continue
            share = left[tokens[i]] / left.sum() / (1.0 if q is None else q[path[-1], tokens[i]])
            if u[i] < float(share):
                path.append(i)
                left = p[i].clone()
            elif q is None:
                left[tokens[i]] = 0.0
            else:
                left = torch.relu(left / left.sum() - q[path[-1]])
        sums = left.cumsum(0)
        last = int(torch.searchsorted(sums, u[0] * sums[-1], right=True))
        counts.append(len(path) - 1)
        paths.append((path[1:] + [-1] * case["depth"])[:case["depth"]])
        said.append(([tokens[i] for i in path[1:]] + [last] + [-1] * case["depth"])[:case["depth"] + 1])
    return {k: torch.tensor(x, device="cuda") for k, x in (("counts", counts), ("nodes", paths), ("tokens", said))}
