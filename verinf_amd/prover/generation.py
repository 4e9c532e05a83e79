"""Answering with a cache of keys and values and with drafted tokens: what stands between the products of a forward pass (`inference`) and
its next token.  A tool beside the proof, as that is (no counterpart in the reference).

    rotary_plan(dim, ...)                         the frequencies of rotary positions, scaled for long contexts where asked
    rotate_heads(x, positions, plan)              heads turned by their tokens' positions
    new_cache(pages, heads, page_size, dim, ...)  a paged cache: bfloat16, float16, or int8 with a scale an entry
    append_tokens(cache, k, v, batch, ...)        new tokens' keys, turned, and values into it
    attend_cache(q, cache, batch, ...)            attention of the new tokens: one a sequence, a prompt's, or a tree of drafts
    verify_drafts(logits, tokens, ...)            a tree of drafts against the target's probabilities, from given random numbers
    keep_drafts(cache, batch, nodes, counts)      the accepted path's entries moved to where the next tokens follow them

A `Cache` and a `Batch` hold tensors whose contents change from step to step; what they check of them they check once, when they are made.  Everything runs
on torch's current stream and can be captured; wrong devices, types, shapes or strides raise RuntimeError.
"""
import ctypes
import math

import torch
from torch.autograd import forward_ad

from .. import _lib
from .inference import _FLOATS, _matrix, _refuse, _vector

MAX_DEPTH = 256
MAX_VOCABULARY = 1 << 20

_KINDS = {**_FLOATS, torch.int8: 5}
_CACHED = (torch.bfloat16, torch.float16, torch.int8)


def _tensor(t, name, dtypes, dims, device):
    """What `_matrix` checks before it looks at strides, for any number of dimensions."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in dtypes and t.dim() == dims and (device is None or t.device == device)
            and not t.requires_grad and not t.is_neg() and forward_ad._current_level < 0):
        _refuse(t, name, dtypes, dims, device)


def _heads(t, name, dtypes, device, out=False):
    """Tokens, heads and columns, and how many elements tokens and heads are apart; columns have unit stride."""
    _tensor(t, name, dtypes, 3, device)
    n, heads, dim = t.shape
    token, head, apart = t.stride()
    if dim > 1 and apart != 1:
        raise RuntimeError(f"{name} must have unit column stride")
    if out and n and heads and dim and _overlaps(t):
        raise RuntimeError(f"{name} has heads that overlap")
    # the distance of a single token or head means nothing
    return n, heads, dim, token if n > 1 else max(token, dim), head if heads > 1 else max(head, dim)


def _overlaps(t):
    """Whether two elements of a tensor may share memory: its strides, from the least, do not hold each what lies inside."""
    inside = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride < inside:
            return True
        inside = stride * (size - 1) + inside
    return False


class _Fixed:
    """What is checked once and goes into every call as it is: made anew where it is to be another."""
    __slots__ = ()

    def _fix(self, **values):
        for name, value in values.items():
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value):
        raise AttributeError(f"{type(self).__name__}.{name} cannot be changed: make another {type(self).__name__}")

    __delattr__ = lambda self, name: self.__setattr__(name, None)              # noqa: E731


class RotaryPlan(_Fixed):
    """Frequencies as whole numbers of 2^-64 turns a position, so that the angle of any position is exact.  Cannot be changed."""
    __slots__ = ("steps", "rotated", "interleaved", "amplitude")

    def __init__(self, steps, rotated, interleaved, amplitude):
        if steps.dtype != torch.int64 or steps.dim() != 1 or not steps.is_contiguous() or 2 * steps.shape[0] != rotated:
            raise RuntimeError(f"a plan of {tuple(steps.shape)} steps for {rotated} columns")
        self._fix(steps=steps, rotated=int(rotated), interleaved=bool(interleaved), amplitude=float(amplitude))


def rotary_plan(dim, base=10000.0, interleaved=False, scaling=None, device="cuda"):
    """Rotary positions of the first `dim` columns of a head: pair i turns by base^(-2 i / dim) radians a position.

    Pairs are columns (i, i + dim / 2), or interleaved (2 i, 2 i + 1).  For contexts longer than a model was trained on, scaling is
    ("linear", factor): all frequencies divided by factor; ("base", factor): base times factor^(dim / (dim - 2)), so that the slowest pair is
    divided by it; ("parts", factor, length[, low, high]): pairs that turn more than `high` (32) times in `length` positions stay, those under
    `low` (1) times are divided, those between in proportion, and what is turned is multiplied by 0.1 ln(factor) + 1."""
    dim = int(dim)
    if dim < 2 or dim > 256 or dim % 2:
        raise RuntimeError(f"rotary_plan: {dim} columns (even, up to 256)")
    if not (base > 1 and math.isfinite(base)):
        raise RuntimeError(f"rotary_plan: a base of {base}")
    try:
        kind, factor, *more = scaling or (None, 1.0)
    except (TypeError, ValueError):
        raise RuntimeError(f"rotary_plan: no scaling {scaling!r}") from None
    if kind not in (None, "linear", "base", "parts") or (kind == "parts") != (len(more) in (1, 3)) or (kind != "parts" and more):
        raise RuntimeError(f"rotary_plan: no scaling {scaling!r}")
    if not (factor >= 1 and math.isfinite(factor)):
        raise RuntimeError(f"rotary_plan: a factor of {factor}")
    half = dim // 2
    if kind == "base" and half > 1:
        # base factor^(half / (half - 1)), which is beyond what a power gives where it is infinite
        if math.log(base) + math.log(factor) * half / (half - 1) >= 709.0:
            raise RuntimeError(f"rotary_plan: a base of {base} and a factor of {factor}")
        base = base * factor ** (half / (half - 1))
    radians = [base ** (-i / half) for i in range(half)]
    amplitude = 1.0
    if kind == "linear":
        radians = [f / factor for f in radians]
    if kind == "parts":
        length, low, high = more[0], *(more[1:] or (1.0, 32.0))
        if not (length > 0 and high > low):
            raise RuntimeError(f"rotary_plan: no scaling {scaling!r}")
        keep = [min(1.0, max(0.0, (length * f / (2 * math.pi) - low) / (high - low))) for f in radians]
        radians = [f * k + f / factor * (1.0 - k) for f, k in zip(radians, keep)]
        amplitude = 0.1 * math.log(factor) + 1.0
    # a double's 53 bits as a whole number of 2^-64 turns, below a turn
    words = [round(f / (2 * math.pi) * 2.0 ** 64) % (1 << 64) for f in radians]
    steps = torch.tensor([w - (1 << 64) if w >> 63 else w for w in words], dtype=torch.int64, device=device)
    return RotaryPlan(steps, dim, bool(interleaved), amplitude)


def _turn(plan, device, dim, who):
    """A plan's address and numbers, as the entries take them."""
    if not isinstance(plan, RotaryPlan):
        raise RuntimeError(f"{who}: plan must be what rotary_plan() returns")
    if plan.steps.device != device:
        raise RuntimeError(f"{who}: plan is on {plan.steps.device}, not {device}")
    if plan.rotated > dim:
        raise RuntimeError(f"{who}: {plan.rotated} of {dim} columns rotated")
    return plan.steps.data_ptr(), plan.rotated, plan.interleaved, plan.amplitude


def rotate_heads(x, positions, plan, out=None):
    """x (n, heads, dim) float32 / bfloat16 / float16 with the first columns of each head turned by its token's position (n,) int64, in 32
    bits; the others as they are.  dim even, up to 256.  out: where to (x itself, to turn it in place); a new tensor by default."""
    n, heads, dim, x_token, x_head = _heads(x, "x", _FLOATS, None)
    dev = x.device
    p = _vector(positions, "positions", n, torch.int64, dev)
    turn = _turn(plan, dev, dim, "rotate_heads")
    if out is None:
        out = torch.empty((n, heads, dim), dtype=x.dtype, device=dev)
        o_token, o_head = heads * dim, dim
    else:
        shape = _heads(out, "out", (x.dtype,), dev, True)
        if shape[:3] != (n, heads, dim):
            raise RuntimeError(f"rotate_heads: out is {tuple(out.shape)}, x {tuple(x.shape)}")
        o_token, o_head = shape[3:]
    if n and heads:
        with _lib.on_device(dev):
            _lib.check(_lib.lib().vi_rotate_heads(_FLOATS[x.dtype], x.data_ptr(), n, heads, dim, x_token, x_head, p, *turn, out.data_ptr(), o_token, o_head,
                                                  _lib.stream_ptr()))
    return out


class Cache(_Fixed):
    """A paged cache: keys and values (pages, heads, page_size, dim) bfloat16, float16 or int8, int8 with key_scales and value_scales
    (pages, heads, page_size) float32, of which an infinite one counts as NaN.  Columns have unit stride, the rest any, so that views do: entries start at multiples of 16 bytes.
    page_size a power of two from 16 to 1024, dim a multiple of 16 up to 256.  Cannot be changed but in what its tensors hold: they are not resized."""
    __slots__ = ("keys", "values", "key_scales", "value_scales", "device", "_args")

    def __init__(self, keys, values, key_scales=None, value_scales=None):
        _tensor(keys, "keys", _CACHED, 4, None)
        dev = keys.device
        _tensor(values, "values", (keys.dtype,), 4, dev)
        if values.shape != keys.shape:
            raise RuntimeError(f"values are {tuple(values.shape)}, keys {tuple(keys.shape)}")
        pages, heads, size, dim = keys.shape
        if size < 16 or size > 1024 or size & (size - 1) or dim < 16 or dim > 256 or dim % 16 or heads < 1:
            raise RuntimeError(f"a cache of {heads} heads, pages of {size} entries of {dim} (heads, powers of two from 16 to 1024, multiples of 16 up to 256)")
        for name, t in (("keys", keys), ("values", values)):
            if t.stride(3) != 1 or (pages and _overlaps(t)):
                raise RuntimeError(f"{name} must have unit column stride and entries that do not overlap")
            if (t.data_ptr() | t.element_size() * (t.stride(0) | t.stride(1) | t.stride(2))) & 15:
                raise RuntimeError(f"{name} must have entries at multiples of 16 bytes")
        scaled = keys.dtype == torch.int8
        scale_strides = []
        for name, t in (("key_scales", key_scales), ("value_scales", value_scales)):
            if scaled:
                _tensor(t, name, (torch.float32,), 3, dev)
                if t.shape != keys.shape[:3] or t.stride(2) != 1 or (pages and _overlaps(t)):
                    raise RuntimeError(f"{name} must be {tuple(keys.shape[:3])}, the last with unit stride")
                scale_strides.append((ctypes.c_int64 * 2)(*t.stride()[:2]))
            elif t is not None:
                raise RuntimeError(f"{name} go with a cache of int8")
            else:
                scale_strides.append((ctypes.c_int64 * 2)())
        args = _lib.CacheArgs(keys.data_ptr(), values.data_ptr(), key_scales.data_ptr() if scaled else None, value_scales.data_ptr() if scaled else None,
                              (ctypes.c_int64 * 3)(*keys.stride()[:3]), (ctypes.c_int64 * 3)(*values.stride()[:3]), *scale_strides,
                              pages, heads, size, dim, _KINDS[keys.dtype])
        self._fix(keys=keys, values=values, key_scales=key_scales, value_scales=value_scales, device=dev, _args=args)


def new_cache(pages, heads, page_size, dim, dtype=torch.bfloat16, device="cuda"):
    """An empty cache, keys and values of a page next to each other."""
    if dtype not in _CACHED:
        raise RuntimeError(f"a cache of {dtype}")
    both = torch.zeros((pages, 2, heads, page_size, dim), dtype=dtype, device=device)
    if dtype != torch.int8:
        return Cache(both[:, 0], both[:, 1])
    scales = torch.zeros((pages, 2, heads, page_size), device=device)
    return Cache(both[:, 0], both[:, 1], scales[:, 0], scales[:, 1])


class Batch(_Fixed):
    """Which rows of the new tokens' tensors belong to which sequence, and where its entries lie: starts (sequences + 1,), rising,
    lengths (sequences,), the entries of a sequence with the new tokens', and pages (sequences, most pages), all int32.

    Entry j of a sequence lies in row j % page_size of page pages[b, j // page_size]; the new tokens' are its last.  Rows of no sequence are
    left alone.  A page outside the cache holds nothing: it is not written, what it should hold is masked.  Two sequences may share pages that
    neither of them writes.  Cannot be changed but in what its tensors hold, which every call reads anew: they are not resized."""
    __slots__ = ("starts", "lengths", "pages", "device", "_args")

    def __init__(self, starts, lengths, pages):
        _tensor(pages, "pages", (torch.int32,), 2, None)
        dev, (sequences, width) = pages.device, pages.shape
        if width > 1 and pages.stride(1) != 1:
            raise RuntimeError("pages must have unit column stride")
        stride = pages.stride(0) if sequences > 1 else width
        if sequences > 1 and width and stride < width:
            raise RuntimeError("pages has rows that overlap")
        args = _lib.BatchArgs(_vector(starts, "starts", sequences + 1, torch.int32, dev), _vector(lengths, "lengths", sequences, torch.int32, dev),
                              pages.data_ptr(), sequences, width, max(stride, width))
        self._fix(starts=starts, lengths=lengths, pages=pages, device=dev, _args=args)


def _both(cache, batch, who):
    if not isinstance(cache, Cache) or not isinstance(batch, Batch):
        raise RuntimeError(f"{who}: a Cache and a Batch")
    if batch.device != cache.device:
        raise RuntimeError(f"{who}: batch is on {batch.device}, not {cache.device}")
    return cache.device


def append_tokens(cache, k, v, batch, positions=None, plan=None):
    """New tokens' keys and values (n, heads, dim) float32 / bfloat16 / float16 into the cache, each sequence's as its last entries.

    plan: keys are turned first, by positions (n,) int64, or by the entries' numbers in their sequences (a tree's drafts need positions: their
    depths behind the context).  Into int8 as `quantize_rows` has it, a scale an entry, from keys turned in 64 bits and rounded to 32."""
    dev = _both(cache, batch, "append_tokens")
    n, heads, dim, k_token, k_head = _heads(k, "k", _FLOATS, dev)
    vn, vheads, vdim, v_token, v_head = _heads(v, "v", (k.dtype,), dev)
    a = cache._args
    if (n, heads, dim) != (vn, vheads, vdim) or (heads, dim) != (a.heads, a.dim):
        raise RuntimeError(f"append_tokens: k is {tuple(k.shape)}, v {tuple(v.shape)}, over a cache of {a.heads} heads of {a.dim}")
    p = None if positions is None else _vector(positions, "positions", n, torch.int64, dev)
    turn = (None, 0, False, 1.0) if plan is None else _turn(plan, dev, dim, "append_tokens")
    if n:
        with _lib.on_device(dev):
            _lib.check(_lib.lib().vi_append_tokens(a, batch._args, _FLOATS[k.dtype], k.data_ptr(), k_token, k_head, v.data_ptr(), v_token, v_head, n, p, *turn,
                                                   _lib.stream_ptr()))


def attend_cache(q, cache, batch, parents=None, scale=None, longest=None, out=None):
    """softmax(scale q k^T) v of new tokens q (n, heads, dim) over the entries of their sequences, with theirs in the cache already.

    bfloat16 or float16 as the cache's (bfloat16 over int8); groups of heads / cache heads share one of the cache's; scale: dim^-0.5.  A new token
    attends to what its sequence had before and to the new tokens up to itself; with parents (n,) int32, in the place of those to its ancestors: a
    token's parent as a number in its sequence, below its own (-1: none).  A sequence with more than 256 new tokens is taken for a chain,
    whatever parents says of it.  A token that attends to nothing gets zeros.  Over int8 queries are below 2^100.  longest: no sequence has more entries (it decides how the work is cut, nothing else).  out: where to; a new
    tensor by default, whose rows of no sequence are zero."""
    dev = _both(cache, batch, "attend_cache")
    a = cache._args
    n, heads, dim, q_token, q_head = _heads(q, "q", (torch.float16 if cache.keys.dtype == torch.float16 else torch.bfloat16,), dev)
    if dim != a.dim or not heads or heads % a.heads:
        raise RuntimeError(f"attend_cache: {heads} heads of {dim} over a cache of {a.heads} of {a.dim}")
    above = None if parents is None else _vector(parents, "parents", n, torch.int32, dev)
    scale = dim ** -0.5 if scale is None else float(scale)
    most = batch._args.width * a.page_size
    longest = most if longest is None else min(max(int(longest), 0), most)
    clear = out is None
    if clear:
        out = torch.empty((n, heads, dim), dtype=q.dtype, device=dev)
        o_token, o_head = heads * dim, dim
    else:
        shape = _heads(out, "out", (q.dtype,), dev, True)
        if shape[:3] != (n, heads, dim):
            raise RuntimeError(f"attend_cache: out is {tuple(out.shape)}, q {tuple(q.shape)}")
        o_token, o_head = shape[3:]
    if n == 0:
        return out
    L = _lib.lib()
    with _lib.on_device(dev):
        sp = _lib.stream_ptr()
        need = _lib.workspace_bytes("attend_cache", a.dtype, dim, a.heads, n, heads, max(batch._args.sequences, 1), longest)
        args = (a, batch._args, _FLOATS[q.dtype], q.data_ptr(), n, heads, q_token, q_head, above, scale, longest, clear, out.data_ptr(), o_token, o_head)
        if not need:
            _lib.check(L.vi_attend_cache(*args, None, 0, sp))
            return out
        with _lib.stream_lock(sp):
            ws = _lib.workspace(need, "attend", sp)
            _lib.check(L.vi_attend_cache(*args, ws.data_ptr(), need, sp))
    return out


def verify_drafts(logits, tokens, starts, parents, uniforms, depth, draft_logits=None, temperature=1.0):
    """Trees of drafted tokens against what the target says of them, so that the tokens that come out are distributed as the target's own.

    A sequence's nodes are rows starts[b] .. starts[b + 1] - 1: a root, whose token is known already, and drafts; parents (n,) int32, a node's parent
    as a number in the sequence, below its own (None: chains).  logits (n, v): row i is the target's behind node i; tokens (n,) int64; uniforms (n,)
    float64 in [0, 1).  From the root on, a node's children are tried in their order: with p = softmax(logits / temperature), child c with token x is
    accepted where uniforms[c] q(x) < p(x), and p becomes max(p - q, 0), scaled to sum to one, behind a refused one.  q is softmax(draft_logits /
    temperature) of the node's row, from which its children have been drawn; without draft_logits it is 1 and p loses the refused token.  Behind the last
    accepted, or `depth` <= 256 of them, comes the token at which p's running sum exceeds uniforms[root].

    Returns (counts (sequences,), nodes (sequences, depth), out (sequences, depth + 1)), int64: accepted drafts, their numbers in the sequence, -1
    behind; their tokens, the one that follows, -1 behind.  All in 64 bits.  A row with a NaN or +inf, or only -inf, has no probabilities: no draft
    below it is accepted, and the token that follows it is -1.  An entry less than 2^-1022 of its row's largest has none either (-inf, or masked far down): it
    is neither accepted nor the token that follows, and as the draft's counts as never drawn.  Drafts whose token is outside [0, v) or whose parent is none are refused; v is at most
    2^20, and a sequence's first 1024 nodes are tried (attend_cache has trees of 256 at most)."""
    n, v, ld = _matrix(logits, "logits", _FLOATS)
    dev = logits.device
    ids = _vector(tokens, "tokens", n, torch.int64, dev)
    _tensor(starts, "starts", (torch.int32,), 1, dev)
    sequences, depth, temperature = starts.shape[0] - 1, int(depth), float(temperature)
    if sequences < 0:
        raise RuntimeError("starts has 0 elements: sequences + 1")
    at = _vector(starts, "starts", sequences + 1, torch.int32, dev)
    above = None if parents is None else _vector(parents, "parents", n, torch.int32, dev)
    u = _vector(uniforms, "uniforms", n, torch.float64, dev)
    if not 0 <= depth <= MAX_DEPTH:
        raise RuntimeError(f"verify_drafts: a depth of {depth} ({MAX_DEPTH} at most)")
    if not 1 <= v <= MAX_VOCABULARY:
        raise RuntimeError(f"verify_drafts: rows of {v} logits ({MAX_VOCABULARY} at most)")
    draft, ld_draft = None, 0
    if draft_logits is not None:
        dn, dv, ld_draft = _matrix(draft_logits, "draft_logits", (logits.dtype,), dev)
        if (dn, dv) != (n, v):
            raise RuntimeError(f"verify_drafts: draft_logits are {dn, dv}, logits {n, v}")
        draft = draft_logits.data_ptr() or None
    counts = torch.empty(sequences, dtype=torch.int64, device=dev)
    nodes = torch.empty((sequences, depth), dtype=torch.int64, device=dev)
    out = torch.empty((sequences, depth + 1), dtype=torch.int64, device=dev)
    if sequences == 0:
        return counts, nodes, out
    kind = _FLOATS[logits.dtype]
    L = _lib.lib()
    with _lib.on_device(dev):
        sp = _lib.stream_ptr()
        need = _lib.workspace_bytes("verify_drafts", kind, n, v, sequences, int(draft is not None))
        with _lib.stream_lock(sp):
            ws = _lib.workspace(need, "drafts", sp)
            _lib.check(L.vi_verify_drafts(kind, logits.data_ptr(), n, v, ld, draft, ld_draft, ids, at, sequences, above, u, temperature, depth, counts.data_ptr(),
                                          nodes.data_ptr(), out.data_ptr(), ws.data_ptr(), need, sp))
    return counts, nodes, out


def keep_drafts(cache, batch, nodes, counts):
    """The entries of accepted drafts moved to where the next tokens follow them: of each sequence's new entries, node nodes[b, d]'s becomes the
    (d + 1)th behind the root's, for d < counts[b].  nodes (sequences, depth) and counts (sequences,) int64 as verify_drafts gives them; numbers rise along a
    path, which ends in front of one that does not or that is none of the sequence's.

    Returns the entries that the sequences have then, (sequences,) int32: the root's is the last of those before, the path's follow.  Where the
    caches of several layers lie together page by page, as (pages, layers * heads, page_size, dim), one call moves all of them."""
    dev = _both(cache, batch, "keep_drafts")
    sequences = batch._args.sequences
    _tensor(nodes, "nodes", (torch.int64,), 2, dev)
    if nodes.shape[0] != sequences or not nodes.is_contiguous():
        raise RuntimeError(f"keep_drafts: nodes must be contiguous, a row for each of {sequences} sequences")
    if nodes.shape[1] > MAX_DEPTH:
        raise RuntimeError(f"keep_drafts: a depth of {nodes.shape[1]} ({MAX_DEPTH} at most)")
    took = _vector(counts, "counts", sequences, torch.int64, dev)
    lengths = torch.empty(sequences, dtype=torch.int32, device=dev)
    if sequences:
        with _lib.on_device(dev):
            _lib.check(_lib.lib().vi_keep_drafts(cache._args, batch._args, nodes.data_ptr() or None, nodes.shape[1], took, lengths.data_ptr(), _lib.stream_ptr()))
    return lengths
