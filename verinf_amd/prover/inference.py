"""A forward pass in 8-bit integers, and what it says of an answer: a tool beside the proof, which nothing in it calls (no counterpart in the
reference; a layer that is proved has 16-bit activations of its own).

    quantize_rows(x)                       rows of floats -> 8-bit integers with a scale each
    int8_matmul(a, b, ...)                 a b^T: exact sums (int32, or field elements, as gl_matmul has them), or scaled
    int8_gated(a, gate, up, ...)           act(a gate^T) * (a up^T), both projections and the activation in one kernel
    token_logprobs(logits, tokens, ...)    log probabilities of given tokens, entropies, the likeliest alternatives

Activations have a scale a token (a row of `a`), weights a scale a channel: they are (n, k), as checkpoints store them, one row a
channel, so `quantize_rows` makes both.  Matrices may be views whose rows are any distance apart; columns have unit stride.
Everything runs on torch's current stream; wrong devices, types, shapes or strides raise RuntimeError.
"""
import torch
from torch.autograd import forward_ad

from .. import _lib

MAX_TOP = 64
MAX_K = 131071

_FLOATS = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_INT8 = (torch.int8,)
_SUMS = {torch.int32: 3, torch.uint64: 4}
_ACTIVATIONS = {"silu": 0, "gelu": 1}


def _refuse(t, name, dtypes, dims, device):
    """Says what is wrong with an argument that _matrix or _vector did not take at once; nothing may be."""
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be CUDA")
    if device is not None and t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, not {device}")
    if t.dtype not in dtypes:
        raise RuntimeError(f"{name} dtype must be {' or '.join(str(d)[6:] for d in dtypes)}")
    if t.dim() != dims:
        raise RuntimeError(f"{name} must have {dims} dimensions")
    if t.is_neg():
        raise RuntimeError(f"{name} is the negative of what its memory holds (take its resolve_neg())")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires a gradient: these operators have none (detach it, or call them under torch.no_grad())")
    if forward_ad._current_level >= 0 and t.is_floating_point() and forward_ad.unpack_dual(t).tangent is not None:
        raise RuntimeError(f"{name} carries a tangent: these operators have no derivative (take the primal of forward_ad.unpack_dual())")


def _matrix(t, name, dtypes, device=None):
    """Rows, columns and how many elements the rows are apart.  The checks are a call's host time, so the usual case is one line."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in dtypes and t.dim() == 2 and not t.requires_grad
            and not t.is_neg() and forward_ad._current_level < 0 and (device is None or t.device == device)):
        _refuse(t, name, dtypes, 2, device)
    m, k = t.shape
    ld, apart = t.stride()
    if k > 1 and apart != 1:
        raise RuntimeError(f"{name} must have unit column stride")
    if m > 1 and ld >= k and ld > 0:
        return m, k, ld
    if m > 1 and k > 0:
        raise RuntimeError(f"{name} has rows that overlap")
    return m, k, (k + 15) & ~15 or 16          # a single row: any distance, one that keeps it aligned


def _vector(t, name, length, dtype, device):
    """The address of a contiguous vector."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == dtype and t.dim() == 1 and not t.requires_grad
            and not t.is_neg() and forward_ad._current_level < 0 and t.device == device):
        _refuse(t, name, (dtype,), 1, device)
    if t.shape[0] != length:
        raise RuntimeError(f"{name} has {t.shape[0]} elements, not {length}")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")
    return t.data_ptr()


def quantize_rows(x):
    """(m, k) float32 / bfloat16 / float16 -> (q, scale): q (m, k) int8 in [-127, 127], scale (m,) float32, x[i] ~ q[i] * scale[i].

    scale = max |x[i]| / 127, q = x[i] * (127 / max |x[i]|) to the nearest integer, half to even, in 32 bits.  A row of zeros
    (or of nothing as large as 127 * 2^-126) has scale 0; one with a NaN or an infinity has scale NaN and integers of zero.  The rows of q are
    a multiple of 16 bytes apart, as the products read them fastest."""
    m, k, ldx = _matrix(x, "x", _FLOATS)
    dev = x.device
    ldq = (k + 15) & ~15 or 16
    q = torch.empty_strided((m, k), (ldq, 1), dtype=torch.int8, device=dev)
    scale = torch.empty(m, dtype=torch.float32, device=dev)
    with _lib.on_device(dev):
        _lib.check(_lib.lib().vi_quantize_rows(_FLOATS[x.dtype], x.data_ptr(), m, k, ldx, q.data_ptr(), ldq, scale.data_ptr(), _lib.stream_ptr()))
    return q, scale


def _weights(who, w, name, k, device):
    """Channels of a weight matrix and how far apart they are."""
    n, kw, ld = _matrix(w, name, _INT8, device)
    if kw != k:
        raise RuntimeError(f"{who}: a has rows of {k}, {name} of {kw}")
    if k > MAX_K:
        raise RuntimeError(f"{who}: an inner dimension of {k}: the 32-bit sums hold {MAX_K}")
    return n, ld


def _aligned(t, ld):
    return not (t.data_ptr() | ld) & 15


def int8_matmul(a, b, a_scale=None, b_scale=None, bias=None, dtype=None):
    """a (m, k) int8 times the transpose of b (n, k) int8.

    Without scales the exact sums: int32 (the default), or with dtype=torch.uint64 the same as field elements, p - |s| below
    zero: what gl_matmul gives for the lifted operands.  With a_scale (m,) and b_scale (n,) float32: (s * a_scale) * b_scale
    (+ bias (n,) float32) in 32 bits, rounded once to dtype: bfloat16 (the default), float16 or float32."""
    m, k, lda = _matrix(a, "a", _INT8)
    dev = a.device
    n, ldb = _weights("int8_matmul", b, "b", k, dev)
    scaled = a_scale is not None or b_scale is not None
    if dtype is None:
        dtype = torch.bfloat16 if scaled else torch.int32
    sa = sb = sbias = None
    if scaled:
        if a_scale is None or b_scale is None:
            raise RuntimeError("int8_matmul: both scales or none")
        if dtype not in _FLOATS:
            raise RuntimeError(f"int8_matmul: scaled sums are no {dtype}")
        sa = _vector(a_scale, "a_scale", m, torch.float32, dev)
        sb = _vector(b_scale, "b_scale", n, torch.float32, dev)
        if bias is not None:
            sbias = _vector(bias, "bias", n, torch.float32, dev)
    else:
        if bias is not None:
            raise RuntimeError("int8_matmul: a bias needs scales")
        if dtype not in _SUMS:
            raise RuntimeError(f"int8_matmul: without scales the sums are int32 or uint64, not {dtype}")
    out = torch.empty(m, n, dtype=dtype, device=dev)
    if m == 0 or n == 0:
        return out
    kind = _FLOATS[dtype] if scaled else _SUMS[dtype]
    L = _lib.lib()
    with _lib.on_device(dev):
        sp = _lib.stream_ptr()
        need = _lib.workspace_bytes("int8_matmul" if _aligned(a, lda) and _aligned(b, ldb) else "int8_matmul_best", m, k, n)
        args = (a.data_ptr(), lda, b.data_ptr(), ldb, m, k, n, sa, sb, sbias, kind, out.data_ptr(), n)
        if not need:
            _lib.check(L.vi_int8_matmul(*args, None, 0, sp))
            return out
        with _lib.stream_lock(sp):
            ws = _lib.workspace(need, "int8", sp)
            _lib.check(L.vi_int8_matmul(*args, ws.data_ptr(), need, sp))
    return out


def int8_gated(a, gate, up, a_scale, gate_scale, up_scale, activation="silu", dtype=torch.bfloat16):
    """act(G) * U, G and U the scaled products of a (m, k) with gate and up, (n, k) int8 each, as `int8_matmul` has them in 32 bits:
    a gated feed-forward block up to its last projection, (m, n), rounded once to dtype (bfloat16, float16 or float32).

    activation: "silu" x / (1 + e^-x), or "gelu" x Phi(x)."""
    m, k, lda = _matrix(a, "a", _INT8)
    dev = a.device
    n, ldg = _weights("int8_gated", gate, "gate", k, dev)
    nu, ldu = _weights("int8_gated", up, "up", k, dev)
    if nu != n:
        raise RuntimeError(f"int8_gated: gate has {n} channels, up {nu}")
    if activation not in _ACTIVATIONS:
        raise RuntimeError(f"int8_gated: no activation {activation!r}")
    if dtype not in _FLOATS:
        raise RuntimeError(f"int8_gated: no outputs of {dtype}")
    sa = _vector(a_scale, "a_scale", m, torch.float32, dev)
    sg = _vector(gate_scale, "gate_scale", n, torch.float32, dev)
    su = _vector(up_scale, "up_scale", n, torch.float32, dev)
    out = torch.empty(m, n, dtype=dtype, device=dev)
    if m == 0 or n == 0:
        return out
    L = _lib.lib()
    with _lib.on_device(dev):
        sp = _lib.stream_ptr()
        need = _lib.workspace_bytes("int8_gated" if _aligned(a, lda) and _aligned(gate, ldg) and _aligned(up, ldu) else "int8_gated_best", m, k, n)
        args = (a.data_ptr(), lda, gate.data_ptr(), ldg, up.data_ptr(), ldu, m, k, n, sa, sg, su, _ACTIVATIONS[activation], _FLOATS[dtype],
                out.data_ptr(), n)
        if not need:
            _lib.check(L.vi_int8_gated(*args, None, 0, sp))
            return out
        with _lib.stream_lock(sp):
            ws = _lib.workspace(need, "int8", sp)
            _lib.check(L.vi_int8_gated(*args, ws.data_ptr(), need, sp))
    return out


def token_logprobs(logits, tokens, top=0, temperature=1.0):
    """Log probabilities of tokens (m,) int64 under the rows of logits (m, v) / temperature, float32 / bfloat16 / float16.

    Returns (logprob (m,), entropy (m,), top_logprobs (m, top), top_tokens (m, top) int64): float32 in nats, and the `top` <= 64
    largest entries of each row in falling order, equal logits by the lowest index.  A token of -1 is not scored (logprob 0), another
    one outside [0, v) gives NaN.  Logits of -inf have log probability -inf and add nothing; a row of nothing else has entropy 0.
    A NaN or +inf makes its row NaN, except for top_tokens (NaN first, then +inf)."""
    m, v, ld = _matrix(logits, "logits", _FLOATS)
    dev = logits.device
    t = _vector(tokens, "tokens", m, torch.int64, dev)
    top, temperature = int(top), float(temperature)
    if not 0 <= top <= MAX_TOP or top > v:
        raise RuntimeError(f"token_logprobs: the {top} largest of {v} ({MAX_TOP} at most)")
    logprob = torch.empty(m, dtype=torch.float32, device=dev)
    entropy = torch.empty(m, dtype=torch.float32, device=dev)
    top_logprobs = torch.empty(m, top, dtype=torch.float32, device=dev)
    top_tokens = torch.empty(m, top, dtype=torch.int64, device=dev)
    kind = _FLOATS[logits.dtype]
    L = _lib.lib()
    with _lib.on_device(dev):
        sp = _lib.stream_ptr()
        need = _lib.workspace_bytes("token_logprobs", kind, m, v, top)
        args = (kind, logits.data_ptr(), m, v, ld, t, temperature, top, logprob.data_ptr(), entropy.data_ptr(), top_logprobs.data_ptr(),
                top_tokens.data_ptr())
        if not need:
            _lib.check(L.vi_token_logprobs(*args, None, 0, sp))
            return logprob, entropy, top_logprobs, top_tokens
        with _lib.stream_lock(sp):
            ws = _lib.workspace(need, "logprobs", sp)
            _lib.check(L.vi_token_logprobs(*args, ws.data_ptr(), need, sp))
    return logprob, entropy, top_logprobs, top_tokens
