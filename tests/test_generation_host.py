"""The cache's, the attention's and the drafts' operators without a GPU: argument checks of the C entries and of the Python functions."""
import ctypes
import math
import os

import pytest

torch = pytest.importorskip("torch")
from verinf_amd import _lib  # noqa: E402


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(_lib.LIB_PATH):
        from verinf_amd.build import build
        build()
    return _lib.lib()


P = 0x1000                                     # never dereferenced


def cache(**other):
    c = _lib.CacheArgs(P, P, P, P, (ctypes.c_int64 * 3)(2 * 16 * 64, 16 * 64, 64), (ctypes.c_int64 * 3)(2 * 16 * 64, 16 * 64, 64), (ctypes.c_int64 * 2)(32, 16), (ctypes.c_int64 * 2)(32, 16),
                       10, 2, 16, 64, 1)
    for name, value in other.items():
        setattr(c, name, value if not isinstance(value, tuple) else (ctypes.c_int64 * len(value))(*value))
    return c


def batch(**other):
    b = _lib.BatchArgs(P, P, P, 3, 4, 4)
    for name, value in other.items():
        setattr(b, name, value)
    return b


def test_entries_refuse_before_any_launch(L):
    def said(rc, code, word):
        assert rc == code and word in L.vi_last_error(), (rc, L.vi_last_error())

    def rotate(dtype=1, x=P, n=2, heads=3, dim=64, xt=192, xh=64, p=P, steps=P, rotated=64, amplitude=1.0, out=P, ot=192, oh=64):
        return L.vi_rotate_heads(dtype, x, n, heads, dim, xt, xh, p, steps, rotated, 0, amplitude, out, ot, oh, None)

    said(rotate(dtype=3), -1, b"dtype")
    said(rotate(n=-1), -1, b"tokens")
    said(rotate(dim=63), -1, b"heads of 63")
    said(rotate(dim=258, rotated=2), -1, b"258")
    said(rotate(rotated=63), -1, b"rotated")
    said(rotate(rotated=66), -1, b"rotated")
    said(rotate(steps=None), -1, b"null")
    said(rotate(amplitude=math.nan), -1, b"amplitude")
    said(rotate(ot=63), -1, b"overlap")
    said(rotate(oh=63), -1, b"overlap")
    for name in ("x", "p", "out"):
        said(rotate(**{name: None}), -1, b"null")
    assert rotate(n=0, x=None, p=None, out=None) == 0

    def append(c=cache(), b=batch(), dtype=1, k=P, n=5, steps=P, rotated=64):
        return L.vi_append_tokens(c, b, dtype, k, 128, 64, P, 128, 64, n, None, steps, rotated, 0, 1.0, None)

    said(append(dtype=5), -1, b"dtype")
    said(append(k=None), -1, b"null")
    said(append(n=-1), -1, b"tokens")
    said(append(rotated=65), -1, b"rotated")
    said(append(c=None), -1, b"null")
    said(append(b=None), -1, b"null")
    assert append(n=0, k=None) == 0 and append(b=batch(sequences=0, lengths=None, pages=None)) == 0 and append(c=cache(pages=0, keys=None)) == 0

    def attend(c=cache(), b=batch(), dtype=1, q=P, n=5, heads=4, scale=1.0, longest=64, out=P, ot=256, oh=64, ws=None, ws_bytes=0):
        return L.vi_attend_cache(c, b, dtype, q, n, heads, 256, 64, None, scale, longest, 1, out, ot, oh, ws, ws_bytes, None)

    for dtype in (0, 2, 5):
        said(attend(dtype=dtype), -1, b"dtype")
    said(attend(c=cache(dtype=5), dtype=2), -1, b"dtype")
    said(attend(heads=3), -1, b"heads")
    said(attend(heads=0), -1, b"heads")
    said(attend(n=1 << 30), -1, b"tokens")
    for scale in (0.0, -1.0, math.nan, math.inf):
        said(attend(scale=scale), -1, b"scale")
    said(attend(longest=-1), -1, b"longer")
    said(attend(ot=63), -1, b"overlap")
    said(attend(q=None), -1, b"null")
    said(attend(b=batch(width=1000, stride=1000), longest=16000), -3, b"workspace")
    assert attend(n=0, q=None) == 0
    assert L.vi_attend_cache_workspace_bytes(1, 64, 2, 5, 4, 3, 16000) > 0
    assert L.vi_attend_cache_workspace_bytes(1, 64, 2, 5, 3, 3, 16000) == 0 and L.vi_attend_cache_workspace_bytes(0, 64, 2, 5, 4, 3, 16000) == 0

    def verify(dtype=0, x=P, n=6, v=10, ld=10, draft=None, ld_draft=0, tokens=P, sequences=2, t=1.0, depth=3, nodes=P, out=P, ws=P, ws_bytes=1 << 30):
        return L.vi_verify_drafts(dtype, x, n, v, ld, draft, ld_draft, tokens, P, sequences, P, P, t, depth, P, nodes, out, ws, ws_bytes, None)

    said(verify(dtype=3), -1, b"dtype")
    said(verify(v=0), -1, b"logits")
    said(verify(v=(1 << 20) + 1, ld=1 << 21), -1, b"logits")
    said(verify(ld=9), -1, b"apart")
    said(verify(draft=P, ld_draft=9), -1, b"apart")
    said(verify(sequences=-1), -1, b"sequences")
    said(verify(depth=257), -1, b"depth")
    said(verify(depth=-1), -1, b"depth")
    for t in (0.0, -1.0, math.nan, math.inf):
        said(verify(t=t), -1, b"temperature")
    for name in ("x", "tokens", "nodes", "out"):
        said(verify(**{name: None}), -1, b"null")
    need = L.vi_verify_drafts_workspace_bytes(0, 6, 10, 2, 0)
    said(verify(ws_bytes=need - 1), -3, b"workspace")
    said(verify(ws=None), -3, b"workspace")
    assert verify(sequences=0) == 0 and L.vi_verify_drafts_workspace_bytes(0, 6, 10, 2, 1) > need

    def keep(c=cache(), b=batch(), nodes=P, depth=3, counts=P, lengths=P + 16):
        return L.vi_keep_drafts(c, b, nodes, depth, counts, lengths, None)

    said(keep(depth=257), -1, b"depth")
    for name in ("nodes", "counts", "lengths"):
        said(keep(**{name: None}), -1, b"null")
    said(keep(lengths=P), -1, b"lengths")
    assert keep(b=batch(sequences=0)) == 0


@pytest.mark.parametrize("wrong,word", [(dict(dtype=0), b"dtype"), (dict(dim=72), b"72"), (dict(dim=272), b"272"), (dict(dim=0), b"heads of 0"), (dict(page_size=24), b"24"),
                                        (dict(page_size=8), b"pages of 8"), (dict(page_size=2048), b"2048"), (dict(heads=0), b"heads"), (dict(pages=-1), b"pages"),
                                        (dict(keys=P + 8), b"16 bytes"), (dict(value_strides=(2048, 1024, 60)), b"16 bytes"), (dict(key_strides=(1 << 31, 1024, 64)), b"apart"),
                                        (dict(key_strides=(1 << 30, 64, 1 << 21)), b"apart"), (dict(keys=None), b"null"), (dict(dtype=5, key_scales=None), b"null")])
def test_every_entry_refuses_such_a_cache(L, wrong, word):
    c, b = cache(**wrong), batch()
    for rc in (L.vi_append_tokens(c, b, 1, P, 128, 64, P, 128, 64, 5, None, None, 0, 0, 1.0, None), L.vi_keep_drafts(c, b, P, 3, P, P + 16, None),
               L.vi_attend_cache(c, b, 1, P, 5, 4, 256, 64, None, 1.0, 64, 1, P, 256, 64, None, 0, None)):
        assert rc == -1 and word in L.vi_last_error(), (wrong, L.vi_last_error())


@pytest.mark.parametrize("wrong", [dict(sequences=-1), dict(width=-1), dict(stride=3), dict(width=1 << 30, stride=1 << 30), dict(starts=None), dict(lengths=None), dict(pages=None)])
def test_every_entry_refuses_such_a_batch(L, wrong):
    c, b = cache(), batch(**wrong)
    for rc in (L.vi_append_tokens(c, b, 1, P, 128, 64, P, 128, 64, 5, None, None, 0, 0, 1.0, None), L.vi_keep_drafts(c, b, P, 3, P, P + 16, None),
               L.vi_attend_cache(c, b, 1, P, 5, 4, 256, 64, None, 1.0, 64, 1, P, 256, 64, None, 0, None)):
        assert rc == -1


def test_plans_of_positions():
    from verinf_amd.prover import generation as gen
    plan = gen.rotary_plan(64, device="cpu")
    assert plan.rotated == 64 and plan.amplitude == 1.0
    for i, w in enumerate(plan.steps.tolist()):
        assert abs((w % (1 << 64)) / 2.0 ** 64 * 2 * math.pi - 10000.0 ** (-i / 32)) <= 2.0 ** -52
    slow = gen.rotary_plan(64, scaling=("linear", 4.0), device="cpu").steps
    assert (slow.double() * 4 - plan.steps.double()).abs().max() <= 2.0 ** 13            # doubles of 2^64 / 2 pi
    base = gen.rotary_plan(64, scaling=("base", 4.0), device="cpu").steps
    assert base[0] == plan.steps[0] and abs(int(base[31]) * 4 / int(plan.steps[31]) - 1) < 1e-12
    parts = gen.rotary_plan(64, scaling=("parts", 4.0, 4096), device="cpu")
    assert parts.steps[0] == plan.steps[0] and abs(int(parts.steps[31]) * 4 / int(plan.steps[31]) - 1) < 1e-12 and parts.amplitude == 0.1 * math.log(4.0) + 1
    for bad in (dict(dim=0), dict(dim=3), dict(dim=258), dict(dim=64, base=1.0), dict(dim=64, base=math.inf), dict(dim=64, scaling=("linear", 0.5)), dict(dim=64, scaling=("other", 2.0)),
                dict(dim=64, scaling=("parts", 2.0)), dict(dim=64, scaling=("linear", 2.0, 5)), dict(dim=64, scaling=("parts", 2.0, 4096, 3.0)), dict(dim=64, scaling=("parts", 2.0, 0)),
                dict(dim=64, scaling=("parts", 2.0, 4096, 5.0, 5.0))):
        with pytest.raises(RuntimeError):
            gen.rotary_plan(device="cpu", **bad)


def test_functions_refuse_tensors_that_are_not_on_the_gpu():
    from verinf_amd.prover import generation as gen
    x, i, p = torch.zeros(2, 3, 64), torch.zeros(2, dtype=torch.int64), gen.rotary_plan(64, device="cpu")
    for call in (lambda: gen.rotate_heads(x, i, p), lambda: gen.Cache(torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16), torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)),
                 lambda: gen.new_cache(4, 2, 16, 64, device="cpu"), lambda: gen.Batch(torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32)),
                 lambda: gen.verify_drafts(torch.zeros(2, 8), i, torch.zeros(2, dtype=torch.int32), None, torch.zeros(2, dtype=torch.float64), 1)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(RuntimeError, match="Tensor"):
        gen.rotate_heads([[1.0]], i, p)
    for call in (lambda: gen.append_tokens(None, x, x, None), lambda: gen.attend_cache(x, None, None), lambda: gen.keep_drafts(None, None, i, i)):
        with pytest.raises(RuntimeError, match="Cache"):
            call()
    with pytest.raises(RuntimeError, match="cache of"):
        gen.new_cache(4, 2, 16, 64, dtype=torch.float32, device="cpu")
