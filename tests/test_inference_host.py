"""The forward pass's operators without a GPU: argument checks of the C entries and of the Python functions."""
import ctypes
import os

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def L():
    from verinf_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from verinf_amd.build import build
        build()
    return _lib.lib()


P1, P2, P3, P4 = (ctypes.c_void_p(0x1000 * i) for i in range(1, 5))       # never dereferenced


def test_entries_refuse_before_any_launch(L):
    def said(rc, code, word):
        assert rc == code and word in L.vi_last_error(), (rc, L.vi_last_error())

    said(L.vi_quantize_rows(3, P1, 1, 4, 4, P2, 4, P3, None), -1, b"dtype")
    said(L.vi_quantize_rows(0, P1, -1, 4, 4, P2, 4, P3, None), -1, b"rows")
    said(L.vi_quantize_rows(0, P1, 1, 4, 3, P2, 4, P3, None), -1, b"apart")
    said(L.vi_quantize_rows(0, P1, 1, 4, 4, P2, 3, P3, None), -1, b"apart")
    said(L.vi_quantize_rows(0, None, 1, 4, 4, P2, 4, P3, None), -1, b"null")
    said(L.vi_quantize_rows(0, P1, 1, 4, 4, P2, 4, None, None), -1, b"null")
    assert L.vi_quantize_rows(0, None, 0, 4, 4, None, 4, None, None) == 0

    def mm(m=2, k=4, n=3, lda=4, ldb=4, a=P1, b=P2, sa=P3, sb=P3, dtype=1, out=P4, ldo=3, ws=None, ws_bytes=0):
        return L.vi_int8_matmul(a, lda, b, ldb, m, k, n, sa, sb, None, dtype, out, ldo, ws, ws_bytes, None)

    said(mm(dtype=7), -1, b"dtype")
    said(mm(m=-1), -1, b"vi_int8_matmul")
    said(mm(k=131072, lda=131072, ldb=131072), -1, b"131071")
    said(mm(lda=3), -1, b"overlap")
    said(mm(ldb=3), -1, b"overlap")
    said(mm(ldo=2), -1, b"overlap")
    said(mm(a=None), -1, b"null")
    said(mm(out=None), -1, b"null")
    said(mm(sb=None), -1, b"scales")
    assert mm(m=0) == 0 and mm(n=0) == 0
    need = L.vi_int8_matmul_workspace_bytes(8, 65536, 128)
    assert need > 0
    said(mm(m=8, k=65536, n=128, lda=65536, ldb=65536, ldo=128, ws=P3, ws_bytes=need - 1), -3, b"workspace")
    assert L.vi_int8_matmul_workspace_bytes(0, 64, 64) == 0 and L.vi_int8_matmul_workspace_bytes(1, 131072, 64) == 0

    def gated(act=0, dtype=1, up=P3, us=P3, ldu=4):
        return L.vi_int8_gated(P1, 4, P2, 4, up, ldu, 2, 4, 3, P3, P3, us, act, dtype, P4, 3, None, 0, None)

    said(gated(act=2), -1, b"activation")
    said(gated(dtype=3), -1, b"dtype")
    said(gated(up=None), -1, b"null")
    said(gated(us=None), -1, b"scales")
    said(gated(ldu=3), -1, b"overlap")

    def lp(dtype=0, m=2, v=10, ld=10, t=1.0, top=3, x=P1, tok=P2, best=P3, ws=None, ws_bytes=0):
        return L.vi_token_logprobs(dtype, x, m, v, ld, tok, t, top, P3, P3, best, best, ws, ws_bytes, None)

    said(lp(dtype=3), -1, b"dtype")
    said(lp(v=0), -1, b"logits")
    said(lp(v=(1 << 24) + 1, ld=1 << 25), -1, b"logits")
    said(lp(ld=9), -1, b"apart")
    said(lp(top=65, v=100, ld=100), -1, b"largest")
    said(lp(top=11), -1, b"largest")
    said(lp(top=-1), -1, b"largest")
    for t in (0.0, -1.0, float("nan"), float("inf")):
        said(lp(t=t), -1, b"temperature")
    said(lp(x=None), -1, b"null")
    said(lp(tok=None), -1, b"null")
    said(lp(best=None), -1, b"null")
    said(lp(v=100000, ld=100000), -3, b"workspace")
    assert lp(m=0) == 0
    assert L.vi_token_logprobs_workspace_bytes(0, 1, 100000, 3) > 0 and L.vi_token_logprobs_workspace_bytes(0, 1, 100000, 65) == 0


def test_functions_refuse_tensors_that_are_not_on_the_gpu():
    from verinf_amd.prover import inference as inf
    x, q, s = torch.zeros(2, 4), torch.zeros(2, 4, dtype=torch.int8), torch.zeros(2)
    with pytest.raises(RuntimeError, match="CUDA"):
        inf.quantize_rows(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        inf.int8_matmul(q, q)
    with pytest.raises(RuntimeError, match="CUDA"):
        inf.int8_gated(q, q, q, s, s, s)
    with pytest.raises(RuntimeError, match="CUDA"):
        inf.token_logprobs(x, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="Tensor"):
        inf.quantize_rows([[1.0]])
