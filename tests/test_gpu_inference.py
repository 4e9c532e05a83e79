"""The forward pass's operators against plain implementations in 64 bits."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from verinf_amd.prover import inference as inf  # noqa: E402

P = (1 << 64) - (1 << 32) + 1
FLOATS = [torch.float32, torch.bfloat16, torch.float16]
# half a unit in the last place, relative, of one rounding to the type; the spacing of its smallest numbers
ROUND = {t: torch.finfo(t).eps / 2 for t in FLOATS}
LEAST = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}


def rows(t, pad, shift=0):
    """The matrix on the GPU with `pad` elements of something else behind each row, `shift` in front of the first."""
    m, k = t.shape
    flat = torch.full((shift + m * (k + pad) + 1,), 77, dtype=t.dtype, device="cuda")
    v = flat[shift:shift + m * (k + pad)].view(m, k + pad)[:, :k]
    v.copy_(t)
    return v


def eighths(m, k, gen):
    return torch.randint(-128, 128, (m, k), generator=gen, dtype=torch.int8)


# ---- quantize_rows ------------------------------------------------------------------------------------------------
def check_quantized(x):
    """x on the GPU; the definition's operations one by one in 32 bits, which numpy rounds as the definition says"""
    q, s = inf.quantize_rows(x)
    assert q.dtype == torch.int8 and s.dtype == torch.float32 and q.shape == x.shape and s.shape == x.shape[:1]
    f = x.float().cpu().numpy()
    top = np.abs(f).max(axis=1, initial=0)
    with np.errstate(all="ignore"):
        fine = np.isfinite(f).all(axis=1) & (top >= np.float32(127) * np.float32(2.0 ** -126))
        step = np.where(fine, np.float32(127) / top, np.float32(0)).astype(np.float32)
        want_q = np.where(fine[:, None], np.rint(f * step[:, None]), 0).astype(np.int8)
        want_s = np.where(fine, top / np.float32(127), np.where(np.isfinite(f).all(axis=1), np.float32(0), np.float32(np.nan)))
    assert np.array_equal(q.cpu().numpy(), want_q)
    assert np.array_equal(s.cpu().numpy(), want_s.astype(np.float32), equal_nan=True)
    # what the integers are for: half a step off at most, three roundings of 2^-24 of 127 steps beside it
    d, s64 = q.cpu().double().numpy() * s.cpu().double().numpy()[:, None], s.cpu().double().numpy()[:, None]
    assert (np.abs(d - f.astype(np.float64)) <= s64 * (0.5 + 127 * 2.0 ** -22))[fine].all()


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("m,k,pad,shift", [(1, 1, 0, 0), (3, 2, 1, 1), (2, 7, 0, 1), (5, 8, 0, 0), (4, 63, 3, 0), (1, 64, 0, 0), (7, 127, 1, 3), (3, 255, 0, 0),
                                           (2, 256, 0, 0), (9, 1000, 0, 0), (2, 2047, 5, 1), (3, 2048, 0, 0), (1, 2049, 0, 0), (5, 4096, 16, 0),
                                           (2, 8191, 0, 0), (4, 11008, 0, 0), (3, 16384, 0, 0), (2, 16385, 3, 0), (1, 40001, 0, 1), (2, 131071, 0, 0),
                                           (1000, 96, 0, 0), (70001, 5, 0, 0)])
def test_rows_are_quantized_as_defined(dtype, m, k, pad, shift):
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(m * 7 + k)) * 3
    check_quantized(rows(x.to(dtype), pad, shift))


@pytest.mark.parametrize("dtype", FLOATS)
def test_rows_that_are_hard_to_quantize(dtype):
    least, most = torch.finfo(dtype).tiny, torch.finfo(dtype).max
    x = torch.randn(16, 300, generator=torch.Generator().manual_seed(1)).to(dtype)
    x[0] = 0
    x[1] = -0.0
    x[2] = 0
    x[2, 299] = least                          # a single entry, of the smallest normal size
    x[3, 17] = math.inf
    x[4, 299] = -math.inf
    x[5, 0] = math.nan
    x[6] = most
    x[7] = -most
    x[8] *= 1e-30 if dtype != torch.float16 else 1e-4
    x[9] = torch.arange(300) % 255 - 127       # every integer, by halves next
    x[10] = (torch.arange(300) % 509 - 254) / 2
    x[10, 0] = 127
    x[11] = 0
    x[11, 5] = least / 2                       # below: no normal number
    x[12] = 2.0 ** -118 if dtype != torch.float16 else 2.0 ** -24
    x[13] = 2.0 ** -121 if dtype != torch.float16 else 0
    check_quantized(x.cuda())


def test_quantize_empty():
    for m, k in ((0, 5), (3, 0), (0, 0)):
        q, s = inf.quantize_rows(torch.empty((m, k), device="cuda"))
        assert q.shape == (m, k) and s.shape == (m,) and (s == 0).all()


# ---- int8_matmul --------------------------------------------------------------------------------------------------
SHAPES = [(1, 1, 1, 0, 0), (1, 16, 1, 0, 0), (1, 64, 64, 0, 0), (2, 5, 3, 0, 0), (3, 0, 4, 0, 0), (1, 4096, 500, 0, 0), (1, 1000, 37, 3, 1), (4, 127, 16, 1, 1), (7, 256, 129, 0, 0),
          (8, 2048, 96, 16, 0), (15, 63, 17, 0, 0), (16, 64, 16, 0, 0), (17, 65, 255, 0, 0), (31, 300, 64, 4, 0), (32, 512, 40, 0, 0), (33, 129, 130, 0, 0), (48, 1411, 333, 13, 0),
          (63, 4096, 257, 0, 0), (64, 1024, 512, 0, 0), (65, 96, 31, 0, 0), (100, 760, 1070, 0, 0), (127, 17, 128, 7, 0), (128, 128, 128, 0, 0), (129, 1031, 65, 0, 0),
          (200, 640, 384, 32, 0), (255, 64, 257, 0, 0), (256, 1088, 256, 0, 0), (257, 192, 513, 0, 16), (400, 3000, 300, 0, 0), (1000, 511, 700, 1, 1), (1000, 576, 1030, 0, 0),
          (2050, 80, 90, 0, 0), (30, 16385, 70, 0, 0), (2000, 320, 2300, 0, 0)]


def operands(m, k, n, pad, shift, weights=1):
    gen = torch.Generator().manual_seed(m * 131 + k * 17 + n)
    a = eighths(m, k, gen)
    return a, [eighths(n, k, gen) for _ in range(weights)], [rows(a, pad, shift)] + [None] * weights, gen


def exact(a, b):
    """whole numbers below 2^53: exact in any order"""
    return (a.cuda().double() @ b.cuda().double().T).cpu()


@pytest.mark.parametrize("m,k,n,pad,shift", SHAPES)
def test_matmul_sums_are_exact(m, k, n, pad, shift):
    a, (b,), _, _ = operands(m, k, n, pad, shift)
    ga, gb = rows(a, pad, shift), rows(b, pad, shift)
    want = exact(a, b).to(torch.int64)
    assert torch.equal(inf.int8_matmul(ga, gb).cpu(), want.to(torch.int32))
    field = inf.int8_matmul(ga, gb, dtype=torch.uint64).cpu().numpy()
    s = want.numpy()
    assert np.array_equal(field, np.where(s < 0, s.astype(np.uint64) + np.uint64(P), s.astype(np.uint64)))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("m,k,n,pad,shift", SHAPES)
def test_matmul_scaled(dtype, m, k, n, pad, shift):
    a, (b,), _, gen = operands(m, k, n, pad, shift)
    sa = torch.rand((m,), generator=gen) * 0.1 + 0.001
    sb = torch.rand((n,), generator=gen) * 0.01 + 0.0001
    for bias in (None, torch.randn((n,), generator=gen)):
        out = inf.int8_matmul(rows(a, pad, shift), rows(b, pad, shift), sa.cuda(), sb.cuda(), bias=None if bias is None else bias.cuda(), dtype=dtype)
        assert out.dtype == dtype and out.shape == (m, n)
        s = exact(a, b) * sa.double()[:, None] * sb.double()
        want = s if bias is None else s + bias.double()
        # the sum's conversion, two products and an addition in 32 bits, then one rounding to the type
        most = want.abs() * (ROUND[dtype] * 1.0001) + 2.0 ** -24 * 4 * (s.abs() + (0 if bias is None else bias.double().abs())) + LEAST[dtype]
        assert ((out.cpu().double() - want).abs() <= most).all()


def test_matmul_of_the_largest_sums():
    """the longest inner dimension, all products of the same sign: 2^31 - 2^14, and its opposite next to it"""
    k = inf.MAX_K
    for m, n in ((1, 3), (40, 70), (130, 140)):
        a = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
        b = torch.full((n, k), -128, dtype=torch.int8, device="cuda")
        b[n // 2] = 127
        got = inf.int8_matmul(a, b).cpu()
        assert (got[:, n // 2] == -128 * 127 * k).all()
        got[:, n // 2] = 128 * 128 * k
        assert (got == 128 * 128 * k).all()


def test_matmul_is_the_field_product_of_the_lifted_operands():
    from verinf_amd.prover import cuda_primitives as cp
    gen = torch.Generator().manual_seed(5)
    a, b = eighths(100, 500, gen).cuda(), eighths(60, 500, gen).cuda()

    def lift(t):
        v = t.to(torch.int64)
        return torch.where(v < 0, v - ((1 << 32) - 1), v).contiguous().view(torch.uint64)

    assert torch.equal(inf.int8_matmul(a, b, dtype=torch.uint64).view(torch.int64), cp.gl_matmul(lift(a), lift(b.T)).view(torch.int64))


def test_matmul_rows_more_than_4_gib_apart():
    ld = (1 << 32) + 64
    flat = torch.empty((2 * ld + 512,), dtype=torch.int8, device="cuda")
    gen = torch.Generator().manual_seed(6)
    for k in (200, 256):
        a, b = flat[:2 * ld].view(2, ld)[:, :k], eighths(300, k, gen)
        flat_b = flat[1024:1024 + 2 * ld - 2048].as_strided((2, k), (ld, 1))
        a.copy_(eighths(2, k, gen))
        flat_b.copy_(eighths(2, k, gen))
        assert torch.equal(inf.int8_matmul(a, b.cuda()).cpu(), exact(a, b).to(torch.int32))
        assert torch.equal(inf.int8_matmul(b.cuda(), flat_b).cpu(), exact(b, flat_b).to(torch.int32))
        assert torch.equal(inf.int8_matmul(flat_b, a).cpu(), exact(flat_b, a).to(torch.int32))


def test_matmul_of_more_than_2_32_outputs():
    m, n, k = 66000, 65552, 32
    gen = torch.Generator().manual_seed(7)
    a, b = eighths(m, k, gen).cuda(), eighths(n, k, gen).cuda()
    one_a, one_b = torch.ones((m,), device="cuda"), torch.full((n,), 2.0 ** -6, device="cuda")
    out = inf.int8_matmul(a, b, one_a, one_b, dtype=torch.float16)
    for at in (0, 255, 32768, 65520, m - 1):
        want = exact(a[at:at + 1], b) * 2.0 ** -6                                 # below 2^13: a single rounding
        assert torch.equal(out[at:at + 1].cpu(), want.to(torch.float16))


def test_scales_that_are_no_numbers_and_outputs_that_overflow():
    a, b = torch.full((3, 64), 100, dtype=torch.int8, device="cuda"), torch.full((5, 64), 100, dtype=torch.int8, device="cuda")
    sa, sb = torch.tensor([1.0, math.nan, 0.0], device="cuda"), torch.tensor([1.0, 1e-3, 0.0, 2.0, math.inf], device="cuda")
    out = inf.int8_matmul(a, b, sa, sb, dtype=torch.float16).cpu()
    assert out[0].tolist()[:4] == [math.inf, 640.0, 0.0, math.inf] and out[0, 4] == math.inf
    assert out[1].isnan().all() and out[2, :4].tolist() == [0.0] * 4 and out[2, 4].isnan()


# ---- int8_gated ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("m,k,n,pad,shift", SHAPES)
def test_gated(act, dtype, m, k, n, pad, shift):
    a, (g, u), _, gen = operands(m, k, n, pad, shift, 2)
    sa = torch.rand((m,), generator=gen) * 0.02 + 0.001
    sg, su = ((torch.rand((n,), generator=gen) * 0.01 + 0.0001) * 40 / math.sqrt(k + 1) for _ in range(2))
    out = inf.int8_gated(rows(a, pad, shift), rows(g, pad, shift), rows(u, pad, shift), sa.cuda(), sg.cuda(), su.cuda(), activation=act, dtype=dtype)
    assert out.dtype == dtype and out.shape == (m, n)
    G, U = exact(a, g) * sa.double()[:, None] * sg.double(), exact(a, u) * sa.double()[:, None] * su.double()
    acted = G * torch.sigmoid(G) if act == "silu" else G * torch.special.ndtr(G)
    want = acted * U
    # G and U: three roundings of 2^-24 each; e^-G with an argument rounded to 2^-24 of its size and two units of the exponential and
    # the reciprocal; the derivative of either activation is below 1.2 in size and silu's relative one below 1 + |G|
    rel = 2.0 ** -24 * (8 + 8 * G.abs())
    err = U.abs() * (acted.abs() * rel + (0 if act == "silu" else G.abs() * 2.0 ** -22))
    most = want.abs() * (ROUND[dtype] * 1.0001) + err + LEAST[dtype]
    assert ((out.cpu().double() - want).abs() <= most).all()


def test_gated_far_out():
    """activations of very large and very small numbers, no NaN where the mathematics has none"""
    a = torch.full((1, 32), 1, dtype=torch.int8, device="cuda")
    g = torch.stack([torch.full((32,), v, dtype=torch.int8) for v in (127, -127, 0, 1, -1)]).cuda()
    one = torch.ones((5,), device="cuda")
    for act in ("silu", "gelu"):
        out = inf.int8_gated(a, g, torch.ones_like(g), torch.ones((1,), device="cuda"), one, one / 32, activation=act, dtype=torch.float32).cpu()[0]
        assert out[0] == 127 * 32 and abs(out[1]) == 0 and abs(out[2]) == 0 and abs(out[3] - 32) < 1e-4 and abs(out[4]) < 1e-10


# ---- token_logprobs -----------------------------------------------------------------------------------------------
def want_logprobs(x, tokens, top, temperature):
    """x: float64 array with NaN, infinities, -inf as they come"""
    m, v = x.shape
    out = [np.zeros(m), np.zeros(m), np.zeros((m, top)), np.zeros((m, top), dtype=np.int64)]
    for i in range(m):
        r = x[i]
        poisoned = np.isnan(r).any() or np.isposinf(r).any()
        z = r / temperature
        with np.errstate(all="ignore"):
            if poisoned:
                lp, h = np.full(v, np.nan), np.nan
            elif np.isneginf(r).all():
                lp, h = r.copy(), 0.0
            else:
                d = z - z.max()
                lp = d - np.log(np.exp(d).sum())
                p = np.exp(lp)
                h = -(p[p > 0] * lp[p > 0]).sum()
        t = tokens[i]
        out[0][i] = 0.0 if t == -1 else lp[t] if 0 <= t < v else np.nan
        out[1][i] = h
        order = np.lexsort((np.arange(v), np.where(np.isnan(r), -np.inf, -np.where(np.isnan(r), 0, r)), ~np.isnan(r)))[:top]
        out[2][i], out[3][i] = lp[order], order
    return out


def check_logprobs(x, tokens, top, temperature=1.0):
    """x on the GPU.  A logit's distance to the largest is rounded twice (2^-23 of it), e^d with it; up to 128 terms are added one
    after another and their sums pairwise: 2^-24 * 160 of Z, so of log Z, and as much again of each exponential's own two units and the logarithm."""
    got = inf.token_logprobs(x, tokens, top=top, temperature=temperature)
    f = x.double().cpu().numpy()
    lp, h, tops, index = want_logprobs(f, tokens.cpu().numpy(), top, temperature)
    assert got[3].dtype == torch.int64 and np.array_equal(got[3].cpu().numpy(), index)
    slack = 2.0 ** -24 * 200

    def near(t, want, most):
        t = t.cpu().double().numpy()
        assert t.shape == want.shape
        same = (t == want) | (np.isnan(t) & np.isnan(want))
        with np.errstate(all="ignore"):
            assert (same | (np.abs(t - want) <= most)).all(), np.nanmax(np.abs(t - want) - most)

    with np.errstate(all="ignore"):
        near(got[0], lp, slack + 2.0 ** -21 * np.abs(lp))
        near(got[2], tops, slack + 2.0 ** -21 * np.abs(tops))
        # d weighted with e^d / Z: its size is below H + log v
        near(got[1], h, slack * (2 + 2 * np.log(x.shape[1])))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("m,v,pad,shift,top,temperature", [
    (1, 1, 0, 0, 1, 1.0), (3, 2, 0, 1, 2, 0.5), (2, 7, 1, 0, 0, 1.0), (4, 63, 0, 0, 63, 1.0), (5, 64, 0, 0, 64, 1.3), (2, 100, 3, 1, 20, 1.0), (3, 1000, 0, 0, 5, 0.7),
    (2, 1023, 0, 0, 1, 1.0), (1, 1024, 0, 0, 64, 1.0), (1, 1025, 0, 0, 64, 1.0), (2, 2048, 0, 0, 33, 1.0), (2, 2049, 1, 0, 33, 1.0), (9, 4097, 0, 0, 8, 1.0),
    (1, 32000, 0, 0, 20, 1.0), (20, 32000, 0, 0, 5, 1.0), (3, 50257, 7, 1, 8, 0.7), (1, 160001, 0, 0, 64, 1.0), (300, 5000, 0, 0, 3, 1.0), (700, 1030, 2, 0, 10, 2.0),
    (1100, 300, 0, 0, 4, 1.0), (2100, 2500, 0, 0, 2, 1.0), (520, 9000, 0, 0, 64, 1.0), (130, 33000, 0, 0, 17, 1.0)])
def test_logprobs(dtype, m, v, pad, shift, top, temperature):
    gen = torch.Generator().manual_seed(m + v)
    x = torch.randn(m, v, generator=gen) * 4
    tokens = torch.randint(0, v, (m,), generator=gen)
    tokens[::3] = x[::3].argmax(1)
    check_logprobs(rows(x.to(dtype), pad, shift), tokens.cuda(), top, temperature)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("v", [70, 1500, 9001, 40000])
@pytest.mark.parametrize("top", [0, 1, 20, 64])
def test_logprobs_of_masks_ties_and_what_is_no_number(dtype, v, top):
    gen = torch.Generator().manual_seed(v)
    lowest = torch.finfo(dtype).min
    x = (torch.randn(22, v, generator=gen) * 3).to(dtype)
    some = torch.rand(v, generator=gen) < 0.99
    x[0] = -math.inf                           # a mask that leaves nothing
    x[1] = lowest                              # the same with the type's lowest value
    x[2, some] = -math.inf
    x[3, some] = lowest
    x[4] = -math.inf
    x[4, v - 1] = 2.0                          # one entry left
    x[5] = lowest
    x[5, v // 2] = -3.0
    x[6] = 1.5                                 # all equal
    x[7] = (torch.arange(v) % 3).to(dtype)     # three values
    x[8] = (torch.arange(v) * (60.0 / v)).to(dtype)                 # rising, with ties in short types
    x[9] = (-torch.arange(v) * (60.0 / v)).to(dtype)
    x[10, 5] = math.nan
    x[11] = math.nan
    x[12, v - 1] = math.inf
    x[13, [3, 60]] = math.inf
    x[13, 61] = math.nan
    x[14] = -math.inf
    x[14, 9] = math.nan
    x[15] = torch.where(torch.arange(v) % 2 == 0, 0.0, -0.0).to(dtype)      # equal too
    x[16, 7] = 60.0                            # nearly certain
    x[17] = torch.finfo(dtype).max
    x[18, : v // 2] = torch.finfo(dtype).max
    x[19, v - 30:] = 5.0                       # ties at the end
    x[20, :40] = -math.inf
    x[20, 40:] = lowest
    tokens = torch.randint(0, v, (22,), generator=gen)
    tokens[2], tokens[4], tokens[16] = 0, v - 1, 7
    tokens[17], tokens[19], tokens[21] = -1, v, -2
    check_logprobs(x.cuda(), tokens.cuda(), top)


def test_logprobs_empty():
    got = inf.token_logprobs(torch.empty((0, 50), device="cuda"), torch.empty((0,), dtype=torch.int64, device="cuda"), top=3)
    assert [tuple(t.shape) for t in got] == [(0,), (0,), (0, 3), (0, 3)]


def test_logprobs_rows_more_than_4_gib_apart():
    ld = (1 << 31) + 5
    flat = torch.empty((2 * ld,), dtype=torch.bfloat16, device="cuda")
    x = flat.view(2, ld)[:, :3000]
    x.copy_(torch.randn(2, 3000, generator=torch.Generator().manual_seed(9)) * 4)
    check_logprobs(x, torch.tensor([7, 2999], device="cuda"), 6)
    q, s = inf.quantize_rows(x)
    q1, s1 = inf.quantize_rows(x.contiguous())
    assert torch.equal(q, q1) and torch.equal(s, s1)


# ---- together -----------------------------------------------------------------------------------------------------
def calls(seed):
    """Every operator, in forms with and without scratch, as one list of outputs."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((9, 2000), generator=gen, device="cuda")
    q, s = inf.quantize_rows(x)
    w, ws = inf.quantize_rows(torch.randn((300, 2000), generator=gen, device="cuda"))
    u, us = inf.quantize_rows(torch.randn((300, 2000), generator=gen, device="cuda"))
    h = inf.int8_gated(q, w, u, s, ws * 0.02, us)
    logits = inf.int8_matmul(q, w, s, ws, dtype=torch.float32)
    big = torch.randn((3, 70000), generator=gen, device="cuda")
    return [q, s, h, logits, inf.int8_matmul(q, w), *inf.token_logprobs(logits, torch.arange(9, device="cuda"), top=4),
            *inf.token_logprobs(big, torch.arange(3, device="cuda"), top=7)]


def test_the_current_stream_is_the_one_used():
    want = calls(3)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = calls(3)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_repeated_calls_give_the_same_bits():
    want = calls(4)
    for _ in range(3):
        for a, b in zip(calls(4), want):
            assert torch.equal(a, b)


def test_calls_captured_into_a_graph():
    q = torch.randint(-127, 128, (5, 4000), dtype=torch.int8, device="cuda")
    w = torch.randint(-127, 128, (400, 4000), dtype=torch.int8, device="cuda")
    s, ws = torch.rand((5,), device="cuda"), torch.rand((400,), device="cuda") * 1e-4
    big = torch.randn((2, 70000), device="cuda")
    t = torch.tensor([1, 69999], device="cuda")

    def step():
        h = inf.int8_gated(q, w, w, s, ws, ws)
        hq, hs = inf.quantize_rows(h)
        return [h, hq, hs, inf.int8_matmul(q, w, s, ws), *inf.token_logprobs(big, t, top=9)]

    want = step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for turn in range(4):
        q.random_(-127, 128, generator=torch.Generator(device="cuda").manual_seed(turn))
        big.normal_(generator=torch.Generator(device="cuda").manual_seed(turn))
        want = step()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_refusals():
    x = torch.zeros((4, 64), device="cuda")
    q, w = x.to(torch.int8), torch.zeros((6, 64), dtype=torch.int8, device="cuda")
    s, ws, t = torch.ones((4,), device="cuda"), torch.ones((6,), device="cuda"), torch.zeros((4,), dtype=torch.int64, device="cuda")
    bad = [lambda: inf.quantize_rows(x.double()), lambda: inf.quantize_rows(x[0]), lambda: inf.quantize_rows(x.T), lambda: inf.quantize_rows(x[:1].expand(4, 64)),
           lambda: inf.quantize_rows(x.clone().requires_grad_()), lambda: inf.quantize_rows(x[:, ::2]),
           lambda: inf.int8_matmul(x, w), lambda: inf.int8_matmul(q, w[:, :63]), lambda: inf.int8_matmul(q, w, s), lambda: inf.int8_matmul(q, w, s, s),
           lambda: inf.int8_matmul(q, w, s, ws, dtype=torch.int32), lambda: inf.int8_matmul(q, w, dtype=torch.float32), lambda: inf.int8_matmul(q, w, bias=ws),
           lambda: inf.int8_matmul(q, w, s, ws, bias=s), lambda: inf.int8_matmul(q, w, s.double(), ws), lambda: inf.int8_matmul(q, w, s[:1].expand(4), ws),
           lambda: inf.int8_matmul(q, w.T), lambda: inf.int8_matmul(q, w.cpu()),
           lambda: inf.int8_matmul(torch.zeros((1, 131072), dtype=torch.int8, device="cuda"), torch.zeros((1, 131072), dtype=torch.int8, device="cuda")),
           lambda: inf.int8_gated(q, w, w[:5], s, ws, ws), lambda: inf.int8_gated(q, w, w, s, ws, ws, activation="relu"),
           lambda: inf.int8_gated(q, w, w, s, ws, ws, dtype=torch.int32), lambda: inf.int8_gated(q, w, w, s, ws, s), lambda: inf.int8_gated(q, w, w[:, :60], s, ws, ws),
           lambda: inf.token_logprobs(x, t[:3]), lambda: inf.token_logprobs(x, t.int()), lambda: inf.token_logprobs(x, t, top=65), lambda: inf.token_logprobs(x, t, top=-1),
           lambda: inf.token_logprobs(x[:, :8], t, top=9), lambda: inf.token_logprobs(x, t, temperature=0.0), lambda: inf.token_logprobs(x, t, temperature=math.nan),
           lambda: inf.token_logprobs(x.to(torch.int32), t), lambda: inf.token_logprobs(x[:, :0], t), lambda: inf.token_logprobs(x.clone().requires_grad_(), t)]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was not refused")


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("m,k,pad,shift", [(1024, 128, 0, 0), (2000, 250, 0, 0), (1500, 256, 3, 1), (2048, 257, 0, 0), (3001, 333, 0, 0), (2500, 1030, 6, 0),
                                           (2049, 2048, 0, 0), (2048, 2049, 0, 0), (1200, 9, 0, 0), (40, 12300, 0, 0)])
def test_many_short_rows_are_quantized_as_defined(dtype, m, k, pad, shift):
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(m + 3 * k)) * 5
    x[m // 2] = 0
    x[m - 1, k - 1] = math.nan
    x[m - 2, 0] = -math.inf
    check_quantized(rows(x.to(dtype), pad, shift))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("m,v,pad,shift,top", [(2, 32768, 0, 0, 9), (2, 32769, 1, 0, 9), (2, 65536, 0, 0, 64), (1, 65537, 0, 1, 7), (256, 4096, 0, 0, 2), (257, 4100, 0, 0, 2), (520, 70000, 0, 0, 5),
                                               (1030, 16390, 0, 0, 64), (3, 131072, 8, 0, 33), (1025, 1024, 0, 0, 1)])
def test_logprobs_where_rows_are_cut_otherwise(dtype, m, v, pad, shift, top):
    gen = torch.Generator(device="cuda").manual_seed(m + v)
    flat = (torch.randn(m, v + pad + shift, generator=gen, device="cuda") * 4).to(dtype)
    flat[m // 2, : v // 3] = -math.inf
    x = flat[:, shift:shift + v]
    check_logprobs(x, torch.randint(0, v, (m,), generator=gen, device="cuda"), top)


def test_more_rows_than_a_launch_has_workgroups_for():
    # 2^23 rows at a time: the last ones are as they would be alone
    m, some = (1 << 23) + 300, 1000
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((m, 3), generator=gen, device="cuda").to(torch.bfloat16)
    t = torch.randint(0, 3, (m,), generator=gen, device="cuda")
    got, lp = inf.quantize_rows(x), inf.token_logprobs(x, t, top=2)
    for part in (slice(0, some), slice(m - some, m)):
        check_quantized(x[part])
        check_logprobs(x[part], t[part], 2)
        for a, b in zip(got + lp, inf.quantize_rows(x[part]) + inf.token_logprobs(x[part], t[part], top=2)):
            assert torch.equal(a[part], b)


@pytest.mark.parametrize("m,k,n", [(1500, 4097, 2500), (2000, 1634, 4096), (700, 2111, 9000), (1241, 8200, 1632)])
def test_unaligned_rows_that_are_copied_first(m, k, n):
    # the same integers at 16-byte boundaries are read in place; sums are exact either way
    gen = torch.Generator().manual_seed(k)
    a, b, c = eighths(m, k, gen), eighths(n, k, gen), eighths(n, k, gen)
    sa, sb = torch.rand(m, generator=gen).cuda(), torch.rand(n, generator=gen).cuda() * 1e-4
    even = -k % 16
    got = inf.int8_matmul(rows(a, 1), rows(b, 3))
    assert torch.equal(got, inf.int8_matmul(rows(a, even), rows(b, even)))
    some = torch.arange(0, m, 97)
    assert torch.equal(got[some.cuda()].cpu(), (a[some].double() @ b.double().T).to(torch.int32))
    assert torch.equal(inf.int8_gated(rows(a, 0, 1), rows(b, 3), rows(c, 0, 2), sa, sb, sb), inf.int8_gated(rows(a, even), rows(b, even), rows(c, even), sa, sb, sb))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("v", [70, 1000, 3000, 9001, 32000, 70001, 200003])
@pytest.mark.parametrize("top", [1, 3, 20, 64])
def test_logprobs_of_negative_zeros(dtype, v, top):
    """-0.0 is equal to 0.0, and goes with it by the lowest index"""
    gen = torch.Generator().manual_seed(v)
    x = (-torch.randn(8, v, generator=gen).abs() - 1).to(dtype)
    x[0] = -0.0
    x[1] = -0.0
    x[1, v // 2] = 5.0                         # one positive entry
    x[2, :16] = -0.0                           # in front of 0.0
    x[2, 64:70] = 0.0
    x[3, 3::64] = -0.0                         # far apart, among negative ones
    x[4] = -0.0
    x[4, v - 1] = 0.0
    x[5] = -math.inf
    x[5, 5:60:7] = -0.0
    x[6, v - 20:] = -0.0
    x[7] = (torch.randn(v, generator=gen).abs() * 1e-9).neg().to(dtype)     # float16: underflows to -0.0
    check_logprobs(x.cuda(), torch.tensor([0, 1, 2, 3, 4, 5, v - 1, 7], device="cuda"), top)
    many = x[:1].expand(300, v).contiguous().cuda()                         # one workgroup of 256 threads a row, or slices of it
    check_logprobs(many, torch.arange(300, device="cuda") % v, top)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("m,n", [(1, 256), (20, 256), (33, 256), (200, 256), (200, 253)])
def test_gelu_of_negative_numbers(dtype, m, n):
    """x Phi(x) far below zero has all its digits: G = 0, -0.1, -0.2 ... -12.8 in the first row, U = 0.1."""
    g = torch.arange(n, dtype=torch.int64).sub(255).div(2, rounding_mode="floor").to(torch.int8)[:, None].cuda()
    one = torch.ones((m, 1), dtype=torch.int8, device="cuda")
    sa = 0.1 / torch.arange(1, m + 1, device="cuda").float()
    sn = torch.ones((n,), device="cuda")
    out = inf.int8_gated(one, g, torch.ones_like(g), sa, sn, sn, activation="gelu", dtype=dtype)
    G = (g[:, 0].float()[None, :] * sa[:, None]).double().cpu()                       # as it is in 32 bits
    want = 0.5 * G * torch.special.erfc(-G * 0.5 ** 0.5) * sa.double().cpu()[:, None]
    # the argument's rounding and that of the constant: 1.5 units of 2^-24, times the 2 t^2 = x^2 by which erfc grows; 16 units of 2^-23 of erfc itself; four products
    rel = 2.0 ** -24 * (1.5 * (1 + G ** 2) + 32 + 4)
    most = want.abs() * (rel + ROUND[dtype] * 1.0001) + LEAST[dtype]
    assert ((out.cpu().double() - want).abs() <= most).all()


# m, k, n, rows at 16-byte boundaries: sizes that between them take every tile, plain and gated (which the CPU build asserts of them), with whole and
# ragged tiles and inner dimensions; unaligned ones read through registers or copied, in one slice and in several
LARGE = [(5000, 448, 3000, True), (3001, 500, 5003, True), (8191, 300, 2000, True), (1025, 4100, 11009, True), (2500, 1411, 4099, True), (2000, 4096, 4099, True),
         (1025, 4096, 8000, True), (4095, 1000, 2000, True), (2049, 4096, 3000, True), (2049, 1411, 1000, True), (4095, 400, 3000, True), (300, 4096, 400, True),
         (1537, 130, 8000, False), (2060, 257, 3000, False), (130, 8200, 3000, False), (4100, 1411, 400, False), (1030, 8200, 400, False)]
LARGE_GATED = [(4095, 1000, 2000, True), (2049, 1411, 3000, True), (4100, 2048, 1500, True), (777, 4100, 5003, True), (2049, 4096, 2000, True), (1300, 4096, 2305, True),
               (2049, 4100, 1500, True), (1300, 1000, 2305, True), (2049, 1000, 1500, True), (300, 4096, 200, True),
               (1000, 257, 8000, False), (333, 1411, 11008, False), (130, 8200, 3000, False), (1537, 1024, 2000, False), (200, 8200, 1030, False)]


def large_operands(m, k, n, aligned, weights):
    gen = torch.Generator(device="cuda").manual_seed(m * 131 + k * 17 + n)
    pads = [-k % 16] * 3 if aligned else [1 + (-k % 16), 3, 5]
    mats = [rows(torch.randint(-128, 128, (r, k), generator=gen, device="cuda", dtype=torch.int8), pad, 0 if aligned else 1) for r, pad in zip([m] + [n] * weights, pads)]
    # rows of every tile, the first and the last among them; sums of them in 64 bits
    some = torch.unique(torch.cat([torch.arange(0, m, max(1, m // 61)), torch.tensor([0, m - 1])])).cuda()
    return mats, [mats[0][some].double() @ w.double().T for w in mats[1:]], some, gen


@pytest.mark.parametrize("m,k,n,aligned", LARGE)
def test_matmul_of_large_tiles(m, k, n, aligned):
    (a, b), (S,), some, gen = large_operands(m, k, n, aligned, 1)
    assert torch.equal(inf.int8_matmul(a, b)[some], S.to(torch.int32))
    s = S.to(torch.int64)
    assert torch.equal(inf.int8_matmul(a, b, dtype=torch.uint64).view(torch.int64)[some], torch.where(s < 0, s - ((1 << 32) - 1), s))
    sa = torch.rand((m,), generator=gen, device="cuda") * 0.1 + 0.001
    sb = torch.rand((n,), generator=gen, device="cuda") * 0.01 + 0.0001
    s = S * sa.double()[some, None] * sb.double()
    for dtype in FLOATS:
        for bias in (None, torch.randn((n,), generator=gen, device="cuda")):
            out = inf.int8_matmul(a, b, sa, sb, bias=bias, dtype=dtype)
            want = s if bias is None else s + bias.double()
            # as of the small ones: the sum's conversion, two products and an addition in 32 bits, then one rounding to the type
            most = want.abs() * (ROUND[dtype] * 1.0001) + 2.0 ** -24 * 4 * (s.abs() + (0 if bias is None else bias.double().abs())) + LEAST[dtype]
            assert ((out[some].double() - want).abs() <= most).all()


@pytest.mark.parametrize("m,k,n,aligned", LARGE_GATED)
def test_gated_of_large_tiles(m, k, n, aligned):
    (a, g, u), (S, T), some, gen = large_operands(m, k, n, aligned, 2)
    sa = torch.rand((m,), generator=gen, device="cuda") * 0.02 + 0.001
    sg, su = ((torch.rand((n,), generator=gen, device="cuda") * 0.01 + 0.0001) * 40 / math.sqrt(k + 1) for _ in range(2))
    G, U = S * sa.double()[some, None] * sg.double(), T * sa.double()[some, None] * su.double()
    for act in ("silu", "gelu"):
        acted = G * torch.sigmoid(G) if act == "silu" else 0.5 * G * torch.special.erfc(-G * 0.5 ** 0.5)
        want = acted * U
        # three roundings of 2^-24 in G and in U; silu's argument, exponential and reciprocal; gelu's relative derivative is below 1 + x^2, and its
        # exponential has no results below 2^-126, which U multiplies
        rel = 2.0 ** -24 * (8 + 8 * G.abs() if act == "silu" else 16 + 8 * G ** 2)
        for dtype in FLOATS:
            out = inf.int8_gated(a, g, u, sa, sg, su, activation=act, dtype=dtype)
            most = want.abs() * (ROUND[dtype] * 1.0001 + rel) + LEAST[dtype] + 2.0 ** -126 * U.abs()
            assert ((out[some].double() - want).abs() <= most).all()


def test_tensors_with_a_tangent_are_refused():
    from torch.autograd import forward_ad
    x, s, ws = torch.randn((4, 64), device="cuda"), torch.ones((4,), device="cuda"), torch.ones((6,), device="cuda")
    q, w, t = torch.zeros((4, 64), dtype=torch.int8, device="cuda"), torch.zeros((6, 64), dtype=torch.int8, device="cuda"), torch.zeros((4,), dtype=torch.int64, device="cuda")
    with forward_ad.dual_level():
        dx, ds, dws = (forward_ad.make_dual(v, torch.ones_like(v)) for v in (x, s, ws))
        for call in (lambda: inf.quantize_rows(dx), lambda: inf.token_logprobs(dx, t), lambda: inf.int8_matmul(q, w, ds, ws), lambda: inf.int8_matmul(q, w, s, ws, bias=dws),
                     lambda: inf.int8_gated(q, w, w, s, dws, ws), lambda: inf.quantize_rows(dx[:, :7])):
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):
                call()
        # others are taken there as anywhere
        assert torch.equal(inf.quantize_rows(x)[0], inf.quantize_rows(forward_ad.unpack_dual(dx).primal)[0])
        inf.int8_gated(q, w, w, s, ws, ws)
        inf.token_logprobs(x, t, top=2)
    for call in (inf.quantize_rows, lambda v: inf.token_logprobs(v, t)[0]):
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (x,), (x,))


def test_negative_views_are_refused():
    """the imaginary part of a conjugate is a view of numbers of the other sign"""
    x = torch.complex(torch.zeros((4, 1), device="cuda"), torch.randn((4, 1), device="cuda")).conj().imag
    assert x.is_neg()
    q, w, t = torch.ones((4, 8), dtype=torch.int8, device="cuda"), torch.ones((6, 8), dtype=torch.int8, device="cuda"), torch.zeros((4,), dtype=torch.int64, device="cuda")
    s, ws = torch.ones((4,), device="cuda"), torch.ones((6,), device="cuda")
    minus, minus_ws = torch._neg_view(s), torch._neg_view(ws)
    for call in (lambda: inf.quantize_rows(x), lambda: inf.token_logprobs(x, t), lambda: inf.int8_matmul(q, w, minus, ws), lambda: inf.int8_matmul(q, w, s, ws, bias=minus_ws),
                 lambda: inf.int8_gated(q, w, w, s, ws, minus_ws), lambda: inf.int8_matmul(torch._neg_view(q), w)):
        with pytest.raises(RuntimeError, match="resolve_neg"):
            call()
    got, scale = inf.quantize_rows(x.resolve_neg())
    assert torch.equal(got[:, 0].float().sign(), x[:, 0].sign()) and (scale > 0).all()


@pytest.mark.parametrize("m,n", [(1, 5), (70, 33), (300, 200)])
def test_products_of_no_inner_dimension(m, n):
    a, b = torch.empty((m, 0), dtype=torch.int8, device="cuda"), torch.empty((n, 0), dtype=torch.int8, device="cuda")
    one_m, one_n, bias = torch.ones((m,), device="cuda"), torch.ones((n,), device="cuda"), torch.arange(n, device="cuda").float()
    assert (inf.int8_matmul(a, b) == 0).all() and (inf.int8_matmul(a, b, dtype=torch.uint64).view(torch.int64) == 0).all()
    assert torch.equal(inf.int8_matmul(a, b, one_m, one_n, bias=bias, dtype=torch.float32), bias.expand(m, n))
    assert (inf.int8_gated(a, b, b, one_m, one_n, one_n, dtype=torch.float32) == 0).all()


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("v", [70, 3000, 9001, 70001])
def test_logprobs_of_logits_far_apart(dtype, v):
    """further than 32 bits hold, which a temperature brings together"""
    x = torch.full((3, v), torch.finfo(dtype).min, dtype=dtype)
    x[0, v // 2] = torch.finfo(dtype).max
    x[1, :5] = torch.finfo(dtype).max
    x[2, v // 2], x[2, 0] = torch.finfo(dtype).max, 1.0
    for temperature in (2.5, 50.0, 1000.0):
        check_logprobs(x.cuda(), torch.tensor([1, v - 1, 0], device="cuda"), 3, temperature)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("m,n", [(1, 128), (20, 128), (40, 128), (40, 125), (300, 256)])
def test_gated_products_that_overflow(act, m, n):
    """G of +inf stays, G of -inf gives 0, a NaN shows"""
    one = torch.ones((m, 16), dtype=torch.int8, device="cuda")
    g = torch.ones((n, 16), dtype=torch.int8, device="cuda")
    g[1::3] = -1
    sm, sn = torch.full((m,), 1e30, device="cuda"), torch.full((n,), 1e30, device="cuda")
    sn[2::3] = math.nan
    su = torch.full((n,), 1e-30, device="cuda")                        # U = 16
    for dtype in FLOATS:
        out = inf.int8_gated(one, g, torch.ones_like(g), sm, sn, su, activation=act, dtype=dtype)
        assert (out[:, 0::3] == math.inf).all() and (out[:, 1::3] == 0).all() and out[:, 2::3].isnan().all()
