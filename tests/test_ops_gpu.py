"""GPU: the operators of ops.py against plain implementations in 64 bits, at the sizes, strides and values where they can go wrong.

Tolerances.  A rounding is off by at most half a step: 2^-24 of the value in fp32, 2^-8 in bf16, 2^-4 in e4m3 (2^-10 below its smallest normal
number, 2^-6).  A sum of k products of which every partial sum is at most S = sum |a||b| in magnitude: each of its k additions rounds once, so
k 2^-24 S; a scale's product and its multiplication round once more for every block of 128: 2 (k / 128) 2^-24 S; the bias one more.
e4m3 operands with bf16 or e4m3 results go through the 8-bit matrix instruction, which lines the eight products of a group up with the
largest and keeps 13 bits below its leading one: the seven others are off by at most 2^-13 of it each, 7 2^-13 S in all."""
import struct
import threading

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
MATMUL = struct.Struct("=QqQqQqqQqqQqQqQqQQqqqqiiiiii")          # dce_matmul_desc
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, F8: 2.0 ** -4}


@pytest.fixture(scope="module")
def ops():
    from deep_contact_estimator_amd import ops
    return ops


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- plain implementations in 64 bits -----------------------------------------------------------------------------------------
def round_e4m3(v):
    """to the nearest e4m3 number, ties to even, of |v| <= 448: a step is 2^(exponent - 3), 2^-9 from 2^-6 down"""
    v = np.asarray(v, np.float64)
    _, p = np.frexp(np.where(np.isfinite(v), v, 1.0))
    step = np.ldexp(1.0, np.maximum(p - 1, -6) - 3)
    return np.where(np.isfinite(v), np.rint(v / step) * step, np.nan)


def block_exponents(most):
    f, p = np.frexp(most)
    return np.where(most == 0, -126, np.clip(np.where(f > 0.875, p - 8, p - 9), -126, 120))


def plain_quantize(x, rows):
    """(m, k) -> values of q, exponents (m / rows, k / 128)"""
    x = x.detach().double().cpu().numpy()
    m, k = x.shape
    kb, mb = -(-k // 128), -(-m // rows)
    q, e = np.zeros((m, k)), np.zeros((mb, kb), np.int64)
    mag = np.where(np.isfinite(x), np.abs(x), 0)
    for t in range(kb):
        for u in range(mb):
            at = slice(u * rows, (u + 1) * rows), slice(t * 128, (t + 1) * 128)
            e[u, t] = block_exponents(mag[at].max())
            q[at] = round_e4m3(np.where(np.isfinite(x[at]), np.ldexp(x[at], -int(e[u, t])), np.nan))
    return q, e


def number(s):
    return s.double() if s.dtype != E8 else torch.exp2(s.view(torch.uint8).double() - 127)


def plain_rows(a, sa):
    """a's rows as 64-bit numbers"""
    a = a.double()
    return a if sa is None else a * number(sa).repeat_interleave(128, 0)[:a.shape[1]].t()


def plain_weights(b, sb):
    b = b.double()
    return b if sb is None else b * number(sb).repeat_interleave(128, -1).repeat_interleave(128, -2)[..., :b.shape[-2], :b.shape[-1]]


def plain_product(a, b, bias, relu, k, coarse=False):
    """value, and the largest error of its sums (coarse: those of the 8-bit matrix instruction)"""
    y = a @ b.t()
    size = a.abs() @ b.abs().t()
    err = ((k + 2 * (k // 128 + 1)) * 2.0 ** -24 + (7 * 2.0 ** -13 if coarse else 0)) * size
    if bias is not None:
        y = y + bias.double()
        err = err + 2.0 ** -24 * y.abs()
    return (y.clamp_min(0) if relu else y), err


def check(got, want, err, kind, what):
    d = (got.double() - want).abs()
    bound = err + HALF[kind] * (want.abs() + err) + 1e-38
    assert not torch.isnan(got.double()).any(), what
    assert (d <= bound).all(), (what, float((d - bound).max()), float((d / bound).max()))


def check_e4m3(q, s, want, err, what):
    """results in e4m3: the scale is that of the row's largest value to within its error, the values one rounding off"""
    n = want.shape[1]
    s = number(s)
    for u in range(s.shape[0]):
        at = slice(u * 128, min(n, (u + 1) * 128))
        most, slack = want[:, at].abs().amax(1), err[:, at].amax(1)
        floor = s[u] == 2.0 ** -126
        assert ((most - slack) <= 448 * s[u]).all(), what
        assert (floor | ((most + slack) > 224 * s[u])).all(), what
        v = want[:, at] / s[u][:, None]
        d = (q[:, at].double() - v).abs()
        e = err[:, at] / s[u][:, None]
        assert (d <= e + 2.0 ** -4 * (v.abs() + e) + 2.0 ** -10).all(), what


# ---- quantize -------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m, k", [(1, 1), (1, 128), (3, 127), (5, 129), (17, 4736), (130, 260), (64, 513), (300, 16)])
@pytest.mark.parametrize("scale", [E8, torch.float32])
def test_quantize_rows(ops, m, k, kind, scale):
    x = (torch.randn(m, k, generator=gen(m * k), device="cuda") * torch.exp2(8 * torch.randn(m, 1, generator=gen(k), device="cuda"))).to(kind)
    q, s = ops.quantize(x, scale_dtype=scale)
    want, e = plain_quantize(x, 1)
    assert q.dtype == F8 and s.dtype == scale and tuple(s.shape) == (-(-k // 128), m)
    assert np.array_equal(number(s).cpu().numpy(), np.exp2(e.T.astype(np.float64)))
    assert np.array_equal(q.double().cpu().numpy(), want)


@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (129, 257), (16, 512), (250, 96), (3, 40, 200), (2, 256, 128)])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_quantize_weights(ops, shape, kind):
    x = (torch.randn(*shape, generator=gen(7), device="cuda") * 0.03).to(kind)
    q, s = ops.quantize(x, rows=128)
    many = x.reshape(-1, *shape[-2:])
    for i in range(many.shape[0]):
        want, e = plain_quantize(many[i], 128)
        assert np.array_equal(number(s).reshape(-1, *s.shape[-2:])[i].cpu().numpy(), np.exp2(e.astype(np.float64)))
        assert np.array_equal(q.reshape(-1, *shape[-2:])[i].double().cpu().numpy(), want)


def test_quantize_edges(ops):
    """zeros, the largest and smallest numbers, numbers on every boundary of the scale and of the rounding, NaN and infinities"""
    x = torch.zeros(12, 256, device="cuda")
    x[1] = 3.4028234663852886e38
    x[2] = 1e-45
    x[3, 0], x[3, 1] = 2.0 ** -126, 2.0 ** -133
    x[4, 0], x[4, 1:5] = 448.0, torch.tensor([447.0, 1.0625, 1.1875, -17.0])      # ties: 1.0625 and 1.1875 lie between two e4m3 numbers
    x[5, 0] = float(np.nextafter(np.float32(448), np.float32(500)))
    x[6, :128] = torch.arange(128) * 2.0 ** -10
    x[6, 0] = 448
    x[7, 3], x[7, 4], x[7, 5], x[7, 6] = float("nan"), float("inf"), -float("inf"), 100.0
    x[8] = float("inf")
    x[9] = float("nan")
    x[10, 0], x[10, 1] = -0.0, -448 * 2.0 ** 30
    for kind in (torch.float32, torch.bfloat16):
        y = x.to(kind)
        q, s = ops.quantize(y)
        want, e = plain_quantize(y, 1)
        assert np.array_equal(number(s).cpu().numpy(), np.exp2(e.T.astype(np.float64)))
        assert np.array_equal(q.double().cpu().numpy(), want, equal_nan=True)


def test_quantize_strides_and_alignment(ops):
    base = torch.randn(40, 700, generator=gen(1), device="cuda").bfloat16()
    for x in (base[:, 1:300], base[3:9, 5:], base.t(), base[::3, 2:2 + 256], base[:1].expand(5, 700)):
        q, s = ops.quantize(x)
        want, e = plain_quantize(x, 1)
        assert np.array_equal(q.double().cpu().numpy(), want) and np.array_equal(number(s).cpu().numpy(), np.exp2(e.T.astype(np.float64)))


# ---- matmul_fp8 -----------------------------------------------------------------------------------------------------------------
def operands(ops, m, n, k, scale, seed, groups=0):
    g = gen(seed)
    x = torch.randn(m, k, generator=g, device="cuda") * torch.exp2(3 * torch.randn(m, 1, generator=g, device="cuda"))
    w = torch.randn(max(groups, 1), n, k, generator=g, device="cuda") * torch.exp2(3 * torch.randn(max(groups, 1), 1, 1, generator=g, device="cuda"))
    a, sa = ops.quantize(x, scale_dtype=scale)
    b, sb = ops.quantize(w, rows=128, scale_dtype=scale)
    if scale == torch.float32:              # scales of any value
        sa, sb = sa * (0.5 + torch.rand(sa.shape, generator=g, device="cuda")), sb * (0.5 + torch.rand(sb.shape, generator=g, device="cuda"))
    bias = torch.randn(max(groups, 1), n, generator=g, device="cuda")
    return (a, sa, b, sb, bias) if groups else (a, sa, b[0], sb[0], bias[0])


SIZES = [(1, 1, 1), (1, 2048, 4736), (2, 16, 128), (15, 17, 129), (16, 128, 256), (17, 130, 127), (30, 512, 2048), (33, 250, 1000), (64, 64, 64), (65, 129, 100), (129, 384, 48),
         (300, 1000, 384), (257, 256, 1419), (700, 512, 512), (1300, 2048, 640),
         (4100, 4200, 256), (4200, 2050, 384), (4099, 4104, 144), (8200, 2000, 128)]          # (enough tiles to fill the chip)


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, F8])
@pytest.mark.parametrize("scale", [E8, torch.float32])
@pytest.mark.parametrize("m, n, k", SIZES)
def test_matmul_fp8(ops, m, n, k, scale, out):
    a, sa, b, sb, bias = operands(ops, m, n, k, scale, m + n + k)
    for bias_, relu in ((bias, True), (None, False)):
        y = ops.matmul_fp8(a, sa, b, sb, bias=bias_, relu=relu, out_dtype=out)
        want, err = plain_product(plain_rows(a, sa), plain_weights(b, sb), bias_, relu, k, out != torch.float32)
        if out == F8:
            assert y[1].dtype == scale and tuple(y[1].shape) == (-(-n // 128), m)
            check_e4m3(*y, want, err, (m, n, k))
        else:
            check(y, want, err, out, (m, n, k, relu))


@pytest.mark.parametrize("scale", [E8, torch.float32])
@pytest.mark.parametrize("m, n, k", [(3, 40, 128), (40, 300, 131), (600, 256, 144), (3000, 1001, 131), (1030, 2048, 256), (2000, 2048, 128), (4096, 2048, 128), (5000, 2048, 144), (8192, 2048, 256)])
def test_scales_of_e4m3_results_next_to_a_border(ops, m, n, k, scale):
    """A block's largest value on 448 * 2^8, and 4 to either side of it (2^-15 of it, which the 8-bit matrix instruction drops next to it): the smallest
    exponent with max <= 448 * 2^e is 8, 8 and 9.  Every fourth row, in one block of every two."""
    a, b = torch.zeros(m, k, device="cuda"), torch.zeros(n, k, device="cuda")
    rows = torch.arange(m, device="cuda")
    a[:, 0] = torch.where(rows % 4 == 0, 256.0, 1.0)
    a[:, 1] = torch.where(rows % 4 == 0, (rows // 4 % 3 - 1) * 2.0, 0.0)
    b[5::256, 0], b[5::256, 1], b[:, 2] = 448.0, 2.0, 1.0
    a[:, 2] = 1.0
    a, b = a.to(F8), b.to(F8)
    sa, sb = torch.ones(-(-k // 128), m, device="cuda"), torch.ones(-(-n // 128), -(-k // 128), device="cuda")
    sa, sb = (v if scale == torch.float32 else torch.full(v.shape, 127, dtype=torch.uint8, device="cuda").view(E8) for v in (sa, sb))
    for bias in (None, torch.zeros(n, device="cuda")):
        q, s = ops.matmul_fp8(a, sa, b, sb, bias=bias, out_dtype=F8)
        y = a.double() @ b.double().t()
        for t in range(-(-n // 128)):
            e = torch.from_numpy(block_exponents(y[:, t * 128:(t + 1) * 128].abs().amax(1).cpu().numpy())).cuda()
            assert torch.equal(number(s)[t], torch.exp2(e.double())), (t, m, n, k)
            assert (q[:, t * 128:(t + 1) * 128].double() * number(s)[t][:, None] - y[:, t * 128:(t + 1) * 128]).abs().le(2.0 ** -4 * y[:, t * 128:(t + 1) * 128].abs() + 8).all()


@pytest.mark.parametrize("m, n, k", [(70, 130, 128), (1030, 300, 131), (8192, 2048, 144)])
def test_scales_where_every_value_is_next_to_a_border(ops, m, n, k):
    a, b = torch.zeros(m, k, device="cuda"), torch.zeros(n, k, device="cuda")
    a[:, 0], a[:, 1], b[:, 0], b[:, 1] = 256.0, (torch.arange(m, device="cuda") % 3 - 1) * 2.0, 448.0, 2.0
    sa, sb = (torch.full(shape, 127, dtype=torch.uint8, device="cuda").view(E8) for shape in ((-(-k // 128), m), (-(-n // 128), -(-k // 128))))
    q, s = ops.matmul_fp8(a.to(F8), sa, b.to(F8), sb, out_dtype=F8)
    e = 8 + (a[:, 1] > 0).double()
    assert torch.equal(number(s), torch.exp2(e).expand(-(-n // 128), m))
    assert torch.equal(q.double(), torch.where(a[:, 1:2] > 0, 224.0, 448.0).double().expand(m, n))
    again = ops.matmul_fp8(a.to(F8), sa, b.to(F8), sb, out_dtype=F8)
    assert torch.equal(again[0].view(torch.uint8), q.view(torch.uint8)) and torch.equal(again[1].view(torch.uint8), s.view(torch.uint8))


@pytest.mark.parametrize("m, n, k", [(2000, 2040, 400), (1571, 2048, 272), (4000, 2048, 656), (5000, 2040, 528), (8100, 2048, 16), (8100, 2000, 240), (8100, 2048, 1040), (3000, 1001, 419), (5000, 300, 63)])
@pytest.mark.parametrize("form", ["bf16", E8, torch.float32])
def test_products_whose_k_ends_inside_a_step(ops, m, n, k, form):
    """in every tile size: what lies behind K in a wider tensor (NaN here) is not part of the sums"""
    gap = 16 if k % 16 == 0 else 1
    a, sa, b, sb, bias, offsets, index = grouped_inputs(ops, m, n, k, 1, form, [m], False, k)

    def widened(t):
        wide = torch.full((*t.shape[:-1], t.shape[-1] + gap), float("nan"), device="cuda").to(t.dtype)
        wide.view(torch.int16 if form == "bf16" else torch.uint8)[..., :k] = t.view(torch.int16 if form == "bf16" else torch.uint8)
        return wide[..., :k]
    for out in (torch.float32, torch.bfloat16):
        y = ops.matmul_grouped(widened(a), widened(b), offsets, a_scale=sa, b_scale=sb, bias=bias, out_dtype=out)
        want, err = plain_grouped(a, sa, b, sb, bias, [m], None, False, form != "bf16" and out != torch.float32)
        check(y, want, err, out, (m, n, k))


def test_matmul_fp8_whole_numbers_are_exact(ops):
    """small whole numbers and powers of two: every sum is exact, so every lane, row and scale is where it belongs or the numbers differ"""
    g = gen(5)
    m, n, k = 200, 300, 520
    a = torch.randint(-8, 9, (m, k), generator=g, device="cuda").float()
    b = torch.randint(-8, 9, (n, k), generator=g, device="cuda").float()
    ea = torch.randint(-3, 4, (5, m), generator=g, device="cuda")
    eb = torch.randint(-3, 4, (3, 5), generator=g, device="cuda")
    for kind in (E8, torch.float32):
        sa, sb = [((e + 127).to(torch.uint8).view(E8) if kind == E8 else torch.exp2(e.float())) for e in (ea, eb)]
        y = ops.matmul_fp8(a.to(F8), sa, b.to(F8), sb, out_dtype=torch.float32)
        assert torch.equal(y.double(), plain_rows(a.to(F8), sa) @ plain_weights(b.to(F8), sb).t())


def test_matmul_fp8_nan_and_scale_edges(ops):
    a, sa, b, sb, bias = operands(ops, 40, 140, 300, E8, 3)
    a.view(torch.uint8)[7, 200] = 0x7f
    y = ops.matmul_fp8(a, sa, b, sb, relu=True, out_dtype=torch.float32)
    assert torch.isnan(y[7]).all() and not torch.isnan(torch.cat([y[:7], y[8:]])).any()
    q, s = ops.matmul_fp8(a, sa, b, sb, out_dtype=F8)
    assert torch.isnan(q[7].float()).all() and not torch.isnan(q[8].float()).any()
    a, sa, b, sb, bias = operands(ops, 40, 140, 300, E8, 3)
    sa.view(torch.uint8)[1, 9] = 255                          # a scale that is no number
    y = ops.matmul_fp8(a, sa, b, sb, out_dtype=torch.float32)
    assert torch.isnan(y[9]).all() and not torch.isnan(y[10]).any()
    sa32, sb32 = number(operands(ops, 40, 140, 300, E8, 3)[1]).float(), number(sb).float()
    sa32[0, 4] = float("nan")
    y = ops.matmul_fp8(a, sa32, b, sb32, out_dtype=torch.float32)
    assert torch.isnan(y[4]).all() and not torch.isnan(y[5]).any()
    # exponents far apart cancel: 2^120 and 2^-120
    one = torch.ones(16, 128, device="cuda").to(F8)
    up, down = torch.full((1, 16), 247, dtype=torch.uint8, device="cuda").view(E8), torch.full((1, 1), 7, dtype=torch.uint8, device="cuda").view(E8)
    assert (ops.matmul_fp8(one, up, one, down, out_dtype=torch.float32) == 128).all()
    # the largest and the smallest values whose every operand is a normal fp32 number: 448 * 2^119, 2^-9 * 2^-117
    for v, up, w, down in ((448.0, 246, 448.0, 10), (448.0, 246, 2.0 ** -9, 10), (2.0 ** -9, 10, 448.0, 246), (2.0 ** -9, 10, 2.0 ** -9, 246)):
        x, y = torch.full((16, 128), v, device="cuda").to(F8), torch.full((16, 128), w, device="cuda").to(F8)
        up, down = torch.full((1, 16), up, dtype=torch.uint8, device="cuda").view(E8), torch.full((1, 1), down, dtype=torch.uint8, device="cuda").view(E8)
        for kind in (torch.float32, torch.bfloat16):
            assert (ops.matmul_fp8(x, up, y, down, out_dtype=kind) == 128 * v * w * 4).all(), (v, w, kind)


def test_matmul_fp8_strides(ops):
    """rows with gaps, rows that are not aligned, results inside a larger tensor whose rest stays as it was"""
    m, n, k = 70, 90, 300
    a, sa, b, sb, bias = operands(ops, m, n, k, torch.float32, 11)
    for pad, lead in ((1, 0), (16, 16), (20, 4), (212, 0), (7, 3)):
        wide = lambda t: torch.zeros(t.shape[0], t.shape[1] + pad, dtype=torch.uint8, device="cuda").fill_(0x7f)          # noqa: E731  (gaps hold NaN)
        aw, bw = wide(a), wide(b)
        lead = min(lead, pad)
        aw[:, lead:lead + k], bw[:, lead:lead + k] = a.view(torch.uint8), b.view(torch.uint8)
        av, bv = aw.view(F8)[:, lead:lead + k], bw.view(F8)[:, lead:lead + k]
        for kind in (torch.float32, torch.bfloat16, F8):
            want, err = plain_product(plain_rows(a, sa), plain_weights(b, sb), bias, False, k, kind != torch.float32)
            big = torch.full((m + 4, n + pad), 3.0, device="cuda").to(kind)
            out = big[2:2 + m, lead:lead + n]
            y = ops.matmul_fp8(av, sa, bv, sb, bias=bias, out_dtype=kind, out=out)
            if kind == F8:
                check_e4m3(out, y[1], want, err, (pad, lead))
            else:
                check(out, want, err, kind, (pad, lead))
            rest = torch.ones(big.shape, dtype=torch.bool, device="cuda")
            rest[2:2 + m, lead:lead + n] = False
            assert (big.float()[rest] == 3).all()


def test_empty_sizes(ops):
    a, sa, b, sb, bias = operands(ops, 4, 8, 128, E8, 1)
    assert ops.matmul_fp8(a[:0], sa[:, :0], b, sb).shape == (0, 8)
    assert ops.matmul_fp8(a, sa, b[:0], sb[:0]).shape == (4, 0)
    y = ops.matmul_fp8(a[:, :0], sa[:0], b[:, :0], sb[:, :0], bias=bias, out_dtype=torch.float32)
    assert torch.equal(y, bias.expand(4, 8))
    q, s = ops.quantize(torch.zeros(0, 256, device="cuda"))
    assert q.shape == (0, 256) and s.shape == (2, 0)


# ---- matmul_grouped -------------------------------------------------------------------------------------------------------------
def counts_of(kind, m, groups, seed):
    if kind == "even":
        return [m // groups + (i < m % groups) for i in range(groups)]
    if kind == "one":
        return [m if i == groups // 2 else 0 for i in range(groups)]
    r = np.random.RandomState(seed)
    c = r.multinomial(m, r.dirichlet(np.full(groups, 0.4)))
    c[0] += c[-1]
    c[-1] = 0                                                # the last group is empty
    return [int(v) for v in c]


def grouped_inputs(ops, m, n, k, groups, form, counts, gather, seed):
    g = gen(seed)
    rows = m + 5 if gather else m
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")
    index = torch.randint(0, rows, (m,), generator=g, device="cuda", dtype=torch.int32) if gather else None        # (rows more than once, rows never)
    if form == "bf16":
        a = torch.randn(rows, k, generator=g, device="cuda").bfloat16()
        b = torch.randn(groups, n, k, generator=g, device="cuda").bfloat16()
        sa = sb = None
        bias = torch.randn(groups, n, generator=g, device="cuda")
    else:
        a, sa, b, sb, bias = operands(ops, rows, n, k, form, seed, groups)
    return a, sa, b, sb, bias, offsets, index


def plain_grouped(a, sa, b, sb, bias, counts, index, relu, coarse=False):
    x, w = plain_rows(a, sa), plain_weights(b, sb)
    if index is not None:
        bad = (index < 0) | (index >= a.shape[0])
        x = torch.where(bad[:, None], 0.0, x[index.clamp(0, a.shape[0] - 1).long()])
    at, ys, es = 0, [], []
    for i, c in enumerate(counts):
        y, e = plain_product(x[at:at + c], w[i], None if bias is None else bias[i], relu, x.shape[1], coarse)
        ys.append(y)
        es.append(e)
        at += c
    return torch.cat(ys), torch.cat(es)


@pytest.mark.parametrize("form", ["bf16", E8, torch.float32])
@pytest.mark.parametrize("m, n, k, groups, kind", [
    (1, 16, 64, 1, "even"), (8, 512, 256, 8, "even"), (5, 40, 100, 9, "ragged"), (30, 128, 512, 4, "ragged"), (64, 130, 129, 3, "ragged"), (65, 96, 200, 2, "one"), (100, 33, 65, 7, "one"),
    (257, 512, 384, 5, "ragged"), (777, 200, 320, 64, "ragged"), (900, 256, 256, 100, "ragged"), (1500, 320, 512, 3, "ragged"), (9000, 2100, 256, 6, "ragged"), (5000, 1500, 384, 7, "ragged"), (5000, 1500, 400, 7, "ragged"), (40, 16, 48, 1024, "ragged")])
def test_matmul_grouped(ops, m, n, k, groups, kind, form):
    counts = counts_of(kind, m, groups, m)
    for gather, out, relu in ((False, torch.float32, False), (True, torch.bfloat16, True)):
        a, sa, b, sb, bias, offsets, index = grouped_inputs(ops, m, n, k, groups, form, counts, gather, m + k)
        y = ops.matmul_grouped(a, b, offsets, index=index, a_scale=sa, b_scale=sb, bias=bias, relu=relu, out_dtype=out)
        want, err = plain_grouped(a, sa, b, sb, bias, counts, index, relu, form != "bf16" and out != torch.float32)
        check(y, want, err, out, (m, n, k, groups, kind, gather))
    if form != "bf16":
        y = ops.matmul_grouped(a, b, offsets, index=index, a_scale=sa, b_scale=sb, bias=bias, relu=True, out_dtype=F8)
        check_e4m3(*y, want, err, (m, n, k, groups, kind))


def test_rows_of_no_group_stay_as_they_were(ops):
    a, sa, b, sb, bias, _, _ = grouped_inputs(ops, 50, 70, 90, 3, "bf16", [50, 0, 0], False, 2)
    offsets = torch.tensor([4, 20, 20, 33], dtype=torch.int32, device="cuda")
    for kind in (torch.float32, torch.bfloat16):
        out = torch.full((50, 70), 9.0, dtype=kind, device="cuda")
        ops.matmul_grouped(a, b, offsets, bias=bias, out_dtype=kind, out=out)
        assert (out[:4] == 9).all() and (out[33:] == 9).all()
        want, err = plain_grouped(a[4:33], None, b, None, bias, [16, 0, 13], None, False)
        check(out[4:33], want, err, kind, "inside")


def test_offsets_are_held_inside_the_rows(ops):
    """offsets that point behind the rows or fall: nothing outside the result is written, the groups that are right come out right"""
    a, sa, b, sb, bias, _, _ = grouped_inputs(ops, 40, 33, 64, 3, "bf16", [40, 0, 0], False, 2)
    big = torch.full((60, 33), 9.0, device="cuda")
    ops.matmul_grouped(a, b, torch.tensor([0, 16, 10, 5000], dtype=torch.int32, device="cuda"), bias=bias, out_dtype=torch.float32, out=big[10:50])
    assert (big[:10] == 9).all() and (big[50:] == 9).all()
    ops.matmul_grouped(a, b, torch.tensor([-7, 16, 30, 40], dtype=torch.int32, device="cuda"), bias=bias, out_dtype=torch.float32, out=big[10:50])
    want, err = plain_grouped(a, None, b, None, bias, [16, 14, 10], None, False)
    check(big[10:50], want, err, torch.float32, "held")


@pytest.mark.parametrize("form", ["bf16", E8, torch.float32])
def test_an_index_outside_the_rows_reads_zeros(ops, form):
    counts = [20, 0, 30]
    a, sa, b, sb, bias, offsets, index = grouped_inputs(ops, 50, 64, 160, 3, form, counts, True, 4)
    index[3], index[25], index[26] = -1, a.shape[0], 2 ** 31 - 1
    y = ops.matmul_grouped(a, b, offsets, index=index, a_scale=sa, b_scale=sb, bias=bias, out_dtype=torch.float32)
    want, err = plain_grouped(a, sa, b, sb, bias, counts, index, False)
    check(y, want, err, torch.float32, "zeros")
    assert torch.equal(y[3], bias[0]) and torch.equal(y[25], bias[2])


def test_broadcast_weights_and_bias(ops):
    a, _, b, _, bias, offsets, _ = grouped_inputs(ops, 60, 48, 128, 4, "bf16", [15] * 4, False, 6)
    y = ops.matmul_grouped(a, b[:1].expand(4, 48, 128), offsets, bias=bias[:1].expand(4, 48), out_dtype=torch.float32)
    want, err = plain_product(a.double(), b[0].double(), bias[0], False, 128)
    check(y, want, err, torch.float32, "broadcast")


def test_far_rows(ops):
    """rows, weights and results that lie more than 2^32 bytes from their start"""
    k, n, step = 128, 32, 1 << 27
    wide = torch.zeros(40, step, dtype=torch.uint8, device="cuda")                    # 5.4 GB: row 39 starts behind 4 GB
    a, sa, b, sb, bias = operands(ops, 40, n, k, E8, 12)
    wide[:, :k] = a.view(torch.uint8)
    wide[:n, 4096:4096 + k] = b.view(torch.uint8)
    out = wide.view(F8)[:, 8192:8192 + n]
    q, s = ops.matmul_fp8(wide.view(F8)[:, :k], sa, wide.view(F8)[:n, 4096:4096 + k], sb, bias=bias, out_dtype=F8, out=out)
    want, err = plain_product(plain_rows(a, sa), plain_weights(b, sb), bias, False, k, True)
    check_e4m3(out, s, want, err, "far")
    x = torch.randn(40, 256, generator=gen(3), device="cuda").bfloat16()
    far = wide.view(torch.bfloat16)[:, 8192:8192 + 256]
    far.copy_(x)
    q, s = ops.quantize(far)
    q2, s2 = ops.quantize(x)
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s.view(torch.uint8), s2.view(torch.uint8))


@pytest.mark.parametrize("guard", [1, 2])
@pytest.mark.parametrize("m, n, k, form, out", [(1, 16, 128, "bf16", 0), (33, 250, 1000, E8, 0), (5, 40, 419, E8, 1), (300, 130, 419, torch.float32, 2), (900, 300, 65, "bf16", 1),
                                                (700, 512, 528, E8, 2), (2000, 2040, 400, torch.float32, 1), (5000, 1500, 384, E8, 1), (8100, 2048, 240, E8, 2), (8100, 2048, 256, torch.float32, 1)])
def test_products_stay_inside_their_buffers(ops, m, n, k, form, out, guard):
    """every buffer of the call ends (1) or begins (2) at an unmapped page"""
    import ctypes as C

    from deep_contact_estimator_amd import _lib, contact_cnn, synth
    kind = (torch.float32, torch.bfloat16, F8)[out]
    a, sa, b, sb, bias, offsets, _ = grouped_inputs(ops, m, n, k, 1, form, [m], False, m)
    lib, hip = _lib.load(), _lib._load_hip_runtime()
    hip.hipMemcpy.argtypes, hip.hipMemcpy.restype = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_int], C.c_int
    model = contact_cnn(device=0, max_batch=1, tune={"guard_alloc": guard})
    model.load_state_dict(synth.make_state_dict(1, "uniform")).eval()
    model.predict(torch.zeros(1, 150, 54, device="cuda"))
    held = []

    def placed(t, nbytes=0):
        p = C.c_void_p()
        _lib.check(lib.dce_debug_alloc(model._ctx, t.numel() * t.element_size() if t is not None else nbytes, C.byref(p)), model._ctx)
        held.append(p)
        if t is not None:
            assert hip.hipMemcpy(p, t.data_ptr(), t.numel() * t.element_size(), 3) == 0
        return p.value
    y = torch.empty(m, n, dtype=kind, device="cuda")
    ys = torch.empty(-(-n // 128), m, dtype=sa.dtype, device="cuda") if out == 2 else None
    nb, kb = -(-n // 128), -(-k // 128)
    torch.cuda.synchronize()
    py, pys = placed(None, y.numel() * y.element_size()), placed(None, ys.numel() * ys.element_size()) if out == 2 else 0
    d = MATMUL.pack(placed(a), k, 0 if sa is None else placed(sa), m, placed(b), k, 0, 0 if sb is None else placed(sb), kb, nb * kb, placed(bias), 0, py, n, pys, m,
                    placed(offsets), 0, m, m, n, k, 1, 1 if form == "bf16" else 2, 1 if form == torch.float32 else 0, out, 0, 0)
    _lib.check(lib.dce_matmul(0, None, d))
    torch.cuda.synchronize()
    assert hip.hipMemcpy(y.data_ptr(), py, y.numel() * y.element_size(), 3) == 0 and (out != 2 or hip.hipMemcpy(ys.data_ptr(), pys, ys.numel() * ys.element_size(), 3) == 0)
    torch.cuda.synchronize()
    for p in held:
        _lib.check(lib.dce_debug_free(model._ctx, p), model._ctx)
    model.close()
    want, err = plain_grouped(a, sa, b, sb, bias, [m], None, False, form != "bf16" and out != 0)
    if out == 2:
        check_e4m3(y, ys, want, err, (m, n, k))
    else:
        check(y, want, err, kind, (m, n, k))


def test_results_may_lie_beside_an_operand_but_not_on_it(ops):
    both = torch.randn(64, 192, generator=gen(2), device="cuda").bfloat16()
    w, off = torch.randn(1, 64, 64, generator=gen(3), device="cuda").bfloat16(), torch.tensor([0, 64], dtype=torch.int32, device="cuda")
    want = ops.matmul_grouped(both[:, 64:128].contiguous(), w, off)
    assert torch.equal(ops.matmul_grouped(both[:, 64:128], w, off, out=both[:, 128:]), want) and torch.equal(both[:, 128:], want)
    assert torch.equal(ops.matmul_grouped(both[:, 64:128], w, off, out=both[:, :64]), want)
    for at in (0, 1, 63, 64):
        with pytest.raises(RuntimeError, match="overlaps"):
            ops.matmul_grouped(both[:, at:at + 64], w, off, out=both[:, 63:127] if at else both[:, :64])
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.matmul_grouped(both[:, :64], w, off, out=w[0])


# ---- group_rows, decide -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
@pytest.mark.parametrize("n, groups", [(0, 3), (1, 1), (1, 7), (30, 4), (64, 64), (65, 2), (500, 1), (2048, 17), (2049, 5), (10000, 1024), (100001, 64), (700000, 33)])
def test_group_rows(ops, n, groups, kind):
    g = gen(n + groups)
    ids = torch.randint(-1, groups + 2, (n,), generator=g, device="cuda").to(kind)          # some belong to no group
    if n > 2:
        ids[0], ids[-1] = -2 ** 31, 2 ** 31 - 1
    if kind == torch.int64 and n > 4:
        ids[2], ids[3] = 2 ** 32, -2 ** 40                                                  # (not group 0)
    offsets, order, place = ops.group_rows(ids, groups)
    h = ids.cpu().numpy().astype(np.int64)
    valid = (h >= 0) & (h < groups)
    key = np.where(valid, h, groups)
    want = np.argsort(key, kind="stable")
    total = int(valid.sum())
    assert np.array_equal(offsets.cpu().numpy(), np.concatenate([[0], np.cumsum(np.bincount(key, minlength=groups + 1)[:groups])]))
    assert np.array_equal(order.cpu().numpy()[:total], want[:total]) and (order.cpu().numpy()[total:] == -1).all()
    at = np.full(n, -1)
    at[want[:total]] = np.arange(total)
    assert np.array_equal(place.cpu().numpy(), at)


def test_decide(ops):
    v = torch.randint(-3, 4, (300, 16), generator=gen(1), device="cuda").float()            # many ties
    v[5, 3] = v[5, 9] = float("nan")
    v[6] = float("nan")
    v[7] = -float("inf")
    index = torch.randint(-1, 301, (500,), generator=gen(2), device="cuda", dtype=torch.int32)
    for ix in (None, index):
        d = ops.decide(v, ix)
        h = v.cpu().numpy()
        if ix is not None:
            i = ix.cpu().numpy()
            h = np.where(((i >= 0) & (i < 300))[:, None], h[np.clip(i, 0, 299)], np.nan)
        assert np.array_equal(d["logits"].cpu().numpy(), h, equal_nan=True)
        want = torch.max(torch.from_numpy(h), 1)[1].numpy()
        first = np.where(np.isnan(h).any(1), np.isnan(h).argmax(1), want)
        assert np.array_equal(d["pred"].cpu().numpy(), first)
        assert np.array_equal(d["contacts"].cpu().numpy(), (first[:, None] >> np.array([3, 2, 1, 0])) & 1)


# ---- as they are used together --------------------------------------------------------------------------------------------------------
def chain(ops, x, ids, heads, w1, s1, b1, w2, s2, b2):
    offsets, order, place = ops.group_rows(ids, heads)
    q, s = ops.quantize(x)
    h, hs = ops.matmul_grouped(q, w1, offsets, index=order, a_scale=s, b_scale=s1, bias=b1, relu=True, out_dtype=F8)
    z = ops.matmul_grouped(h, w2, offsets, a_scale=hs, b_scale=s2, bias=b2, out_dtype=torch.float32)
    return ops.decide(z, place)


def chain_inputs(ops, n, heads, seed):
    g = gen(seed)
    x = torch.randn(n, 300, generator=g, device="cuda").bfloat16()
    ids = torch.randint(0, heads, (n,), generator=g, device="cuda", dtype=torch.int32)
    w1, s1 = ops.quantize(torch.randn(heads, 256, 300, generator=g, device="cuda") / 17, rows=128)
    w2, s2 = ops.quantize(torch.randn(heads, 16, 256, generator=g, device="cuda") / 16, rows=128)
    b1, b2 = (torch.randn(heads, k, generator=g, device="cuda") for k in (256, 16))
    return x, ids, heads, w1, s1, b1, w2, s2, b2


@pytest.mark.parametrize("n, heads", [(1, 3), (40, 5), (600, 8), (3000, 2)])
def test_two_layers_of_a_bank(ops, n, heads):
    """group_rows, quantize, two grouped products of which the first hands the second its operand, decide.  Held stage by stage: each stage's inputs are
    the stage's before it, so that a value next to an e4m3 border may fall to either side."""
    x, ids, _, w1, s1, b1, w2, s2, b2 = inputs = chain_inputs(ops, n, heads, n)
    d = chain(ops, *inputs)
    offsets, order, place = ops.group_rows(ids, heads)
    q, s = ops.quantize(x)
    h, hs = ops.matmul_grouped(q, w1, offsets, index=order, a_scale=s, b_scale=s1, bias=b1, relu=True, out_dtype=F8)
    counts = offsets.diff().tolist()
    want, err = plain_grouped(q, s, w1, s1, b1, counts, order, True, True)
    check_e4m3(h, hs, want, err, n)
    want, err = plain_grouped(h, hs, w2, s2, b2, counts, None, False)
    check(d["logits"], want[place.long()], err[place.long()], torch.float32, n)
    assert torch.equal(d["pred"], torch.max(d["logits"], 1)[1].int())


def test_the_same_call_gives_the_same_bits_also_beside_others(ops):
    inputs = chain_inputs(ops, 900, 6, 1)
    want = chain(ops, *inputs)["logits"].clone()
    got = {}

    def work(i):
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(st):
            got[i] = [chain(ops, *inputs)["logits"] for _ in range(8)]
        st.synchronize()
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert len(got) == 4 and all(torch.equal(v, want) for r in got.values() for v in r)


def test_captured_and_replayed(ops):
    """the chain in a graph, replayed on new inputs in place, with eager calls of the same operators in between; two graphs of it, in turn"""
    sets = [chain_inputs(ops, n, 5, n) for n in (300, 2100)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in sets:
            chain(ops, *s)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(chain(ops, *s))
        graphs.append(g)
    for turn in range(4):
        for i, s in enumerate(sets):
            fresh = chain_inputs(ops, s[0].shape[0], 5, 100 + turn)
            s[0].copy_(fresh[0])
            s[1].copy_(fresh[1])
            want = chain(ops, *s)
            graphs[i].replay()
            torch.cuda.synchronize()
            for k in want:
                assert torch.equal(outs[i][k], want[k]), (turn, i, k)


def test_refusals_on_the_device(ops):
    a, sa, b, sb, bias = operands(ops, 8, 16, 256, E8, 1)
    with pytest.raises(RuntimeError, match="expected a_scale"):
        ops.matmul_fp8(a, sa[:1], b, sb)
    with pytest.raises(RuntimeError, match="need a_scale"):
        ops.matmul_fp8(a, None, b, sb)
    with pytest.raises(RuntimeError, match="scales must both"):
        ops.matmul_fp8(a, sa, b, number(sb).float())
    with pytest.raises(RuntimeError, match="columns"):
        ops.matmul_fp8(a[:, :128], sa[:1], b, sb)
    with pytest.raises(RuntimeError, match="bias"):
        ops.matmul_fp8(a, sa, b, sb, bias=bias[:8])
    with pytest.raises(RuntimeError, match="out must"):
        ops.matmul_fp8(a, sa, b, sb, out=torch.empty(8, 17, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(RuntimeError, match="tensors on"):
        ops.matmul_fp8(a, sa, b.cpu(), sb)
    x = torch.zeros(4, 128, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="inference"):
        ops.quantize(x)
    with torch.no_grad():
        ops.quantize(x)
