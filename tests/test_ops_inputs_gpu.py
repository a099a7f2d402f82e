"""GPU: tensors that are not what their memory holds, and tensors of autograd: the operators take them as torch's own do, or refuse them."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from deep_contact_estimator_amd import contact_cnn, ops, synth   # noqa: E402


def same(a, b):
    return all(torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8)) for x, y in zip(a, b))


def test_views_that_stand_for_the_negative_of_their_memory():
    """such a view and a tensor of its values give the same bits"""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(70, 256, generator=g, device="cuda")
    neg, plain = torch._neg_view(x), -x
    assert neg.is_neg() and torch.equal(neg, plain)
    assert same(ops.quantize(neg), ops.quantize(plain))
    assert same(ops.quantize(neg, rows=128), ops.quantize(plain, rows=128))
    conj = torch.complex(x, x + 1).conj().imag                     # (how such views come about)
    assert conj.is_neg() and same(ops.quantize(conj), ops.quantize(-(x + 1)))
    w, offsets = torch.randn(2, 48, 256, generator=g, device="cuda").bfloat16(), torch.tensor([0, 30, 70], dtype=torch.int32, device="cuda")
    bias = torch.randn(2, 48, generator=g, device="cuda")
    a = x.bfloat16()
    want = ops.matmul_grouped(-a, w, offsets, bias=-bias)
    assert torch.equal(ops.matmul_grouped(torch._neg_view(a), w, offsets, bias=torch._neg_view(bias)), want)
    assert torch.equal(ops.matmul_grouped(-a, torch._neg_view(-w), offsets, bias=-bias), want)
    v = torch.randn(40, 16, generator=g, device="cuda")
    got, want = ops.decide(torch._neg_view(v)), ops.decide(-v)
    assert all(torch.equal(got[k], want[k]) for k in want)
    out = torch.zeros(70, 48, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="negative of their memory"):
        ops.matmul_grouped(a, w, offsets, out=torch._neg_view(out))


def test_the_models_too():
    x = torch.randn(3, 150, 54, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    for precision in ("fp32", "bf16_fc"):
        m = contact_cnn(device=0, precision=precision, max_batch=8)
        m.load_state_dict(synth.make_state_dict(1, "uniform")).eval()
        assert torch.equal(m(torch._neg_view(x)), m(-x))
        if precision == "bf16_fc":
            assert torch.equal(m.features(torch._neg_view(x)), m.features(-x))
        m.close()


def test_tangents_are_refused_and_not_lost():
    """a dual tensor of forward-mode differentiation, as any operand; its primal alone is an ordinary tensor"""
    import torch.autograd.forward_ad as fw
    g = torch.Generator(device="cuda").manual_seed(3)
    x, w, v = (torch.randn(*s, generator=g, device="cuda") for s in ((8, 128), (1, 16, 128), (5, 16)))
    a, b, offsets, bias = x.bfloat16(), w.bfloat16(), torch.tensor([0, 8], dtype=torch.int32, device="cuda"), torch.zeros(1, 16, device="cuda")
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))      # noqa: E731
        for grad in (torch.enable_grad, torch.no_grad):
            with grad():
                for call in (lambda: ops.quantize(dual(x)), lambda: ops.decide(dual(v)), lambda: ops.matmul_grouped(dual(a), b, offsets),
                             lambda: ops.matmul_grouped(a, dual(b), offsets), lambda: ops.matmul_grouped(a, b, offsets, bias=dual(bias))):
                    with pytest.raises(RuntimeError, match="tangent"):
                        call()
        assert same(ops.quantize(fw.unpack_dual(dual(x)).primal), ops.quantize(x))
        with torch.inference_mode():
            assert same(ops.quantize(x), ops.quantize(x.clone()))


def test_results_on_the_scales_that_a_product_reads_are_refused():
    x, w = torch.randn(256, 256, device="cuda"), torch.randn(256, 256, device="cuda")
    (q, s), (b, bs) = ops.quantize(x), ops.quantize(w, rows=128)
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.matmul_fp8(q, s, b, bs, out_dtype=torch.float8_e4m3fn, out_scale=s)
    two = torch.empty(2, *s.shape, dtype=torch.uint8, device="cuda").view(s.dtype)
    two.view(torch.uint8)[0] = s.view(torch.uint8)
    want = ops.matmul_fp8(q, s, b, bs, out_dtype=torch.float8_e4m3fn)
    got = ops.matmul_fp8(q, two[0], b, bs, out_dtype=torch.float8_e4m3fn, out_scale=two[1])          # beside them
    assert same(got, want) and torch.equal(two[0].view(torch.uint8), s.view(torch.uint8))


def test_writing_to_out_is_told_to_autograd():
    """a tensor that a backward pass still needs, given as `out` meanwhile: the backward pass refuses it, as after torch's own in-place operators"""
    g = torch.Generator(device="cuda").manual_seed(4)
    x, w = torch.randn(8, 16, generator=g, device="cuda"), torch.randn(1, 16, 16, generator=g, device="cuda").bfloat16()
    offsets = torch.tensor([0, 8], dtype=torch.int32, device="cuda")
    out = torch.ones(8, 16, device="cuda")
    p = torch.ones(8, 16, device="cuda", requires_grad=True)
    y = (p * out).sum()
    before = out._version
    ops.matmul_grouped(x.bfloat16(), w, offsets, out_dtype=torch.float32, out=out)
    assert out._version == before + 1
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()
    (q, s), (b, bs) = ops.quantize(torch.randn(8, 256, generator=g, device="cuda")), ops.quantize(torch.randn(130, 256, generator=g, device="cuda"), rows=128)
    out, scale = torch.empty(8, 130, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(2, 8, dtype=torch.uint8, device="cuda").view(s.dtype)
    versions = out._version, scale._version
    ops.matmul_fp8(q, s, b, bs, out_dtype=out.dtype, out=out, out_scale=scale)
    assert (out._version, scale._version) == (versions[0] + 1, versions[1] + 1)
    with torch.inference_mode():
        out = torch.empty(8, 16, device="cuda")
    ops.matmul_grouped(x.bfloat16(), w, offsets, out_dtype=torch.float32, out=out)                 # (has no version)
