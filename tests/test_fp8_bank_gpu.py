"""GPU: the paths that run the operators of ops.py -- the precision fp8_fc, the conv stack alone (features), the bank of FC heads.

Bounds are worked out from the numbers themselves, in 64 bits: a value rounded to bf16 is off by 2^-8 of itself, to e4m3 by 2^-4 (2^-10 of its block's
scale below the smallest normal number; the scale is at most 1/224 of the block's largest value), a sum of k products by k 2^-24 of the sum of their
magnitudes (7 2^-13 of it more in the 8-bit matrix instruction, test_ops_gpu.py); ReLU passes an error on, a layer its weights' magnitudes times it."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from deep_contact_estimator_amd import contact_bank, contact_cnn, ops, synth   # noqa: E402

F8 = torch.float8_e4m3fn


def windows(n, seed=0):
    return torch.randn(n, 150, 54, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def model(precision, seed=1, **kw):
    m = contact_cnn(device=0, precision=precision, **kw)
    m.load_state_dict(synth.make_state_dict(seed, "uniform")).eval()
    return m


def permuted(w):
    """fc.0's columns in the order t * 128 + c"""
    return w.reshape(-1, 128, 37).transpose(1, 2).reshape(w.shape).contiguous()


def f8_error(x, rows=1):
    """how far x's e4m3 form may be from x: (.., n, k)"""
    k = x.shape[-1]
    a = x.abs()
    top = torch.nn.functional.pad(a, (0, -k % 128)).unflatten(-1, (-1, 128)).amax(-1)
    if rows != 1:
        top = torch.nn.functional.pad(top, (0, 0, 0, -top.shape[-2] % rows)).unflatten(-2, (-1, rows)).amax(-2).repeat_interleave(rows, -2)[..., :x.shape[-2], :]
    return 2.0 ** -4 * a + 2.0 ** -10 / 224 * top.repeat_interleave(128, -1)[..., :k]


def layer(x, ex, w, ew, b, relu, coarse):
    """x W^T + b in 64 bits for operands off by at most ex, ew, and how far the result may be off"""
    y = x @ w.t() + b
    size = (x.abs() + ex) @ (w.abs() + ew).t()
    e = ex @ w.abs().t() + (x.abs() + ex) @ ew.t() + (x.shape[1] * 2.0 ** -23 + (7 * 2.0 ** -13 if coarse else 0)) * size + 2.0 ** -24 * (y.abs() + b.abs())
    return (y.clamp_min(0) if relu else y), e


def chain(feat, sd, f8, h2_fp32, off=None):
    """logits of a mode from its bf16 features, and how far they may be off; off: from the logits of other features, this far from its own"""
    f = feat.double()
    off = 0 * f if off is None else off
    sd = {k: torch.from_numpy(v).cuda().double() for k, v in sd.items() if k.startswith("fc.")}
    w1 = permuted(sd["fc.0.weight"])
    if f8:
        h, e = layer(f, f8_error(f.abs() + off) + off, w1, f8_error(w1, 128), sd["fc.0.bias"], True, True)
        e = e + f8_error(h.abs() + e)
        h, e = layer(h, e, sd["fc.3.weight"], f8_error(sd["fc.3.weight"], 128), sd["fc.3.bias"], True, True)
    else:
        h, e = layer(f, off, w1, 2.0 ** -8 * w1.abs(), sd["fc.0.bias"], True, False)
        e = e + 2.0 ** -8 * (h.abs() + e)
        h, e = layer(h, e, sd["fc.3.weight"], 2.0 ** -8 * sd["fc.3.weight"].abs(), sd["fc.3.bias"], True, False)
    if h2_fp32:
        return layer(h, e, sd["fc.6.weight"], 0 * sd["fc.6.weight"], sd["fc.6.bias"], False, False)
    e = e + 2.0 ** -8 * (h.abs() + e)
    return layer(h, e, sd["fc.6.weight"], 2.0 ** -8 * sd["fc.6.weight"].abs(), sd["fc.6.bias"], False, False)


def bits(out):
    return (out["pred"][:, None] >> torch.tensor([3, 2, 1, 0], device=out["pred"].device)) & 1


@pytest.mark.parametrize("n", [1, 2, 33, 256, 257, 700])
def test_fp8_fc_is_its_stages(n):
    """the precision's h2 is what features -> quantize -> matmul_fp8 -> matmul_fp8 gives, bit for bit; its logits are fc.6 of that"""
    sd = synth.make_state_dict(1, "uniform")
    m = model("fp8_fc", max_batch=1024)
    x = windows(n)
    t = {k: torch.from_numpy(v).cuda() for k, v in sd.items()}
    q, s = ops.quantize(m.features(x))
    w1, s1 = ops.quantize(permuted(t["fc.0.weight"]), rows=128)
    w2, s2 = ops.quantize(t["fc.3.weight"], rows=128)
    h, hs = ops.matmul_fp8(q, s, w1, s1, bias=t["fc.0.bias"], relu=True, out_dtype=F8)
    h2 = ops.matmul_fp8(h, hs, w2, s2, bias=t["fc.3.bias"], relu=True, out_dtype=torch.float32)
    taps = m.forward_taps(x.cpu().numpy())
    assert set(taps) == {"h2", "logits"} and np.array_equal(taps["h2"], h2.cpu().numpy())
    out = m.predict(x)
    assert np.array_equal(taps["logits"], out["logits"].cpu().numpy())
    assert any("e4m3" in k for k in m.last_plan())
    want, err = layer(h2.double(), 0 * h2.double(), t["fc.6.weight"].double(), 0 * t["fc.6.weight"].double(), t["fc.6.bias"].double(), False, False)
    assert ((out["logits"].double() - want).abs() <= err).all()
    assert torch.equal(out["pred"], out["logits"].max(1)[1].int()) and torch.equal(out["contacts"].long(), bits(out))
    m.close()


@pytest.mark.parametrize("n", [3, 300, 2500])
def test_fp8_fc_stays_within_what_its_roundings_allow(n):
    m = model("fp8_fc", max_batch=4096)
    x = windows(n, 1)
    want, err = chain(m.features(x), synth.make_state_dict(1, "uniform"), True, True)
    got = m.predict(x)["logits"].double()
    assert ((got - want).abs() <= err).all()
    # ... and of an fp32 evaluation: the same bound around the fp32 features, with how far the mode's bf16 features are from them
    full = model("fp32", max_batch=4096)
    f32 = torch.from_numpy(full.forward_taps(x.cpu().numpy())["feat"]).cuda().double().view(n, 128, 37).transpose(1, 2).reshape(n, 4736)
    want, err = chain(f32, synth.make_state_dict(1, "uniform"), True, True, off=(m.features(x).double() - f32).abs())
    assert ((got - want).abs() <= err).all()
    ref = full.predict(x)
    d = (got - ref["logits"].double()).abs().max() / ref["logits"].abs().max()
    flips = (m.predict(x)["pred"] != ref["pred"]).float().mean()
    print(f"fp8_fc, {n} windows: largest difference {float(d):.2e} of the largest logit, class changed in {float(flips):.2%}")
    m.close(); full.close()


def test_fp8_fc_chunks_sequences_and_online():
    m = model("fp8_fc", max_batch=64)
    x = windows(150, 2)
    whole = m.predict(x)["logits"]
    for i in range(0, 150, 64):
        assert torch.equal(m.predict(x[i:i + 64])["logits"], whole[i:i + 64])
    seq = synth.make_sequence(170, 3).astype(np.float32)
    one = m.infer_sequence(seq[-150:])["logits"]
    m.online_reset()
    for row in seq:
        got = m.online_push(row)
    assert np.array_equal(got[0], one[0]) and got[1] == int(one[0].argmax())
    dev = m.infer_sequence(torch.from_numpy(seq).cuda())
    assert np.array_equal(dev["logits"].cpu().numpy(), m.infer_sequence(seq)["logits"])
    m.close()


def test_fp8_fc_back_and_forth_between_precisions():
    """a context finalized again in another precision, and back, gives what fresh ones give"""
    x = windows(300, 4)
    a = model("fp8_fc", max_batch=512)
    first = a.predict(x)["logits"].clone()
    b = model("fp32", max_batch=512)
    for precision in ("fp32", "fp8_fc", "bf16_fc", "fp8_fc"):
        a._precision, a._finalized = precision, False
        got = a.predict(x)["logits"]
        if precision == "fp8_fc":
            assert torch.equal(got, first)
        elif precision == "fp32":
            assert torch.equal(got, b.predict(x)["logits"])
    a.close(); b.close()


@pytest.mark.parametrize("guard", [1, 2])
def test_fp8_fc_stays_inside_its_buffers(guard):
    """every buffer of the context ends (1) or begins (2) at an unmapped page"""
    plain, m = model("fp8_fc", max_batch=300), model("fp8_fc", max_batch=300, tune={"guard_alloc": guard})
    for n in (1, 31, 300):
        x = windows(n, n)
        assert torch.equal(m.predict(x)["logits"], plain.predict(x)["logits"])
    m.close(); plain.close()


def test_options_of_the_conv_stack():
    x = windows(20, 5)
    want, err = None, None
    for tune in (None, {"x3_permk": 0}, {"x3_conv": 0}, {"bf16_conv_h2": 0}):
        m = model("fp8_fc", max_batch=64, tune=tune)
        got = m.predict(x)["logits"].double()
        if want is None:
            want, err = chain(m.features(x), synth.make_state_dict(1, "uniform"), True, True)
        # (another conv kernel: features that differ in their last bf16 bit, within twice what the first one's roundings allow)
        assert ((got - want).abs() <= 2 * err).all(), tune
        m.close()


def test_refusals():
    m = model("fp8_fc", max_batch=16)
    with pytest.raises(RuntimeError, match="DCE_FP8_FC"):
        m.conv_layer_taps(windows(2).cpu().numpy())
    m.close()
    m = model("fp32", max_batch=16)
    with pytest.raises(RuntimeError, match="bf16 features"):
        m.features(windows(2))
    with pytest.raises(RuntimeError, match="CUDA"):
        m.features(windows(2).cpu())
    m.close()
    m = model("bf16_fc", max_batch=16, tune={"x3_conv": 0})
    with pytest.raises(RuntimeError, match="x3_conv"):
        m.features(windows(2))
    m.close()
    with pytest.raises(RuntimeError, match="precision"):
        contact_bank(precision="fp32")
    b = contact_bank(device=0, max_batch=16)
    with pytest.raises(RuntimeError, match="load_state_dict first"):
        b.predict(windows(2), torch.zeros(2, dtype=torch.int32))
    sd = synth.make_state_dict(1, "uniform")
    with pytest.raises(RuntimeError, match="heads"):
        b.load_state_dict(sd, [])
    with pytest.raises(RuntimeError, match="missing"):
        b.load_state_dict(sd, [sd, {"fc.0.weight": sd["fc.0.weight"]}])
    with pytest.raises(RuntimeError, match="mismatch"):
        b.load_state_dict(sd, [{**sd, "fc.3.bias": np.zeros(3, np.float32)}])
    b.load_state_dict(sd, [sd])
    with pytest.raises(RuntimeError, match="one head a window"):
        b.predict(windows(2), torch.zeros(3, dtype=torch.int32))


@pytest.mark.parametrize("n", [0, 1, 300])
def test_features_do_not_depend_on_the_call(n):
    """windows and raw rows, whole and in chunks of a smaller max_batch where the same conv kernel runs"""
    m = model("bf16_fc", max_batch=512)
    x = windows(n, 6)
    f = m.features(x)
    assert f.shape == (n, 4736) and f.dtype == torch.bfloat16
    if n:
        t = m.forward_taps(x.cpu().numpy())["feat"]                              # (channel by channel; another kernel above 256 windows)
        t = torch.from_numpy(t.astype(np.int32) << 16).view(torch.float32).cuda().view(n, 128, 37).transpose(1, 2).reshape(n, 4736)
        assert ((f.float() - t).abs() <= 2.0 ** -7 * t.abs() + 1e-3 * t.abs().max()).all()
        seq = torch.randn(n + 149, 54, device="cuda")
        whole = m.features(seq, raw_sequence=True)
        few = model("bf16_fc", max_batch=200)
        assert whole.shape == (n, 4736) and torch.equal(few.features(seq[:349 if n > 200 else None], raw_sequence=True), model("bf16_fc", max_batch=256).features(seq[:349 if n > 200 else None], raw_sequence=True))
        few.close()
    m.close()


def heads_of(count):
    """heads that differ: other seeds, and of another size"""
    out = []
    for i in range(count):
        sd = dict(synth.make_state_dict(10 + i, "uniform"))
        sd["fc.6.bias"] = sd["fc.6.bias"] + np.float32(i)
        out.append(sd)
    return out


@pytest.mark.parametrize("precision", ["bf16_fc", "fp8_fc"])
@pytest.mark.parametrize("n, count", [(1, 1), (7, 3), (300, 4), (900, 2)])
def test_bank(n, count, precision):
    base, heads = synth.make_state_dict(1, "uniform"), heads_of(count)
    bank = contact_bank(device=0, max_batch=1024, precision=precision).load_state_dict(base, heads)
    assert len(bank) == count
    x = windows(n, n)
    head = torch.randint(0, count, (n,), generator=torch.Generator().manual_seed(n)).to(torch.int32)
    if n > 5:
        head[3], head[4] = -1, count
    out = bank.predict(x, head.cuda())
    feat = bank._conv.features(x)
    for i, sd in enumerate(heads):
        mine = (head == i).nonzero()[:, 0].cuda()
        if len(mine):
            want, err = chain(feat[mine], sd, precision == "fp8_fc", False)
            assert ((out["logits"][mine].double() - want).abs() <= err).all(), i
    none = ((head < 0) | (head >= count)).cuda()
    assert torch.isnan(out["logits"][none]).all() and (out["pred"][none] == 0).all() and not torch.isnan(out["logits"][~none]).any()
    assert torch.equal(out["pred"][~none], out["logits"][~none].max(1)[1].int()) and torch.equal(out["contacts"].long(), bits(out))
    host = bank.predict(x.cpu().numpy(), head.numpy())
    assert np.array_equal(host["logits"], out["logits"].cpu().numpy(), equal_nan=True)


def test_bank_of_one_head_is_the_model():
    """the checkpoint's own head: the bank differs from contact_cnn by its roundings alone"""
    sd = synth.make_state_dict(1, "uniform")
    bank = contact_bank(device=0, max_batch=512).load_state_dict(sd, [sd])
    m = model("bf16_fc", max_batch=512)
    seq = torch.from_numpy(synth.make_sequence(400, 3).astype(np.float32)).cuda()
    got = bank.infer_sequence(seq, torch.zeros(251, dtype=torch.int64, device="cuda"))["logits"].double()
    want, err = chain(bank._conv.features(seq, raw_sequence=True), sd, False, False)
    assert ((got - want).abs() <= err).all()
    assert ((m.infer_sequence(seq)["logits"].double() - want).abs() <= err).all()
    m.close()


@pytest.mark.parametrize("precision", ["bf16_fc", "fp8_fc"])
def test_bank_on_another_stream_and_in_a_graph(precision):
    """windows and heads replaced in place, eager calls in between; more windows than max_batch, heads outside the bank"""
    sd = synth.make_state_dict(1, "uniform")
    b = contact_bank(device=0, precision=precision, max_batch=512).load_state_dict(sd, [synth.make_state_dict(i + 1, "uniform") for i in range(3)])
    g = torch.Generator(device="cuda").manual_seed(3)
    x, head = torch.randn(700, 150, 54, generator=g, device="cuda"), torch.randint(-1, 4, (700,), generator=g, device="cuda", dtype=torch.int32)

    def same(got, want):
        return all(torch.equal(torch.nan_to_num(got[k].float()), torch.nan_to_num(want[k].float())) for k in want)
    want = b.predict(x, head)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = b.predict(x, head)
    side.synchronize()
    assert same(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = b.predict(x, head)
    for _ in range(3):
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        head.copy_(torch.randint(-1, 4, (700,), generator=g, device="cuda", dtype=torch.int32))
        want = b.predict(x, head)
        graph.replay()
        torch.cuda.synchronize()
        assert same(out, want)
    b._conv.close()
