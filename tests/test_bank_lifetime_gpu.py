"""GPU: a bank's weights stay where they are until every stream that was given work on them is through with it."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from deep_contact_estimator_amd import contact_bank, synth   # noqa: E402


@pytest.mark.parametrize("precision", ["bf16_fc", "fp8_fc"])
def test_reload_while_another_stream_still_works(precision):
    """weights staged on one stream, a call queued on another behind a long wait, new heads loaded meanwhile, and the memory that they gave back, if any, filled
    with NaN: the queued call's results are those of its own heads"""
    sd = synth.make_state_dict(1, "uniform")
    heads = [synth.make_state_dict(i + 1, "uniform") for i in range(3)]
    bank = contact_bank(device=0, precision=precision, max_batch=64).load_state_dict(sd, heads)
    g = torch.Generator(device="cuda").manual_seed(1)
    x, head = torch.randn(60, 150, 54, generator=g, device="cuda"), torch.randint(0, 3, (60,), generator=g, device="cuda", dtype=torch.int32)
    want = bank.predict(x, head)["logits"].clone()
    sizes = [(t.numel(), t.dtype) for layer in bank._layers[1] for t in layer if t is not None]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)                              # (about a tenth of a second)
        got = bank.predict(x, head)["logits"]
    bank.load_state_dict(sd, heads[::-1])
    junk = [torch.empty(n, dtype=torch.uint8 if kind.itemsize == 1 else kind, device="cuda") for n, kind in sizes for _ in range(2)]
    for t in junk:
        t.fill_(0x7f if t.dtype == torch.uint8 else float("nan"))
    side.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    assert torch.equal(bank.predict(x, 2 - head)["logits"], want)
    bank._conv.close()


def test_the_first_call_on_another_stream_finds_the_weights_whole():
    sd = synth.make_state_dict(1, "uniform")
    x, head = torch.randn(5, 150, 54, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda")
    bank = contact_bank(device=0, max_batch=8).load_state_dict(sd, [sd])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    out = []
    for s in streams:
        with torch.cuda.stream(s):
            out.append(bank.predict(x, head)["logits"])
    torch.cuda.synchronize()
    assert all(torch.equal(o, bank.predict(x, head)["logits"]) for o in out)
    assert len(bank._streams) == 4
    bank._conv.close()


def test_no_windows():
    sd = synth.make_state_dict(1, "uniform")
    bank = contact_bank(device=0, max_batch=8).load_state_dict(sd, [sd])
    for x in (torch.zeros(0, 150, 54), torch.zeros(0, 150, 54, device="cuda")):
        for head in ([], torch.zeros(0), torch.zeros(0, dtype=torch.int32, device="cuda")):
            out = bank.predict(x, head)
            assert out["logits"].shape == (0, 16) and out["pred"].shape == (0,) and out["contacts"].shape == (0, 4)
    bank._conv.close()
