"""CPU: what contact_bank refuses before anything reaches a device."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("head", [np.zeros(2), np.array([-0.5, 0.9]), torch.tensor([0.0, 1.0]), torch.tensor([-0.5, 0.9]).bfloat16(), torch.zeros(2, dtype=torch.complex64)])
def test_heads_are_whole_numbers(head):
    from deep_contact_estimator_amd import contact_bank
    bank = contact_bank(max_batch=4)
    for x in (np.zeros((2, 150, 54), np.float32), torch.zeros(2, 150, 54)):
        with pytest.raises(RuntimeError, match="whole numbers"):
            bank.predict(x, head)
    with pytest.raises(RuntimeError, match="whole numbers"):
        bank.infer_sequence(np.zeros((151, 54), np.float32), head)


def test_no_windows_and_no_heads():
    """an empty list, which numpy takes for floats, is no wrong type: the call ends where a call without a device ends"""
    from deep_contact_estimator_amd import _lib, contact_bank, synth
    if _lib.load().dce_device_count() > 0:
        pytest.skip("GPU present")
    bank = contact_bank(max_batch=4).load_state_dict(synth.make_state_dict(1), [synth.make_state_dict(1)])
    for head in ([], np.zeros(0), torch.zeros(0)):
        with pytest.raises(RuntimeError, match="no HIP device|no CPU"):
            bank.predict(np.zeros((0, 150, 54), np.float32), head)


@pytest.mark.parametrize("kind", ["numpy", "torch"])
def test_loaded_weights_are_the_callers_no_longer(kind):
    """arrays that change after load_state_dict (a training loop's parameters) change neither the model nor the bank, whose weights go up with the first call"""
    from deep_contact_estimator_amd import contact_bank, contact_cnn, synth
    sd = {k: np.array(v) for k, v in synth.make_state_dict(1).items()}
    want = {k: v.copy() for k, v in sd.items()}
    given = {k: torch.from_numpy(v) for k, v in sd.items()} if kind == "torch" else sd
    model = contact_cnn(max_batch=4)
    model.load_state_dict(given)
    bank = contact_bank(max_batch=4).load_state_dict(given, [given, given])
    for v in sd.values():
        v += 1
    for held in (model.state_dict(), bank._conv.state_dict()):
        assert all(np.array_equal(held[k], want[k]) for k in want)
    for head in bank._heads:
        assert head and all(np.array_equal(head[k], want[k]) for k in head)
