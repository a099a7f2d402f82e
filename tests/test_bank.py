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
