"""GPU: the largest sizes that the argument checks allow: a launch holds fewer than 2^32 threads, and a call has to run or be refused in words."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from deep_contact_estimator_amd import _lib, ops   # noqa: E402


@pytest.mark.parametrize("n", [(1 << 24) - 3, (1 << 24) + 5, (1 << 28) + 1])
def test_decide(n):
    """classes of more rows than a launch has sixteenths of threads (17 million rows: workgroups take more than one set of sixteen)"""
    lib = _lib.load()
    logits = torch.zeros(16, 16, device="cuda")
    logits[torch.arange(16), (torch.arange(16) * 5 + 3) % 16] = 1.0
    index = torch.arange(n, dtype=torch.int32, device="cuda").remainder_(17)             # (16: outside)
    pred = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    _lib.check(lib.dce_decide(0, None, logits.data_ptr(), 16, index.data_ptr(), n, None, pred.data_ptr(), None))
    torch.cuda.synchronize()
    for lo in range(0, n, 1 << 24):
        part = index[lo:lo + (1 << 24)]
        assert torch.equal(pred[lo:lo + (1 << 24)], torch.where(part < 16, (part * 5 + 3) % 16, 0))


@pytest.mark.parametrize("k", [16, 5])
@pytest.mark.parametrize("m", [((1 << 23) - 9) * 128, (1 << 30) - 128, 1 << 30])
def test_a_product_of_as_many_rows_as_there_may_be(m, k):
    """a billion gathered rows, one column.  Rows at any address go in tiles of 128 x 128, 512 threads each: m / 128 of them, one more for the group's last
    rows, rounded up to eight, have to be fewer than 2^23: (2^23 - 9) + 1 = 2^23 - 8 are; (2^30 - 128) / 128 + 1 = 2^23 are not, and are refused."""
    a = torch.arange(3 * k, device="cuda").view(3, k).bfloat16()
    w, offsets = torch.ones(1, 1, k, dtype=torch.bfloat16, device="cuda"), torch.tensor([0, m], dtype=torch.int64, device="cuda").int()
    index = torch.arange(m, dtype=torch.int32, device="cuda").remainder_(3)
    if k == 5 and m > ((1 << 23) - 9) * 128:
        with pytest.raises(RuntimeError, match="more tiles than a launch has"):
            ops.matmul_grouped(a, w, offsets, index=index)
        return
    y = ops.matmul_grouped(a, w, offsets, index=index)
    want = a.float().sum(1).bfloat16()
    for lo in range(0, m, 1 << 26):
        assert torch.equal(y[lo:lo + (1 << 26), 0], want[index[lo:lo + (1 << 26)].long()])


def test_offsets_that_fall_again_and_again():
    """0, m, 0, m, ..: 512 groups of all m rows each, more tiles than 32 bits count.  The launch is as large as m rows need: what it computes is right and
    what it does not is left alone, and nothing is written beside the result"""
    m, groups, k = 1 << 28, 1024, 16
    a = torch.arange(2 * k, device="cuda").view(2, k).bfloat16()
    w = torch.ones(groups, 1, k, dtype=torch.bfloat16, device="cuda")
    offsets = (torch.arange(groups + 1, device="cuda") % 2 * m).int()
    index = torch.arange(m, dtype=torch.int32, device="cuda").remainder_(2)
    big = torch.full((m + 512, 1), 9.0, dtype=torch.bfloat16, device="cuda")
    ops.matmul_grouped(a, w, offsets, index=index, out=big[256:256 + m])
    want = a.float().sum(1).bfloat16()
    assert (big[:256] == 9).all() and (big[256 + m:] == 9).all()
    for lo in range(0, m, 1 << 26):
        y = big[256 + lo:256 + lo + (1 << 26), 0]
        assert ((y == want[index[lo:lo + (1 << 26)].long()]) | (y == 9)).all()
