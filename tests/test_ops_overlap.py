"""CPU: what the operators write may not lie where they read, in any argument; strides that no address space holds."""

import pytest

pytest.importorskip("torch")
from test_ops import _matmul, _quantize, lib   # noqa: E402, F401
import ctypes as C   # noqa: E402

MB = 1 << 20
# a square layer in e4m3: 256 rows of 256, scales (2, 256), every argument a megabyte of its own
E4M3 = dict(a=1 * MB, lda=256, a_scale=2 * MB, ld_a_scale=256, b=3 * MB, ldb=256, b_scale=4 * MB, ld_b_scale=2, bias=5 * MB, y=6 * MB, ldy=256, y_scale=7 * MB, ld_y_scale=256,
            offsets=8 * MB, index=9 * MB, a_rows=256, m=256, n=256, k=256, groups=1, in_type=2, scale_type=0, out_type=2)


def answer(lib, call, desc):   # noqa: F811
    rc = call(0, None, desc)
    return rc, lib.dce_last_error(None) if rc else b""


def accepted(lib, call, desc):   # noqa: F811
    """not refused: without a device such a call ends at the device"""
    rc, said = answer(lib, call, desc)
    return rc == -2 and b"no CPU fallback" in said


@pytest.fixture
def no_gpu(lib):   # noqa: F811
    if lib.dce_device_count() > 0:
        pytest.skip("GPU present: the calls that are not refused would run")


@pytest.mark.parametrize("scale_type", [0, 1])
@pytest.mark.parametrize("what", ["a", "a_scale", "b", "b_scale", "bias", "offsets", "index"])
@pytest.mark.parametrize("written", ["y", "y_scale"])
def test_matmul_results_on_what_it_reads(lib, no_gpu, what, written, scale_type):   # noqa: F811
    d = dict(E4M3, scale_type=scale_type)
    assert accepted(lib, lib.dce_matmul, _matmul(**d))
    ss = 4 if scale_type else 1
    size = {"a": 65536, "b": 65536, "a_scale": 512 * ss, "b_scale": 4 * ss, "bias": 1024, "offsets": 8, "index": 1024, "y": 65536, "y_scale": 512 * ss}
    for at in (0, size[what] - 4, 4 - size[written]):                  # at its start, at its last bytes, with its own last bytes at its start
        rc, said = answer(lib, lib.dce_matmul, _matmul(**{**d, written: d[what] + at}))
        assert rc == -1 and b"overlaps" in said, (what, written, at)
    for at in (size[what], -size[written]):                            # beside it
        assert accepted(lib, lib.dce_matmul, _matmul(**{**d, written: d[what] + at})), (what, written, at)


def test_matmul_results_on_each_other(lib, no_gpu):   # noqa: F811
    for at in (0, 65532, -508):
        rc, said = answer(lib, lib.dce_matmul, _matmul(**{**E4M3, "y_scale": E4M3["y"] + at}))
        assert rc == -1 and b"overlaps" in said, at
    for at in (65536, -512):
        assert accepted(lib, lib.dce_matmul, _matmul(**{**E4M3, "y_scale": E4M3["y"] + at}))
    # y_scale has no part in other results
    assert accepted(lib, lib.dce_matmul, _matmul(**{**E4M3, "out_type": 1, "y_scale": E4M3["a_scale"]}))
    assert accepted(lib, lib.dce_matmul, _matmul(**{**E4M3, "k": 0, "y_scale": E4M3["a_scale"]}))


def test_matmul_groups(lib, no_gpu):   # noqa: F811
    """the scales and biases of every group; one that all groups share"""
    d = dict(E4M3, groups=5, b_group=65536, b_scale_group=64, bias_group=512, b=16 * MB)
    assert accepted(lib, lib.dce_matmul, _matmul(**d))
    for what, at in (("b_scale", 4 * 64), ("b_scale", 4 * 64 + 3), ("bias", 4 * 2048), ("bias", 4 * 2048 + 1020), ("b", 4 * 65536 + 65532)):
        rc, said = answer(lib, lib.dce_matmul, _matmul(**{**d, "y_scale": d[what] + at}))
        assert rc == -1 and b"overlaps" in said, (what, at)
    assert accepted(lib, lib.dce_matmul, _matmul(**{**d, "y_scale": d["b_scale"] + 4 * 64 + 4}))
    shared = dict(d, b_group=0, b_scale_group=0, bias_group=0)
    assert accepted(lib, lib.dce_matmul, _matmul(**shared))
    assert accepted(lib, lib.dce_matmul, _matmul(**{**shared, "y_scale": d["bias"] + 1024}))
    rc, said = answer(lib, lib.dce_matmul, _matmul(**{**shared, "y_scale": d["bias"] + 1020}))
    assert rc == -1 and b"overlaps" in said


@pytest.mark.parametrize("kw", [dict(ld_a_scale=1 << 50), dict(ld_b_scale=1 << 50), dict(ld_y_scale=1 << 50), dict(groups=2, bias_group=1 << 60), dict(groups=2, b_scale_group=1 << 60)])
def test_matmul_strides_without_end(lib, kw):   # noqa: F811
    rc, said = answer(lib, lib.dce_matmul, _matmul(**{**E4M3, **kw}))
    assert rc == -1 and b"out of range" in said


QUANT = dict(x=1 * MB, ldx=256, q=2 * MB, ldq=256, scale=3 * MB, ld_scale=4, rows=4, k=256, x_type=0, scale_type=0)


def test_quantize_scales_and_matrices(lib, no_gpu):   # noqa: F811
    assert accepted(lib, lib.dce_quantize, _quantize(**QUANT))
    for what, size in (("x", 4096), ("q", 1024)):
        for at in (0, size - 1, -7):
            rc, said = answer(lib, lib.dce_quantize, _quantize(**{**QUANT, "scale": QUANT[what] + at}))
            assert rc == -1 and b"overlap" in said, (what, at)
        assert accepted(lib, lib.dce_quantize, _quantize(**{**QUANT, "scale": QUANT[what] + size}))
        assert accepted(lib, lib.dce_quantize, _quantize(**{**QUANT, "scale": QUANT[what] - 8}))
    # several matrices: 3 of 4 x 256, fp32 4096 bytes, e4m3 1024
    many = dict(QUANT, batch=3, block_rows=128, x_batch=1024, q_batch=1024)
    assert accepted(lib, lib.dce_quantize, _quantize(**many))
    for kw in (dict(q=MB), dict(q=MB + 2 * 4096), dict(q=MB - 3 * 1024 + 1), dict(scale=MB + 3 * 4096 - 1), dict(scale=2 * MB + 3 * 1024 - 1), dict(scale=2 * MB - 5)):
        rc, said = answer(lib, lib.dce_quantize, _quantize(**{**many, **kw}))
        assert rc == -1 and b"overlap" in said, kw
    assert accepted(lib, lib.dce_quantize, _quantize(**{**many, "q": MB - 3 * 1024})) and accepted(lib, lib.dce_quantize, _quantize(**{**many, "q": MB + 3 * 4096}))
    # q in the gaps of x: 4096 bytes of every 8192
    gaps = dict(many, x_batch=2048, q_batch=8192, q=MB + 4096, scale=3 * MB)
    assert accepted(lib, lib.dce_quantize, _quantize(**gaps))
    assert answer(lib, lib.dce_quantize, _quantize(**{**gaps, "q": MB + 4095}))[0] == -1
    for kw in (dict(x_batch=1 << 60), dict(q_batch=1 << 60), dict(block_rows=1, batch=1, ld_scale=1 << 60)):
        rc, said = answer(lib, lib.dce_quantize, _quantize(**{**many, **kw}))
        assert rc == -1 and b"out of range" in said, kw


def test_group_rows(lib, no_gpu):   # noqa: F811
    n, groups = 1 << 20, 4
    at = dict(ids=16 * MB, offsets=96 * MB, order=32 * MB, place=48 * MB, work=64 * MB)
    work = lib.dce_group_rows_work(n, groups)
    size = dict(ids=4 * n, offsets=4 * (groups + 1), order=4 * n, place=4 * n, work=4 * work)

    def call(**kw):
        p = {k: C.c_void_p(v) for k, v in {**at, **kw}.items()}
        return lib.dce_group_rows(0, None, p["ids"], 4, n, groups, p["offsets"], p["order"], p["place"], p["work"]), lib.dce_last_error(None)
    assert work > 0 and call()[0] == -2
    for one in at:
        for other in at:
            if one != other:
                for where in (at[other], at[other] + size[other] - 4, at[other] - size[one] + 4):
                    rc, said = call(**{one: where})
                    assert rc == -1 and b"overlap" in said, (one, other)
                assert call(**{one: at[other] + size[other]})[0] == -2, (one, other)


def test_decide(lib, no_gpu):   # noqa: F811
    n, rows = 100, 60
    at = dict(logits=1 * MB, index=2 * MB, out=3 * MB, pred=4 * MB, contacts=5 * MB)
    size = dict(logits=64 * rows, index=4 * n, out=64 * n, pred=4 * n, contacts=4 * n)

    def call(**kw):
        p = {k: C.c_void_p(v) if v else None for k, v in {**at, **kw}.items()}
        return lib.dce_decide(0, None, p["logits"], rows, p["index"], n if p["index"] else rows, p["out"], p["pred"], p["contacts"]), lib.dce_last_error(None)
    assert call()[0] == -2
    for one in ("out", "pred", "contacts"):
        for other in at:
            if one != other:
                for where in (at[other], at[other] + size[other] - 4, at[other] - size[one] + 4):
                    rc, said = call(**{one: where})
                    assert rc == -1 and b"overlap" in said, (one, other)
                assert call(**{one: at[other] + size[other]})[0] == -2
    assert call(out=at["logits"], index=0)[0] == -2                   # in place, row for row
    assert call(out=at["logits"] + 64, index=0)[0] == -1


def test_many_matrices_are_looked_through_quickly(lib, no_gpu):   # noqa: F811
    """65535 matrices of x and as many of q between them: no pair of them all is compared with every other"""
    import time
    d = dict(x=1 << 30, ldx=64, x_batch=4096, q=(1 << 30) + 4096, ldq=64, q_batch=16384, scale=1 << 40, batch=65535, rows=16, k=64, block_rows=128, x_type=0, scale_type=0)
    at = time.monotonic()
    assert accepted(lib, lib.dce_quantize, _quantize(**d))
    assert answer(lib, lib.dce_quantize, _quantize(**{**d, "q": d["q"] - 1}))[0] == -1           # the last byte of every matrix of x
    last = {**d, "q": d["x"] + 65534 * 16384 + 4095}                    # ... of the last one alone
    assert answer(lib, lib.dce_quantize, _quantize(**last))[0] == -1
    assert accepted(lib, lib.dce_quantize, _quantize(**{**last, "q": last["q"] + 1}))
    assert time.monotonic() - at < 2
