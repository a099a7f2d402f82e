"""CPU: the operators of ops.py refuse what they cannot compute, before anything reaches a device; what their descriptors look like to C."""
import ctypes as C
import os
import re
import struct

import pytest

torch = pytest.importorskip("torch")
QUANTIZE = struct.Struct("=QqqQqqQqqqqiiii")                       # the descriptors as a C caller packs them
MATMUL = struct.Struct("=QqQqQqqQqqQqQqQqQQqqqqiiiiii")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from deep_contact_estimator_amd import _lib, build
    if not os.path.exists(build.LIB):
        build.build()
    return _lib.load()


def _fields(name):
    """(type, field) of a descriptor of include/dce.h, in order"""
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "dce.h")).read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
    found = []
    for kind, names in re.findall(r"(const void\*|const float\*|const int32_t\*|void\*|uint8_t\*|int64_t|int32_t)\s+([^;]+);", body):
        found += [(kind, n.strip()) for n in names.split(",")]
    return found


@pytest.mark.parametrize("name, packed", [("dce_quantize_desc", QUANTIZE), ("dce_matmul_desc", MATMUL)])
def test_descriptors_match_the_header(name, packed):
    fields = _fields(name)
    codes = "".join("Q" if k.endswith("*") else "q" if k == "int64_t" else "i" for k, _ in fields)
    assert packed.format == "=" + codes
    kinds = {"Q": C.c_void_p, "q": C.c_int64, "i": C.c_int32}
    struct_type = type(name, (C.Structure,), {"_fields_": [(f, kinds[c]) for (_, f), c in zip(fields, codes)]})
    assert C.sizeof(struct_type) == packed.size            # no padding between the fields


def _quantize(**kw):
    d = dict(x=4096, ldx=256, x_batch=0, q=8192, ldq=256, q_batch=0, scale=1024, ld_scale=4, batch=1, rows=4, k=256, x_type=0, scale_type=0, block_rows=1, reserved=0)
    d.update(kw)
    return QUANTIZE.pack(*d.values())


def _matmul(**kw):
    d = dict(a=4096, lda=256, a_scale=4096, ld_a_scale=4, b=4096, ldb=256, b_group=0, b_scale=4096, ld_b_scale=2, b_scale_group=0, bias=0, bias_group=0,
             y=1 << 24, ldy=64, y_scale=0, ld_y_scale=0, offsets=0, index=0, a_rows=4, m=4, n=64, k=256, groups=1, in_type=2, scale_type=0, out_type=0, relu=0, reserved=0)
    d.update(kw)
    return MATMUL.pack(*d.values())


@pytest.mark.parametrize("kw, word", [
    (dict(x_type=2), b"x must be"), (dict(scale_type=2), b"scale type"), (dict(block_rows=64), b"a block has"), (dict(rows=-1), b"out of range"),
    (dict(k=1 << 25), b"out of range"), (dict(batch=2), b"one matrix"), (dict(ldx=255), b"stride"), (dict(ldq=255), b"stride"), (dict(x=0), b"NULL"), (dict(q=0), b"NULL"),
    (dict(scale=0), b"NULL"), (dict(x=4098), b"aligned"), (dict(scale=1026, scale_type=1), b"aligned"), (dict(ld_scale=3), b"ld_scale"),
    (dict(batch=2, block_rows=128, q_batch=1000, rows=4), b"overlap"), (dict(ldx=1 << 50), b"stride"), (dict(ldq=1 << 50), b"stride"), (dict(x=8192), b"overlap")])
def test_quantize_refuses(lib, kw, word):
    assert lib.dce_quantize(0, None, _quantize(**kw)) == -1
    assert word in lib.dce_last_error(None)


@pytest.mark.parametrize("kw, word", [
    (dict(in_type=0), b"bf16 or e4m3"), (dict(out_type=3), b"result type"), (dict(in_type=1, out_type=2), b"e4m3 operands"), (dict(scale_type=7), b"scale type"),
    (dict(m=-1), b"out of range"), (dict(n=1 << 25), b"out of range"), (dict(k=1 << 25), b"out of range"), (dict(m=1 << 31, a_rows=1 << 31), b"out of range"),
    (dict(groups=0), b"groups"), (dict(groups=1025, offsets=64), b"groups"), (dict(groups=2), b"offsets"), (dict(a_rows=3), b"rows"), (dict(lda=255), b"stride"), (dict(ldb=255), b"stride"),
    (dict(ldy=63), b"stride"), (dict(a=0), b"NULL"), (dict(b=0), b"NULL"), (dict(y=0), b"NULL"), (dict(a_scale=0), b"a_scale"), (dict(b_scale=0), b"a_scale"),
    (dict(ld_a_scale=3), b"scale"), (dict(ld_b_scale=1), b"scale"), (dict(out_type=2), b"y_scale"), (dict(out_type=2, y_scale=64, ld_y_scale=3), b"y_scale"),
    (dict(y=8194), b"aligned"), (dict(bias=4097), b"aligned"), (dict(in_type=1, a=4097), b"aligned"), (dict(scale_type=1, a_scale=4098), b"aligned"),
    (dict(groups=2, offsets=64, b_group=-1), b"negative"), (dict(groups=2, offsets=64, b_group=1 << 50), b"group stride"), (dict(lda=1 << 50), b"row stride"), (dict(ldb=1 << 50), b"row stride"),
    (dict(ldy=1 << 50), b"row stride"), (dict(a=1 << 20, y=1 << 20), b"overlaps"), (dict(b=1 << 20, y=(1 << 20) + 64 * 256 - 4), b"overlaps"),
    (dict(a=1 << 20, y=(1 << 20) - 4 * 64 * 4 + 4), b"overlaps"), (dict(groups=3, offsets=64, b=1 << 20, b_group=1 << 16, y=(1 << 20) + (2 << 16)), b"overlaps")])
def test_matmul_refuses(lib, kw, word):
    assert lib.dce_matmul(0, None, _matmul(**kw)) == -1
    assert word in lib.dce_last_error(None)


def test_empty_calls_touch_nothing(lib):
    assert lib.dce_quantize(0, None, _quantize(rows=0, x=0, q=0, scale=0)) == 0
    assert lib.dce_quantize(0, None, _quantize(k=0, x=0, q=0, scale=0)) == 0
    assert lib.dce_matmul(0, None, _matmul(m=0, a_rows=0, a=0, y=0, a_scale=0)) == 0
    assert lib.dce_matmul(0, None, _matmul(n=0, b=0, y=0)) == 0
    assert lib.dce_decide(0, None, None, 0, None, 0, None, None, None) == 0


def test_overlap_is_found_where_it_is(lib):
    """every place of y around a, against the bytes themselves: the same stride, and either one without gaps"""
    if lib.dce_device_count() > 0:
        pytest.skip("GPU present: the calls that are not refused would run")
    base = 1 << 20
    for lda, ldy, k, n, rows in ((24, 24, 8, 6, 3), (8, 24, 8, 6, 3), (24, 6, 8, 6, 3), (8, 6, 8, 6, 4), (20, 20, 8, 8, 1)):
        a = {base + 2 * (i * lda + j) + u for i in range(rows) for j in range(k) for u in (0, 1)}
        for d in range(-100, 101):
            at = base + 2 * d
            y = {at + 2 * (i * ldy + j) + u for i in range(rows) for j in range(n) for u in (0, 1)}
            desc = _matmul(a=base, lda=lda, b=64, ldb=k, y=at, ldy=ldy, a_rows=rows, m=rows, n=n, k=k, in_type=1, out_type=1, a_scale=0, b_scale=0)
            refused = lib.dce_matmul(0, None, desc) == -1
            assert refused == bool(a & y), (lda, ldy, d, lib.dce_last_error(None))


def test_null_descriptors_and_grouping_refusals(lib):
    assert lib.dce_quantize(0, None, None) == -1 and lib.dce_matmul(0, None, None) == -1
    assert lib.dce_group_rows_work(-1, 4) == -1 and lib.dce_group_rows_work(10, 0) == -1 and lib.dce_group_rows_work(10, 1025) == -1
    assert lib.dce_group_rows_work(100, 64) == 0 and lib.dce_group_rows_work(1 << 30, 1024) > 0
    p = C.c_void_p(4096)
    assert lib.dce_group_rows(0, None, p, 2, 10, 4, p, p, p, None) == -1
    assert lib.dce_group_rows(0, None, None, 4, 10, 4, p, p, p, None) == -1
    assert lib.dce_group_rows(0, None, p, 4, 10, 4, None, p, p, None) == -1
    assert lib.dce_group_rows(0, None, p, 4, 1 << 20, 4, p, p, p, None) == -1 and b"workspace" in lib.dce_last_error(None)
    assert lib.dce_group_rows(0, None, C.c_void_p(4100), 8, 10, 4, p, p, p, None) == -1 and b"aligned" in lib.dce_last_error(None)
    assert lib.dce_decide(0, None, p, 3, None, 4, None, p, None) == -1
    assert lib.dce_decide(0, None, None, 3, p, 4, None, p, None) == -1


def test_a_call_without_a_device_says_so(lib):
    if lib.dce_device_count() > 0:
        pytest.skip("GPU present")
    assert lib.dce_quantize(0, None, _quantize()) == -2 and b"no CPU fallback" in lib.dce_last_error(None)
    assert lib.dce_matmul(0, None, _matmul()) == -2 and b"no CPU fallback" in lib.dce_last_error(None)


def test_python_refuses_cpu_tensors_and_wrong_types():
    from deep_contact_estimator_amd import ops
    x = torch.zeros(4, 256)
    f8 = x.to(torch.float8_e4m3fn)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.quantize(x)
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        ops.quantize(x.double())
    with pytest.raises(RuntimeError, match="1 row"):
        ops.quantize(x, rows=64)
    with pytest.raises(RuntimeError, match="scale_dtype"):
        ops.quantize(x, scale_dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="expected"):
        ops.quantize(x[None])
    with pytest.raises(RuntimeError, match="both be"):
        ops.matmul_fp8(f8, None, x, None)
    with pytest.raises(RuntimeError, match="results of"):
        ops.matmul_grouped(x.bfloat16(), x.bfloat16()[None], torch.zeros(2, dtype=torch.int32), out_dtype=torch.float8_e4m3fn)
    with pytest.raises(RuntimeError, match="offsets"):
        ops.matmul_grouped(x.bfloat16(), x.bfloat16()[None], torch.zeros(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="groups, n, k"):
        ops.matmul_grouped(x.bfloat16(), x.bfloat16(), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="index"):
        ops.matmul_grouped(x.bfloat16(), x.bfloat16()[None], torch.zeros(2, dtype=torch.int32), index=torch.zeros(2))
    with pytest.raises(RuntimeError, match="ids"):
        ops.group_rows(torch.zeros(3), 2)
    with pytest.raises(RuntimeError, match="groups"):
        ops.group_rows(torch.zeros(3, dtype=torch.int32), 0)
    with pytest.raises(RuntimeError, match="logits"):
        ops.decide(torch.zeros(3, 15))
