"""The matrix products of the FC layers as operators of their own, on CUDA tensors (include/dce.h: dce_quantize, dce_matmul,
dce_group_rows, dce_decide).

    q, s = quantize(x)                                    # activations: e4m3 and a power of two for every 128 values of a row
    wq, ws = quantize(w, rows=128)                        # weights: ... for every 128 x 128 block
    y = matmul_fp8(q, s, wq, ws, bias=b, relu=True)       # relu(x @ w.T + b); out_dtype=torch.float8_e4m3fn -> (q, s) again

    offsets, order, place = group_rows(head_of_window, heads)       # a weight matrix for each group of rows
    y = matmul_grouped(x, w, offsets, index=order, bias=b)          # w (heads, n, k); rows of y in the groups' order

Every call is queued on torch's current stream of its tensors' device, waits for nothing and keeps nothing; inputs that live on
another stream are the caller's to order (as with torch's own operators).  Calls may be captured into a graph.  There is no CPU path.
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _lib

BLOCK = 128
GROUPS_MAX = 1024
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu

_TYPES = {torch.float32: 0, torch.bfloat16: 1, E4M3: 2}


@functools.lru_cache(None)
def _entries():
    """The extension module with the entries (csrc/torch_entries.cpp), bound to the library."""
    lib = _lib.load()
    try:
        from . import _entries as e
    except ImportError as err:
        raise RuntimeError(f"{_lib.ENTRIES_PATH} does not load ({err}): build it with `python -m deep_contact_estimator_amd.build`") from err
    from .build import entries_abi
    if getattr(e, "ABI", None) != entries_abi():
        raise RuntimeError(f"{_lib.ENTRIES_PATH} was built for {getattr(e, 'ABI', 'another torch')}, this is {entries_abi()}: build it with `python -m deep_contact_estimator_amd.build`")
    address = lambda f: C.cast(f, C.c_void_p).value                # noqa: E731
    e.bind(*(address(f) for f in (lib.dce_quantize, lib.dce_matmul, lib.dce_group_rows, lib.dce_group_rows_work, lib.dce_decide, lib.dce_last_error)),
           torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (lambda device: 0), _lib.DceError)
    return e


def quantize(x, rows: int = 1, scale_dtype=E8M0):
    """x (m, k) fp32 | bf16 -> (q, scale): q (m, k) float8_e4m3fn, scale a power of two for every block: e is the smallest with
    max|x| <= 448 * 2^e (held inside [-126, 120]), q = x * 2^-e rounded once.  NaN and infinities become NaN and set no scale.

    rows = 1: blocks of 1 x 128 (activations), scale (ceil(k / 128), m).  rows = 128: blocks of 128 x 128 (weights; x may be
    (groups, n, k)), scale (.., ceil(n / 128), ceil(k / 128)).  scale_dtype: float8_e8m0fnu (the exponent's byte) or float32."""
    if scale_dtype is not E8M0 and scale_dtype is not torch.float32:
        raise RuntimeError(f"quantize: scale_dtype must be float8_e8m0fnu or float32, not {scale_dtype}")
    return _entries().quantize(x, rows, scale_dtype is E8M0)


def _out(what, dtype):
    code = _TYPES.get(dtype)
    if code is None:
        raise RuntimeError(f"{what}: results of {dtype}")
    return code


def matmul_fp8(a, a_scale, b, b_scale, bias=None, relu: bool = False, out_dtype=torch.bfloat16, out=None, out_scale=None):
    """act(a @ b.T + bias) of e4m3 operands: a (m, k) with a_scale (ceil(k / 128), m), b (n, k) with b_scale (ceil(n / 128),
    ceil(k / 128)), as quantize makes them, or float32 numbers of which the products of one of a and one of b are normal float32
    numbers or zero; bias (n,) float32; act = ReLU if relu.  Sums are fp32 and are rounded once to out_dtype: float32, bfloat16, or float8_e4m3fn -- then (q, scale) with a power of two for every 128 columns of a
    row, in the operands' scale dtype: the next product's a and a_scale.  For bfloat16 and float8_e4m3fn results the matrix instruction
    drops less than 2^-13 of the largest of eight products from each of the others: sums are off by up to 7 * 2^-13 of the sum of
    their products' magnitudes, 1.5e-5 of a result on random operands; where products cancel, more of it, and an e4m3 scale may
    follow (include/dce.h).  An operand's value that is no normal float32 number may count as infinite or as zero.  out may lie
    beside a and b in one tensor; out and out_scale overlap nothing that the call reads, nor each other.  Any sizes and row strides;
    rows that start at multiples of 16 bytes run fastest."""
    return _entries().matmul("matmul_fp8", a, a_scale, b, b_scale, bias, relu, _out("matmul_fp8", out_dtype), out, out_scale, None, None)


def matmul_grouped(a, b, offsets, index=None, a_scale=None, b_scale=None, bias=None, relu: bool = False, out_dtype=torch.bfloat16, out=None,
                   out_scale=None):
    """Row j of the result, offsets[g] <= j < offsets[g + 1], is act(a[index[j]] @ b[g].T + bias[g]) (a[j] without index): one weight
    matrix for each group of rows, however the rows fall.  a (rows, k) and b (groups, n, k) both bfloat16, or both float8_e4m3fn with
    a_scale (ceil(k / 128), rows) and b_scale (groups, ceil(n / 128), ceil(k / 128)); bias (groups, n) float32; offsets (groups + 1)
    int32, never falling, and index int32 on the device, as group_rows makes them: nothing is read back.  An index outside a reads as
    a row of zeros; rows that no group covers stay as they were in `out` (in a fresh result they hold nothing of use)."""
    if offsets is None:
        raise RuntimeError("matmul_grouped: offsets must be int32 (groups + 1,), got None")
    return _entries().matmul("matmul_grouped", a, a_scale, b, b_scale, bias, relu, _out("matmul_grouped", out_dtype), out, out_scale, offsets, index)


def group_rows(ids, groups: int):
    """ids (n,) int32 | int64 -> (offsets (groups + 1), order (n), place (n)), int32: order[j] is the row at place j, rows of a group in
    their own order (-1 behind the last group), place[i] the place of row i (-1 where the id is outside [0, groups))."""
    return _entries().group_rows(ids, groups)


def decide(logits, index=None):
    """(rows, 16) float32 logits, picked by index (n,) int32 -> dict(logits (n, 16), pred (n,) int32, contacts (n, 4) uint8), as
    contact_cnn.predict returns them; an index outside the rows gives NaN logits and class 0."""
    return _entries().decide(logits, index)
