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
import struct

import torch

from . import _lib

BLOCK = 128
GROUPS_MAX = 1024
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu

_TYPES = {torch.float32: 0, torch.bfloat16: 1, E4M3: 2}
_SCALES = {E8M0: 0, torch.float32: 1}
_QUANTIZE = struct.Struct("=QqqQqqQqqqqiiii")                      # dce_quantize_desc
_MATMUL = struct.Struct("=QqQqQqqQqqQqQqQqQQqqqqiiiiii")           # dce_matmul_desc
_entries = None


def _lib_entries():
    global _entries
    if _entries is None:
        lib = _lib.load()
        _entries = (lib.dce_quantize, lib.dce_matmul, lib.dce_group_rows, lib.dce_group_rows_work, lib.dce_decide)
    return _entries


_grad_on, _raw_stream = torch.is_grad_enabled, torch._C._cuda_getCurrentRawStream


def _at(t, what):
    """The device of a call's first tensor."""
    dev = t.get_device()
    if dev < 0:
        raise RuntimeError(f"{what}: deep_contact_estimator_amd runs on MI355X only; there is no CPU path (got a tensor on {t.device})")
    return dev


def _same(dev, what, *tensors):
    """... is that of the others too, and none wants a gradient."""
    grad = _grad_on()
    for t in tensors:
        if t is not None:
            if t.get_device() != dev:
                raise RuntimeError(f"{what}: tensors on cuda:{dev} and on {t.device}")
            if grad and t.requires_grad:
                raise RuntimeError(f"{what}: deep_contact_estimator_amd implements the inference path only: detach the tensor, or call under torch.no_grad()")


def _rowed(t):
    """`t` with its last axis without gaps and rows that do not overlap -- itself where it is so already -- and its strides (of an axis of one
    entry, whose stride says nothing, what a matrix without gaps has)."""
    st, shape = t.stride(), t.shape
    n = shape[-1]
    if (st[-1] == 1 or n <= 1) and (st[-2] >= n or shape[-2] <= 1):
        if shape[-2] > 1:
            return t, st
        return t, (*st[:-2], max(n, 1), 1)
    t = t.contiguous()
    return t, t.stride()


def _vector(t):
    return t if t.is_contiguous() else t.contiguous()


def _check(rc):
    if rc:
        _lib.check(rc, None)


def quantize(x, rows: int = 1, scale_dtype=E8M0):
    """x (m, k) fp32 | bf16 -> (q, scale): q (m, k) float8_e4m3fn, scale a power of two for every block: e is the smallest with
    max|x| <= 448 * 2^e (held inside [-126, 120]), q = x * 2^-e rounded once.  NaN and infinities become NaN and set no scale.

    rows = 1: blocks of 1 x 128 (activations), scale (ceil(k / 128), m).  rows = 128: blocks of 128 x 128 (weights; x may be
    (groups, n, k)), scale (.., ceil(n / 128), ceil(k / 128)).  scale_dtype: float8_e8m0fnu (the exponent's byte) or float32."""
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise RuntimeError(f"quantize: x must be float32 or bfloat16, not {x.dtype}")
    if scale_dtype not in _SCALES:
        raise RuntimeError(f"quantize: scale_dtype must be float8_e8m0fnu or float32, not {scale_dtype}")
    if rows not in (1, BLOCK):
        raise RuntimeError(f"quantize: a block has 1 row or {BLOCK}, not {rows}")
    dims = x.dim()
    if dims != 2 and (rows == 1 or dims != 3):
        raise RuntimeError(f"quantize: expected (m, k){' or (groups, n, k)' if rows != 1 else ''}, got {tuple(x.shape)}")
    dev = _at(x, "quantize")
    _same(dev, "quantize", x)
    x, st = _rowed(x)
    shape = x.shape
    m, k = shape[-2:]
    kb = (k + 127) // 128
    at = x.device
    q = torch.empty(shape, dtype=E4M3, device=at)
    if rows == 1:
        scale = torch.empty((kb, m), dtype=scale_dtype, device=at)
    else:
        scale = torch.empty((*shape[:-2], (m + 127) // 128, kb), dtype=scale_dtype, device=at)
    rc = _lib_entries()[0](dev, _raw_stream(dev), _QUANTIZE.pack(
        x.data_ptr(), st[-2], st[0] if dims == 3 else 0, q.data_ptr(), k, m * k, scale.data_ptr(), m, shape[0] if dims == 3 else 1, m, k,
        _TYPES[x.dtype], _SCALES[scale_dtype], rows, 0))
    if rc:
        _check(rc)
    return q, scale


def _matmul(what, a, a_scale, b, b_scale, bias, relu, out_dtype, out, out_scale, offsets, index):
    kind = a.dtype
    f8 = kind == E4M3
    if b.dtype != kind or not (f8 or kind == torch.bfloat16):
        raise RuntimeError(f"{what}: operands must both be bfloat16 or float8_e4m3fn, not {kind} and {b.dtype}")
    out_type = _TYPES.get(out_dtype)
    if out_type is None or (out_type == 2 and not f8):
        raise RuntimeError(f"{what}: results of {out_dtype} from {kind}")
    dev = _at(a, what)
    _same(dev, what, a, b, a_scale, b_scale, bias, out, out_scale, offsets, index)
    grouped = offsets is not None
    if a.dim() != 2 or b.dim() != 2 + grouped:
        raise RuntimeError(f"{what}: expected a (rows, k) and b ({'groups, ' if grouped else ''}n, k), got {tuple(a.shape)} and {tuple(b.shape)}")
    a, sa = _rowed(a)
    b, sb = _rowed(b)
    rows, k = a.shape
    count, n, kw = b.shape if grouped else (1, *b.shape)
    m = rows if index is None else index.shape[0]
    if kw != k:
        raise RuntimeError(f"{what}: a has {k} columns, b {kw}")
    scale_type = pa = pb = lsa = lsb = gsb = pbias = gbias = py = ls = 0
    if f8:
        if a_scale is None or b_scale is None:
            raise RuntimeError(f"{what}: float8_e4m3fn operands need a_scale and b_scale")
        scale = a_scale.dtype
        scale_type = _SCALES.get(scale)
        if scale_type is None or b_scale.dtype != scale:
            raise RuntimeError(f"{what}: scales must both be float8_e8m0fnu or float32, not {scale} and {b_scale.dtype}")
        kb, nb = (k + 127) // 128, (n + 127) // 128
        want = (count, nb, kb) if grouped else (nb, kb)
        if a_scale.shape != (kb, rows) or b_scale.shape != want:
            raise RuntimeError(f"{what}: expected a_scale {(kb, rows)} and b_scale {want}, got {tuple(a_scale.shape)} and {tuple(b_scale.shape)}")
        a_scale, st = _rowed(a_scale)
        lsa = st[0]
        b_scale, st = _rowed(b_scale)
        lsb = st[-2]
        gsb = st[0] if grouped else 0
        pa, pb = a_scale.data_ptr(), b_scale.data_ptr()
    elif a_scale is not None or b_scale is not None:
        raise RuntimeError(f"{what}: bfloat16 operands have no scales")
    if bias is not None:
        want = (count, n) if grouped else (n,)
        if bias.dtype != torch.float32 or bias.shape != want:
            raise RuntimeError(f"{what}: bias must be float32 {want}, got {bias.dtype} {tuple(bias.shape)}")
        st = bias.stride()
        if st[-1] != 1 and n > 1:
            bias = bias.contiguous()
            st = bias.stride()
        pbias, gbias = bias.data_ptr(), st[0] if grouped else 0
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype, device=a.device)
        ldy = n
    else:
        ldy, step = out.stride() if out.dim() == 2 else (0, 0)
        if out.shape == (m, n) and m <= 1:
            ldy = n
        if out.dtype != out_dtype or out.shape != (m, n) or (n > 1 and step != 1) or ldy < n:
            raise RuntimeError(f"{what}: out must be a {out_dtype} ({m},{n}) tensor whose rows have no gaps and do not overlap")
    if out_type == 2:
        if out_scale is None:
            out_scale = torch.empty((nb, m), dtype=scale, device=a.device)
        elif out_scale.dtype != scale or out_scale.shape != (nb, m) or not out_scale.is_contiguous():
            raise RuntimeError(f"{what}: out_scale must be a contiguous {scale} ({nb},{m}) tensor")
        py, ls = out_scale.data_ptr(), m
    elif out_scale is not None:
        raise RuntimeError(f"{what}: out_scale belongs to float8_e4m3fn results")
    rc = _lib_entries()[1](dev, _raw_stream(dev), _MATMUL.pack(
        a.data_ptr(), sa[0], pa, lsa, b.data_ptr(), sb[-2], sb[0] if grouped else 0, pb, lsb, gsb, pbias, gbias, out.data_ptr(), ldy, py, ls,
        offsets.data_ptr() if grouped else 0, 0 if index is None else index.data_ptr(), rows, m, n, k, count, _TYPES[kind], scale_type, out_type, 1 if relu else 0, 0))
    if rc:
        _check(rc)
    return (out, out_scale) if out_type == 2 else out


def matmul_fp8(a, a_scale, b, b_scale, bias=None, relu: bool = False, out_dtype=torch.bfloat16, out=None, out_scale=None):
    """act(a @ b.T + bias) of e4m3 operands: a (m, k) with a_scale (ceil(k / 128), m), b (n, k) with b_scale (ceil(n / 128),
    ceil(k / 128)), as quantize makes them or of any value (float32); bias (n,) float32; act = ReLU if relu.  Sums are fp32 and are
    rounded once to out_dtype: float32, bfloat16, or float8_e4m3fn -- then (q, scale) with a power of two for every 128 columns of a
    row, in the operands' scale dtype: the next product's a and a_scale.  Any sizes and row strides; rows that start at multiples of
    16 bytes run fastest."""
    return _matmul("matmul_fp8", a, a_scale, b, b_scale, bias, relu, out_dtype, out, out_scale, None, None)


def matmul_grouped(a, b, offsets, index=None, a_scale=None, b_scale=None, bias=None, relu: bool = False, out_dtype=torch.bfloat16, out=None,
                   out_scale=None):
    """Row j of the result, offsets[g] <= j < offsets[g + 1], is act(a[index[j]] @ b[g].T + bias[g]) (a[j] without index): one weight
    matrix for each group of rows, however the rows fall.  a (rows, k) and b (groups, n, k) both bfloat16, or both float8_e4m3fn with
    a_scale (ceil(k / 128), rows) and b_scale (groups, ceil(n / 128), ceil(k / 128)); bias (groups, n) float32; offsets (groups + 1)
    int32, never falling, and index int32 on the device, as group_rows makes them: nothing is read back.  An index outside a reads as
    a row of zeros; rows that no group covers stay as they were in `out` (in a fresh result they hold nothing of use)."""
    if b.dim() != 3 or not 1 <= b.shape[0] <= GROUPS_MAX:
        raise RuntimeError(f"matmul_grouped: expected b (1 .. {GROUPS_MAX} groups, n, k), got {tuple(b.shape)}")
    if offsets.dtype != torch.int32 or offsets.shape != (b.shape[0] + 1,):
        raise RuntimeError(f"matmul_grouped: offsets must be int32 ({b.shape[0] + 1},), got {offsets.dtype} {tuple(offsets.shape)}")
    offsets = _vector(offsets)
    if index is not None:
        if index.dtype != torch.int32 or index.dim() != 1:
            raise RuntimeError(f"matmul_grouped: index must be int32 (m,), got {index.dtype} {tuple(index.shape)}")
        index = _vector(index)
    return _matmul("matmul_grouped", a, a_scale, b, b_scale, bias, relu, out_dtype, out, out_scale, offsets, index)


def group_rows(ids, groups: int):
    """ids (n,) int32 | int64 -> (offsets (groups + 1), order (n), place (n)), int32: order[j] is the row at place j, rows of a group in
    their own order (-1 behind the last group), place[i] the place of row i (-1 where the id is outside [0, groups))."""
    if ids.dim() != 1 or ids.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"group_rows: ids must be int32 or int64 (n,), got {ids.dtype} {tuple(ids.shape)}")
    groups = int(groups)
    if not 1 <= groups <= GROUPS_MAX:
        raise RuntimeError(f"group_rows: 1 .. {GROUPS_MAX} groups, not {groups}")
    dev = _at(ids, "group_rows")
    ids = _vector(ids)
    n = ids.shape[0]
    lib = _lib_entries()
    need = lib[3](n, groups)
    if need < 0:
        _check(need)
    made = torch.empty(groups + 1 + 2 * n + need, dtype=torch.int32, device=ids.device)
    offsets, order, place, work = made.split_with_sizes((groups + 1, n, n, need))
    p = made.data_ptr()
    rc = lib[2](dev, _raw_stream(dev), ids.data_ptr(), ids.element_size(), n, groups, p, p + 4 * (groups + 1), p + 4 * (groups + 1 + n),
                p + 4 * (groups + 1 + 2 * n) if need else None)
    if rc:
        _check(rc)
    return offsets, order, place


def decide(logits, index=None):
    """(rows, 16) float32 logits, picked by index (n,) int32 -> dict(logits (n, 16), pred (n,) int32, contacts (n, 4) uint8), as
    contact_cnn.predict returns them; an index outside the rows gives NaN logits and class 0."""
    if logits.dtype != torch.float32 or logits.dim() != 2 or logits.shape[1] != 16:
        raise RuntimeError(f"decide: expected float32 (rows, 16) logits, got {logits.dtype} {tuple(logits.shape)}")
    dev = _at(logits, "decide")
    _same(dev, "decide", logits, index)
    logits, at = logits.contiguous(), logits.device
    if index is not None:
        if index.dtype != torch.int32 or index.dim() != 1:
            raise RuntimeError(f"decide: index must be int32 (n,), got {index.dtype} {tuple(index.shape)}")
        index = _vector(index)
    n = logits.shape[0] if index is None else index.shape[0]
    out = {"logits": torch.empty((n, 16), dtype=torch.float32, device=at), "pred": torch.empty((n,), dtype=torch.int32, device=at),
           "contacts": torch.empty((n, 4), dtype=torch.uint8, device=at)}
    _check(_lib_entries()[4](dev, _raw_stream(dev), logits.data_ptr(), logits.shape[0], None if index is None else index.data_ptr(), n,
                             out["logits"].data_ptr(), out["pred"].data_ptr(), out["contacts"].data_ptr()))
    return out
