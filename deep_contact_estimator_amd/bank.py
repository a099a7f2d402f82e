"""One conv stack, many FC heads: every window takes the FC layers of its own head.

The reference trains one checkpoint for all its data (src/train.py:145-153).  Here the conv stack of one checkpoint serves any number of
heads -- a robot's, a gait's, a terrain's own fc.0 / fc.3 / fc.6 (src/contact_cnn.py:47-58), fine-tuned behind the shared stack -- and a
batch may mix them as the windows come:

    bank = contact_bank(precision="bf16_fc").load_state_dict(checkpoint, [head_a, head_b, ...])
    out = bank.predict(windows, head)                      # head (n,): which head each window takes

The windows' features are grouped by head on the device and each layer is one grouped product (ops.matmul_grouped): nothing is read
back, and a head without windows costs nothing.
"""
from __future__ import annotations

from typing import Mapping, Sequence

import numpy as np

from . import ops
from .contact_cnn import _is_torch, contact_cnn
from .synth import STATE_DICT_SHAPES

FEAT_T, FEAT_C = 37, 128                                   # a window's features: (c, t) in the reference's order, (t, c) in the kernels'
HEAD_KEYS = [k for k, _ in STATE_DICT_SHAPES if k.startswith("fc.")]


class contact_bank:
    """contact_cnn with a bank of FC heads.  precision: "bf16_fc" -- bf16 features, weights and activations, fp32 sums; "fp8_fc" -- fc.0 and
    fc.3 in e4m3 with a power of two for every 128 values (dce.h DCE_FP8_FC), the rest bf16.  max_batch, tune: contact_cnn's.
    Calls on CUDA tensors run on torch's current stream and may be captured once one has run; the conv stack's context serves one stream at a
    time, replayed graphs included (as contact_cnn's).  load_state_dict ends the graphs captured before it: they hold the addresses of weights that
    it gives back (as contact_cnn's do), so capture again."""

    def __init__(self, device=None, max_batch: int = 32768, precision: str = "bf16_fc", tune=None):
        if precision not in ("bf16_fc", "fp8_fc"):
            raise RuntimeError(f"contact_bank: precision must be bf16_fc or fp8_fc, not {precision}")
        self._conv = contact_cnn(device=device, max_batch=max_batch, precision=precision, tune=tune)
        self._f8 = precision == "fp8_fc"
        self._heads: list[dict[str, np.ndarray]] = []
        self._layers = None
        self._streams: set[int] = set()                    # that the layers' memory is known to be used on

    def load_state_dict(self, state_dict: Mapping, heads: Sequence[Mapping]):
        """state_dict: a checkpoint of the reference (its conv stack is used); heads: one mapping with the six fc.* keys for each head (a whole
        checkpoint will do).  Graphs captured before this call must not be replayed after it."""
        if not 1 <= len(heads) <= ops.GROUPS_MAX:
            raise RuntimeError(f"contact_bank: 1 .. {ops.GROUPS_MAX} heads, not {len(heads)}")
        shapes, found = dict(STATE_DICT_SHAPES), []
        for i, h in enumerate(heads):
            missing = [k for k in HEAD_KEYS if k not in h]
            if missing:
                raise RuntimeError(f"contact_bank: head {i}: missing key(s) {missing}")
            one = {}
            for k in HEAD_KEYS:
                v = h[k].detach().cpu().numpy() if _is_torch(h[k]) else h[k]
                one[k] = np.array(v, dtype=np.float32, order="C")         # (a copy: what the caller does to its arrays later is not the bank's)
                if one[k].shape != shapes[k]:
                    raise RuntimeError(f"contact_bank: head {i}: size mismatch for {k}: {one[k].shape}, model {shapes[k]}")
            found.append(one)
        self._conv.load_state_dict(state_dict)
        self._heads, self._layers = found, None
        return self

    def __len__(self):
        return len(self._heads)

    def _on_device(self, device):
        """[(weights, scales, bias)] of the three layers, stacked over the heads."""
        import torch
        stream = torch.cuda.current_stream(device)
        if self._layers is not None and self._layers[0] == device:
            if stream.cuda_stream not in self._streams:    # (memory of one stream's pool: given back, it is not to be used again before this stream is through with it)
                for t in (t for layer in self._layers[1] for t in layer if t is not None):
                    t.record_stream(stream)
                self._streams.add(stream.cuda_stream)
            return self._layers[1]
        if not self._heads:
            raise RuntimeError("load_state_dict first: the bank has no heads")
        layers = []
        for key in ("fc.0", "fc.3", "fc.6"):
            shape = self._heads[0][key + ".weight"].shape
            kind = torch.float8_e4m3fn if self._f8 and key != "fc.6" else torch.bfloat16
            w = torch.empty((len(self._heads), *shape), dtype=kind, device=device)
            s = torch.empty((len(self._heads), -(-shape[0] // 128), -(-shape[1] // 128)), dtype=ops.E8M0, device=device) if kind != torch.bfloat16 else None
            for i, h in enumerate(self._heads):            # (a head at a time: fc.0's fp32 weights of a thousand heads are 39 GB)
                v = torch.from_numpy(h[key + ".weight"]).to(device)
                if key == "fc.0":
                    v = v.view(-1, FEAT_C, FEAT_T).transpose(1, 2).reshape(shape)
                if s is None:
                    w[i] = v.bfloat16()
                else:
                    q, e = ops.quantize(v, rows=128)
                    w.view(torch.uint8)[i], s.view(torch.uint8)[i] = q.view(torch.uint8), e.view(torch.uint8)
            layers.append((w, s, torch.from_numpy(np.stack([h[key + ".bias"] for h in self._heads])).to(device)))
        stream.synchronize()                               # (whatever stream the next call is on finds them whole)
        self._layers, self._streams = (device, layers), {stream.cuda_stream}
        return layers

    def _run(self, x, head, raw_sequence: bool):
        import torch
        if not _is_torch(head):
            head = torch.from_numpy(np.ascontiguousarray(head))
        if head.numel() and (head.dtype.is_floating_point or head.dtype.is_complex):             # (an empty list has no type of its own)
            raise RuntimeError(f"contact_bank: head must be whole numbers, got {head.dtype}")     # (-0.5 is no head: rounded towards zero it would be one)
        host = not (_is_torch(x) and x.is_cuda)
        if host:
            self._conv._ensure_ctx()
            at = torch.device("cuda", self._conv._dev_index)
            x = (x if _is_torch(x) else torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32))).to(at)
        feat = self._conv.features(x, raw_sequence)
        head = head.to(feat.device)
        if head.dtype not in (torch.int32, torch.int64):
            head = head.long()
        if tuple(head.shape) != (feat.shape[0],):
            raise RuntimeError(f"expected one head a window, ({feat.shape[0]},), got {tuple(head.shape)}")
        (w0, s0, b0), (w3, s3, b3), (w6, _, b6) = self._on_device(feat.device)
        with torch.no_grad():
            offsets, order, place = ops.group_rows(head, len(self._heads))
            if self._f8:
                q, s = ops.quantize(feat)
                h, hs = ops.matmul_grouped(q, w0, offsets, index=order, a_scale=s, b_scale=s0, bias=b0, relu=True, out_dtype=ops.E4M3)
                h = ops.matmul_grouped(h, w3, offsets, a_scale=hs, b_scale=s3, bias=b3, relu=True)
            else:
                h = ops.matmul_grouped(feat, w0, offsets, index=order, bias=b0, relu=True)
                h = ops.matmul_grouped(h, w3, offsets, bias=b3, relu=True)
            out = ops.decide(ops.matmul_grouped(h, w6, offsets, bias=b6, out_dtype=torch.float32), place)
        return {k: v.cpu().numpy() for k, v in out.items()} if host else out

    def predict(self, x, head):
        """(n,150,54) z-scored windows, head (n,) -> dict(logits (n,16), pred (n,), contacts (n,4)), as contact_cnn.predict; a window whose head
        is outside [0, len(bank)) gets NaN logits and class 0."""
        contact_cnn._check_windows(x)
        return self._run(x, head, False)

    def infer_sequence(self, seq, head):
        """Raw (T,54) rows, head (T-149,) of the windows that end at rows 149 .. T-1 -> the same, row j for data row j+149."""
        return self._run(seq, head, True)
