"""Rotary positions of q and k heads, RMSNorm ahead of them where the model has one, as an operator of its own: the
prologues inside the attention turn 64 dims in the half layout; this one turns any even part of the head, in both
layouts, with frequencies scaled for long texts, in the rows of a projection or out of them.

    rotary = Rotary(n_rot=128, theta=1e7, layout="interleaved", scaling={"kind": "parts", "factor": 8, "original": 16384})
    q, k = rotary.heads(qkv, nh, nkv, hd)             # views of the projection's rows
    rotary.apply(q, k, pos, q_norm, k_norm, q_out=q, k_out=k)
    out = TextAttention(nh, nkv, n_rot=0).forward(qkv, None, None, pos3, plan)

Formulas: include/clef_hip_attn.h.
"""
import ctypes
import math

import numpy as np
import torch

from . import _lib
from .attention import _DTYPE_OUT, _arg, _device, _launch, _on, _err, init_device


class Rotary:
    """Frequencies and layout of a model's rotary positions. layout "half" (dims j and j + n_rot / 2 turn together) or
    "interleaved" (2j and 2j + 1). axes: int32 positions a row; pair j goes by position j % axes. scaling: None, or
    a dict of "kind" ("linear", "base" or "parts"), "factor" and for "parts" "original" (the length that the model was
    trained for), "low" and "high" (1 and 32: pairs that turn less over it are stretched, that turn more are kept). magnitude
    multiplies all turned dims (None: 0.1 ln factor + 1 for "parts", else 1). freqs: radians a position of each pair,
    float64 [n_rot / 2], in place of the formula.

    "parts" is linear in the turns of a pair. Checkpoints whose programs make it linear in the pair's index, between rounded
    borders, need freqs; ones scaled with low 1 and high 4 usually have no magnitude: magnitude=1."""

    def __init__(self, n_rot, theta=1e7, layout="half", axes=1, scaling=None, magnitude=None, freqs=None, eps=1e-6, device="cuda"):
        if layout not in _lib.ROTARY_LAYOUTS:
            raise ValueError(f"layout {layout!r}: half or interleaved")
        if not 1 <= axes <= 4:
            raise ValueError(f"{axes} position axes: 1 to 4 are supported")
        s = {"kind": None, "factor": 1.0, "original": 0.0, "low": 1.0, "high": 32.0}
        unknown = set(scaling or {}) - set(s)
        s.update(scaling or {})
        if unknown or s["kind"] not in _lib.ROTARY_SCALINGS or (scaling and s["kind"] is None):
            raise ValueError(f"scaling {scaling!r}: kind linear, base or parts, factor, original, low, high")
        table, err = np.zeros(max(n_rot // 2, 1)), _err()
        _lib.check(_lib.load().clef_hip_rotary_freqs(n_rot, theta, _lib.ROTARY_SCALINGS[s["kind"]], s["factor"], s["original"], s["low"], s["high"],
                                                     table.ctypes.data_as(ctypes.POINTER(ctypes.c_double)), err, len(err)), err)
        if freqs is not None:
            freqs = np.asarray(freqs, dtype=np.float64)
            if scaling is not None or freqs.shape != table.shape or not np.isfinite(freqs).all():
                raise ValueError(f"freqs takes the place of a scaling: {n_rot // 2} finite values")
            table = freqs / (2 * math.pi)
        if magnitude is None:
            magnitude = 0.1 * math.log(s["factor"]) + 1 if s["kind"] == "parts" else 1.0
        if not math.isfinite(magnitude):
            raise ValueError(f"magnitude {magnitude}")
        self.n_rot, self.layout, self.axes, self.eps, self.magnitude = int(n_rot), layout, int(axes), eps, float(magnitude)
        self._layout = _lib.ROTARY_LAYOUTS[layout]
        self.device = _device(device)
        if self.device.type == "cuda":
            init_device(self.device)
        self.freq = torch.from_numpy(table).to(self.device)     # turns a position

    @staticmethod
    def heads(qkv, nh, nkv, hd, gated=True):
        """The q and k heads [T][heads][hd] of projection rows, [query | gate] of each q head where the model gates, then
        the k heads, then the v heads, as views."""
        wide = 2 if gated else 1
        if qkv.dim() != 2 or qkv.shape[1] < (wide * nh + 2 * nkv) * hd:
            raise ValueError(f"rows {tuple(qkv.shape)} do not hold {nh} / {nkv} heads of {hd}")
        q = qkv[:, :wide * nh * hd].unflatten(1, (nh, wide * hd))[:, :, :hd]
        return q, qkv[:, wide * nh * hd:(wide * nh + nkv) * hd].unflatten(1, (nkv, hd))

    def _view(self, t, name, shape, dtype):
        """Address, row and head stride of heads. One test for the ordinary case; the faults are told apart only where it fails."""
        if t.__class__ is torch.Tensor and t.dtype is dtype and t.shape == shape and t.device == self.device:
            row, head, one = t.stride()
            if one == 1:
                return t.data_ptr(), row, head
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch tensor")
        if t.shape != shape:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
        if t.dtype is not dtype:
            raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")
        if t.device != self.device:
            raise ValueError(f"{name} is on {t.device}, expected {self.device}")
        if t.numel():
            raise ValueError(f"the dims of a head of {name} must be contiguous")
        return t.data_ptr(), 0, 0

    def _heads(self, x, out, norm, name, T, hd, dtype, out_dtype):
        if x is None:
            if out is not None or norm is not None:
                raise ValueError(f"{name}: an output or norm without heads")
            return 0, None, None, 0, 0, 0, 0, None
        shape = (T, x.shape[1] if isinstance(x, torch.Tensor) and x.dim() == 3 else -1, hd)
        px, row, head = self._view(x, name, shape, dtype)
        po, out_row, out_head = (px, row, head) if out is x and out_dtype is dtype else self._view(out, name + "_out", shape, out_dtype)
        return shape[1], px, po, row, head, out_row, out_head, None if norm is None else _arg(norm, name + "_norm", (hd,), torch.float32, self.device)

    def apply(self, q, k, pos, q_norm=None, k_norm=None, q_out=None, k_out=None, stream=None):
        """q [T][nh][hd] and k [T][nkv][hd] (or None), bf16, f16 or f32, turned by pos (int32 [T] or [T][axes]), each after its
        RMSNorm where a weight [hd] f32 is given. Rows and heads may lie apart (views of a projection's rows). q_out and
        k_out: new tensors where they are None; q and k themselves for a rotation in place; of q's type, or bf16 where q is
        f32, which rounds once where a projection's bf16 rows have been rounded before. Returns (q_out, k_out)."""
        if not isinstance(q, torch.Tensor) or q.dim() != 3 or q.dtype not in _DTYPE_OUT:
            raise TypeError("q must be a bf16, f16 or f32 tensor [T][heads][hd]")
        T, _, hd = q.shape
        dtype = q.dtype
        given = k_out if q_out is None else q_out
        narrow = dtype is torch.float32 and isinstance(given, torch.Tensor) and given.dtype is torch.bfloat16
        out_dtype = torch.bfloat16 if narrow else dtype
        if q_out is None:
            with _on(stream):
                q_out = torch.empty_like(q, dtype=out_dtype, memory_format=torch.contiguous_format)
        if k_out is None and k is not None:
            with _on(stream):
                k_out = torch.empty_like(k, dtype=out_dtype, memory_format=torch.contiguous_format)
        if not isinstance(pos, torch.Tensor) or pos.dtype is not torch.int32 or pos.device != self.device or not pos.is_contiguous():
            raise ValueError("pos must be contiguous int32 on the operator's device")
        if pos.shape != (T, self.axes) and (self.axes > 1 or pos.shape != (T,)):
            raise ValueError(f"pos has shape {tuple(pos.shape)}, expected {(T, self.axes)}")
        a = _lib.RotaryArgs(T, hd, self.n_rot, self._layout, self.axes, _DTYPE_OUT[dtype], self.eps, self.magnitude, pos.data_ptr(), self.freq.data_ptr(),
                            *self._heads(q, q_out, q_norm, "q", T, hd, dtype, out_dtype), *self._heads(k, k_out, k_norm, "k", T, hd, dtype, out_dtype), int(narrow))
        _launch(_lib.load().clef_hip_rotary, a, self.device, stream)
        return q_out, k_out
