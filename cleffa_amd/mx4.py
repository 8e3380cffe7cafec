"""Microscaled 4-bit matrices on torch device memory, and the products with them: the projections either side of the
attention with weights in 4 bits, for prompts with activations in 4 bits too.

    w = Mx4Matrix.quantised(w_qkv)                  # once: [row][H] bf16, f16 or f32 weights
    x = Mx4Matrix(T, H)                             # a pass's activations
    qkv = mx4_gemm(x.quantise(h), w)                # or mx4_gemm(h, w): activations stay in bf16

Formats and layouts: include/clef_hip_attn.h. ``Mx4Matrix.from_codes`` takes codes and scales as files store them.

Calls run on the current stream, or on ``stream``; what they make lies in that stream's memory, as if made with it current. What
they are given has to stay until the call has run (``Tensor.record_stream`` where it is dropped before).
"""
import ctypes

import torch

from . import _lib
from .attention import _DTYPE_OUT, _arg, _device, _err, _launch, _on, init_device
from .gemm import Y_BF16, Y_F32

_Y_TYPES = {torch.bfloat16: Y_BF16, torch.float32: Y_F32}


def _rows_arg(t, name, shape, dtype, device, step=1):
    """Address and row stride of a matrix whose rows may lie apart (by multiples of ``step`` elements). One test for the
    ordinary case; the faults are told apart only where it fails."""
    if t.__class__ is torch.Tensor and t.dtype is dtype and t.shape == shape and t.device == device:
        row, one = t.stride()
        p = t.data_ptr()
        if one == 1 and row >= shape[1] and not row % step and (step == 1 or not p & 15):
            return p, row
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype is not dtype:
        raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    rows, cols = shape
    if cols > 1 and rows and t.stride(1) != 1:
        raise ValueError(f"the values of a row of {name} must be contiguous")
    row = t.stride(0) if rows > 1 else -(-cols // step) * step
    if row < cols or row % step:
        raise ValueError(f"rows of {name} are {row} elements apart: at least {cols} and a multiple of {step} are needed")
    if step > 1 and t.data_ptr() % 16:
        raise ValueError(f"{name} must be 16-byte aligned")
    return t.data_ptr(), row


class Mx4Matrix:
    """A matrix [rows][K] of e2m1 codes with a power-of-two scale for each 32 values of a row (K a multiple of 32), in
    ``codes`` and ``scales`` (uint8, in the order of the matrix instructions)."""

    def __init__(self, rows, K, device="cuda", codes=None, scales=None):
        n_codes, n_scales, err = ctypes.c_size_t(0), ctypes.c_size_t(0), _err()
        _lib.check(_lib.load().clef_hip_mx4_sizes(int(rows), int(K), ctypes.byref(n_codes), ctypes.byref(n_scales), err, len(err)), err)
        self.rows, self.K, self.device = int(rows), int(K), _device(device)
        if self.device.type == "cuda":
            init_device(self.device)
        self._codes = torch.empty(n_codes.value, dtype=torch.uint8, device=self.device) if codes is None else codes
        self._scales = torch.empty(n_scales.value, dtype=torch.uint8, device=self.device) if scales is None else scales
        # the buffers are the matrix's for good: their addresses are checked and taken once
        self._ptrs = (_arg(self._codes, "codes", (n_codes.value,), torch.uint8, self.device),
                      _arg(self._scales, "scales", (n_scales.value,), torch.uint8, self.device))

    codes = property(lambda self: self._codes)
    scales = property(lambda self: self._scales)

    def nbytes(self):
        return self._codes.numel() + self._scales.numel()

    def first(self, rows):
        """The first rows (a multiple of 16, or all) as a matrix in the same buffers."""
        if not 0 <= rows <= self.rows or (rows % 16 and rows != self.rows):
            raise ValueError(f"the first {rows} of {self.rows} rows: a multiple of 16, or all")
        tiles = -(-rows // 16)
        return Mx4Matrix(rows, self.K, self.device, self._codes[:tiles * -(-self.K // 128) * 1024], self._scales[:tiles * -(-self.K // 512) * 256])

    @classmethod
    def quantised(cls, x, stream=None):
        """x [rows][K] in 4 bits, in new buffers."""
        if x.dim() != 2:
            raise ValueError(f"a matrix is needed, not {tuple(x.shape)}")
        with _on(stream):
            m = cls(x.shape[0], x.shape[1], x.device)
        return m.quantise(x, stream=stream)

    @classmethod
    def from_codes(cls, codes, scales, stream=None):
        """From uint8 codes [rows][K / 2], the first of two in the lower four bits, and uint8 scale exponents + 127
        [rows][K / 32], as files store them (on the device)."""
        if codes.dim() != 2 or scales.dim() != 2:
            raise ValueError(f"codes and scales must be matrices, not {tuple(codes.shape)} and {tuple(scales.shape)}")
        with _on(stream):
            m = cls(codes.shape[0], 2 * codes.shape[1], codes.device)
        return m._pack(codes, scales, 0, stream)

    def to_codes(self, stream=None):
        """(codes [rows][K / 2], scales [rows][K / 32]), as from_codes takes them."""
        with _on(stream):
            codes = torch.empty(self.rows, self.K // 2, dtype=torch.uint8, device=self.device)
            scales = torch.empty(self.rows, self.K // _lib.MX4_BLOCK, dtype=torch.uint8, device=self.device)
        self._pack(codes, scales, 1, stream)
        return codes, scales

    def _pack(self, codes, scales, to_flat, stream):
        if codes.shape != (self.rows, self.K // 2) or scales.shape != (self.rows, self.K // _lib.MX4_BLOCK):
            raise ValueError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not fit {self.rows} x {self.K} values")
        flat = _arg(codes, "codes", codes.shape, torch.uint8, self.device)
        if scales.dtype is not torch.uint8 or scales.device != self.device or not scales.is_contiguous():
            raise ValueError("scales must be contiguous uint8 on the codes' device")
        own, rows, K = self._ptrs, self.rows, self.K
        lib = _lib.load()
        _launch(lambda a, s, err, n: lib.clef_hip_mx4_pack(rows, K, flat, scales.data_ptr(), *own, to_flat, s, err, n), ctypes.c_int(0), self.device, stream)
        return self

    def quantise(self, x, stream=None):
        """x [rows][K] (bf16, f16 or f32; rows may lie apart by multiples of 8) into this matrix. Returns it."""
        if not isinstance(x, torch.Tensor) or x.dtype not in _DTYPE_OUT:
            raise TypeError(f"x must be a bf16, f16 or f32 tensor, not {getattr(x, 'dtype', type(x))}")
        px, row = _rows_arg(x, "x", (self.rows, self.K), x.dtype, self.device, 8)
        _launch(_lib.load().clef_hip_mx4_quantise, _lib.Mx4RowsArgs(self.rows, self.K, _DTYPE_OUT[x.dtype], row, px, *self._ptrs), self.device, stream)
        return self

    def values(self, out=None, out_dtype="bf16", stream=None):
        """The values that the codes stand for, [rows][K] (bf16 or f32, both exact)."""
        if out is None:
            if out_dtype not in ("bf16", "f32"):
                raise ValueError(f"out_dtype {out_dtype!r}: bf16 or f32")
            with _on(stream):
                out = torch.empty(self.rows, self.K, dtype=torch.bfloat16 if out_dtype == "bf16" else torch.float32, device=self.device)
        if not isinstance(out, torch.Tensor) or out.dtype not in _Y_TYPES:
            raise TypeError("out must be a bf16 or f32 tensor")
        px, row = _rows_arg(out, "out", (self.rows, self.K), out.dtype, self.device, 8)
        _launch(_lib.load().clef_hip_mx4_values, _lib.Mx4RowsArgs(self.rows, self.K, _DTYPE_OUT[out.dtype], row, px, *self._ptrs), self.device, stream)
        return out


def mx4_gemm(X, W, Y=None, out="bf16", residual=None, stream=None):
    """Y [T][N] = X . W^T (+ residual): W an Mx4Matrix [N][K], X an Mx4Matrix [T][K] or a bf16 tensor [T][K] whose rows may lie
    apart by multiples of 8. Y bf16 or f32 (its own type where it is given, else ``out``), rows may lie apart;
    residual f32 [T][N], with an f32 Y, which it may be."""
    if not isinstance(W, Mx4Matrix):
        raise TypeError("W must be an Mx4Matrix")
    dev, N, K = W.device, W.rows, W.K
    if isinstance(X, Mx4Matrix):
        if X.device != dev:
            raise ValueError(f"X is on {X.device}, W on {dev}")
        T, xk, xb, x_row, xc = X.rows, X.K, None, 0, X._ptrs
    else:
        if not isinstance(X, torch.Tensor) or X.dim() != 2:
            raise TypeError("X must be an Mx4Matrix or a matrix in bf16")
        T, xk, xc = X.shape[0], X.shape[1], (None, None)
    if xk != K:
        raise ValueError(f"inner dims differ: X has {xk}, W has {K}")
    if xc[0] is None and T:
        xb, x_row = _rows_arg(X, "X", (T, K), torch.bfloat16, dev, 8)
    if Y is None:
        if out not in ("bf16", "f32"):
            raise ValueError(f"out {out!r}: bf16 or f32")
        with _on(stream):
            Y = torch.empty(T, N, dtype=torch.bfloat16 if out == "bf16" and residual is None else torch.float32, device=dev)
    if not isinstance(Y, torch.Tensor) or Y.dtype not in _Y_TYPES:
        raise TypeError("Y must be a bf16 or f32 tensor")
    py, y_row = _rows_arg(Y, "Y", (T, N), Y.dtype, dev)
    if T == 0:
        return Y
    pr, r_row = (None, 0) if residual is None else _rows_arg(residual, "residual", (T, N), torch.float32, dev)
    a = _lib.Mx4GemmArgs(T, N, K, _Y_TYPES[Y.dtype], *W._ptrs, *xc, xb, x_row, y_row, r_row, py, pr)
    _launch(_lib.load().clef_hip_mx4_gemm, a, dev, stream)
    return Y
