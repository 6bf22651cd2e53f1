"""The dense side of a decode step, over torch CUDA tensors: residual
addition + RMSNorm, and products with 4-bit weights.

Thin wrappers over the C ABI (include/mitten_kv.h), like mitten_b200.paged:
every computation runs in libmitten_kv.so, on the tensors' device and that
device's current stream unless one is given; there is no CPU implementation.
"""
from __future__ import annotations

import torch

from . import _lib as L

_CODES = {torch.bfloat16: L.MTN_DTYPE_BF16, torch.float32: L.MTN_DTYPE_F32, torch.float8_e4m3fn: L.MTN_DTYPE_E4M3}
_FLOATS = (torch.bfloat16, torch.float32)


def _rows(t: torch.Tensor, name: str, dtypes) -> None:
    """A CUDA tensor [rows, elements] of unit-stride rows that do not overlap."""
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor (there is no CPU implementation)")
    if t.dim() != 2 or t.dtype not in dtypes:
        raise ValueError(f"{name}: expected a 2-D tensor of {' or '.join(map(str, dtypes))}, got {t.dim()}-D {t.dtype}")
    if t.numel() and (t.stride(1) != 1 and t.shape[1] > 1 or t.stride(0) < t.shape[1] and t.shape[0] > 1):
        raise ValueError(f"{name}: rows must have unit stride and not overlap")


def _stride(t: torch.Tensor) -> int:
    """Elements between rows; a single row's stride says nothing."""
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def _same_device(x: torch.Tensor, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, the rows on {x.device}")


def _stream_of(x: torch.Tensor, stream) -> int:
    return int((torch.cuda.current_stream(x.device) if stream is None else stream).cuda_stream)


def add_rms_norm(x: torch.Tensor, w1: torch.Tensor | None = None, eps: float = 1e-6, *,
                 residual: torch.Tensor | None = None, sum_out: torch.Tensor | None = None,
                 out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                 scales: torch.Tensor | None = None, stream=None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """s = x + residual; out = s / sqrt(mean(s^2) + eps) * w1, for rows x [n, hidden] (mtn_add_rms_norm).

    `residual` takes the sum in place unless `sum_out` is given, rounded to its type; the norm reads the sum as
    it is stored.  `w1` is 1 + w in f32.  `out_dtype` (x's type by default): bf16, f32, or float8_e4m3fn with one
    f32 scale per row (out * scale is the value).  Returns (out, scales), scales None unless out is e4m3."""
    if x.is_cuda and x.device.index != torch.cuda.current_device():
        with torch.cuda.device(x.device):
            return add_rms_norm(x, w1, eps, residual=residual, sum_out=sum_out, out=out, out_dtype=out_dtype,
                                scales=scales, stream=stream)
    _rows(x, "x", _FLOATS)
    n, hidden = x.shape
    if w1 is not None and (w1.dtype != torch.float32 or w1.shape != (hidden,) or not w1.is_contiguous()):
        raise ValueError("w1 must be a contiguous f32 tensor of one value per element")
    if out is None:
        out = torch.empty((n, hidden), dtype=out_dtype or x.dtype, device=x.device)
    elif out_dtype is not None and out.dtype != out_dtype:
        raise ValueError("out and out_dtype disagree")
    _rows(out, "out", _CODES)
    if out.shape != x.shape:
        raise ValueError("out must have x's shape")
    if residual is None:
        if sum_out is not None:
            raise ValueError("sum_out without a residual")
    else:
        sum_out = residual if sum_out is None else sum_out
        _rows(residual, "residual", _FLOATS)
        _rows(sum_out, "sum_out", (residual.dtype,))
        if residual.shape != x.shape or sum_out.shape != x.shape:
            raise ValueError("residual and sum_out must have x's shape")
    if out.dtype == torch.float8_e4m3fn:
        if scales is None:
            scales = torch.empty(n, dtype=torch.float32, device=x.device)
        elif scales.dtype != torch.float32 or scales.shape != (n,) or not scales.is_contiguous():
            raise ValueError("scales must be a contiguous f32 tensor of one value per row")
    elif scales is not None:
        raise ValueError("scales go with an e4m3 output only")
    _same_device(x, w1=w1, out=out, residual=residual, sum_out=sum_out, scales=scales)
    if n == 0:
        return out, scales
    L.check(L.lib().mtn_add_rms_norm(
        x.data_ptr(), _CODES[x.dtype], _stride(x), None if residual is None else residual.data_ptr(),
        0 if residual is None else _stride(residual), None if residual is None else sum_out.data_ptr(),
        0 if residual is None else _stride(sum_out), 0 if residual is None else _CODES[residual.dtype],
        None if w1 is None else w1.data_ptr(), eps, n, hidden, out.data_ptr(), _CODES[out.dtype], _stride(out),
        None if scales is None else scales.data_ptr(), _stream_of(x, stream)))
    return out, scales


class W4Weight:
    """A weight matrix [n, k] as 4-bit codes with one bf16 scale per `group` elements of a row, in the layout
    mtn_w4_matvec reads.  Made once (from_float quantises, from_codes packs) and kept."""

    def __init__(self, n: int, k: int, group: int, device):
        nb = L.lib().mtn_w4_packed_bytes(n, k)
        ns = L.lib().mtn_w4_scales_bytes(n, k, group)
        if nb == 0 or ns == 0:
            raise ValueError(f"no 4-bit layout for [{n}, {k}] in groups of {group}")
        self.n, self.k, self.group = n, k, group
        self.packed = torch.empty(nb, dtype=torch.uint8, device=device)
        self.scales = torch.empty(ns // 2, dtype=torch.bfloat16, device=device)

    @property
    def device(self) -> torch.device:
        return self.packed.device

    @classmethod
    def from_float(cls, weight: torch.Tensor, group: int = 128, stream=None) -> "W4Weight":
        """Quantise bf16 / f32 weights [n, k]: per group scale = bf16(max|w| / 7), code = round(w / scale)."""
        _rows(weight, "weight", _FLOATS)
        w = cls(*weight.shape, group, weight.device)
        with torch.cuda.device(weight.device):
            L.check(L.lib().mtn_w4_quantize(weight.data_ptr(), _CODES[weight.dtype], _stride(weight), w.n, w.k, group,
                                            w.packed.data_ptr(), w.scales.data_ptr(), _stream_of(weight, stream)))
        return w

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor, group: int = 128, stream=None) -> "W4Weight":
        """Pack int8 codes [n, k] (-8..7) and bf16 scales [n, ceil(k / group)]."""
        _rows(codes, "codes", (torch.int8,))
        _rows(scales, "scales", (torch.bfloat16,))
        w = cls(*codes.shape, group, codes.device)
        if scales.shape != (w.n, -(-w.k // group)):
            raise ValueError("scales must be [n, ceil(k / group)]")
        _same_device(codes, scales=scales)
        with torch.cuda.device(codes.device):
            L.check(L.lib().mtn_w4_pack(codes.data_ptr(), _stride(codes), scales.data_ptr(), _stride(scales), w.n, w.k,
                                        group, w.packed.data_ptr(), w.scales.data_ptr(), _stream_of(codes, stream)))
        return w

    def dequantize(self, dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None,
                   stream=None) -> torch.Tensor:
        """The values code * scale, row-major [n, k] in f32 (exact) or bf16."""
        if out is None:
            out = torch.empty((self.n, self.k), dtype=dtype, device=self.device)
        _rows(out, "out", _FLOATS)
        if out.shape != (self.n, self.k):
            raise ValueError("out must be [n, k]")
        _same_device(self.packed, out=out)
        with torch.cuda.device(self.device):
            L.check(L.lib().mtn_w4_dequantize(self.packed.data_ptr(), self.scales.data_ptr(), self.n, self.k, self.group,
                                              out.data_ptr(), _CODES[out.dtype], _stride(out), _stream_of(out, stream)))
        return out


def w4_matvec(x: torch.Tensor, weight: W4Weight, *, x_scales: torch.Tensor | None = None,
              out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None, stream=None) -> torch.Tensor:
    """x [m, k] times the transposed 4-bit weight: [m, n] in bf16 or f32 (mtn_w4_matvec), sums in f32.

    x: bf16, f32, or float8_e4m3fn with `x_scales`, one f32 per row (add_rms_norm's e4m3 output).  `out_dtype`
    defaults to x's type, or bf16 for e4m3.  Meant for the few rows of a decode step: the weights are read once
    per 16 rows; for a prompt's many rows dequantise and use a matrix product."""
    if x.is_cuda and x.device.index != torch.cuda.current_device():
        with torch.cuda.device(x.device):
            return w4_matvec(x, weight, x_scales=x_scales, out=out, out_dtype=out_dtype, stream=stream)
    _rows(x, "x", _CODES)
    m = x.shape[0]
    if x.shape[1] != weight.k:
        raise ValueError(f"x has {x.shape[1]} columns, the weight {weight.k}")
    if (x.dtype == torch.float8_e4m3fn) != (x_scales is not None):
        raise ValueError("x_scales go with float8_e4m3fn rows, and only with them")
    if x_scales is not None and (x_scales.dtype != torch.float32 or x_scales.shape != (m,)
                                 or not x_scales.is_contiguous()):
        raise ValueError("x_scales must be a contiguous f32 tensor of one value per row")
    if out is None:
        out = torch.empty((m, weight.n), device=x.device,
                          dtype=out_dtype or (x.dtype if x_scales is None else torch.bfloat16))
    elif out_dtype is not None and out.dtype != out_dtype:
        raise ValueError("out and out_dtype disagree")
    _rows(out, "out", _FLOATS)
    if out.shape != (m, weight.n):
        raise ValueError("out must be [rows, n]")
    _same_device(x, weight=weight, x_scales=x_scales, out=out)
    if m == 0:
        return out
    L.check(L.lib().mtn_w4_matvec(x.data_ptr(), _CODES[x.dtype], _stride(x),
                                  None if x_scales is None else x_scales.data_ptr(), m, weight.packed.data_ptr(),
                                  weight.scales.data_ptr(), weight.n, weight.k, weight.group, out.data_ptr(),
                                  _CODES[out.dtype], _stride(out), _stream_of(x, stream)))
    return out
