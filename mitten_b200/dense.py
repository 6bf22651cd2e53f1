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
_FLOATS = {torch.bfloat16: L.MTN_DTYPE_BF16, torch.float32: L.MTN_DTYPE_F32}

# A decode step makes hundreds of these calls, each of a few microseconds: the
# checks read every property of a tensor once.
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device


def _rows(t: torch.Tensor, name: str, dtypes, device: int) -> tuple[int, int]:
    """(type code, elements between rows) of a tensor [rows, elements] on `device` whose unit-stride rows do not
    overlap; raises for any other."""
    code = dtypes.get(t.dtype)
    if code is None or t.dim() != 2:
        raise ValueError(f"{name}: expected a 2-D tensor of {' or '.join(map(str, dtypes))}, got {t.dim()}-D {t.dtype}")
    if t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{device}")
    row, unit = t.stride()
    n, width = t.shape
    if unit != 1 or row < width:
        if (unit != 1 and width > 1 and n) or (row < width and n > 1):
            raise ValueError(f"{name}: rows must have unit stride and not overlap")
        if n <= 1:
            row = width  # a single row's stride says nothing
    return code, row


def _values(t: torch.Tensor, name: str, n: int, device: int) -> int:
    """Address of a contiguous f32 tensor of n values on `device`."""
    if t.dtype != torch.float32 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous f32 tensor of {n} values")
    if t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{device}")
    return t.data_ptr()


def _device_of(x: torch.Tensor, name: str) -> int:
    if not x.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor (there is no CPU implementation)")
    return x.get_device()


def _stream_of(device: int) -> int:
    return torch._C._cuda_getCurrentRawStream(device)


def _on(stream, device: int):
    """Makes `stream` (None: the current one) and its device current, so that the memory allocated for a result
    belongs to the stream that writes it."""
    if stream is None:
        return torch.cuda.device(device)
    if stream.device_index != device:
        raise ValueError(f"the stream is cuda:{stream.device_index}'s, the tensors are on cuda:{device}")
    return torch.cuda.stream(stream)


def add_rms_norm(x: torch.Tensor, w1: torch.Tensor | None = None, eps: float = 1e-6, *,
                 residual: torch.Tensor | None = None, sum_out: torch.Tensor | None = None,
                 out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                 scales: torch.Tensor | None = None, stream=None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """s = x + residual; out = s / sqrt(mean(s^2) + eps) * w1, for rows x [n, hidden] (mtn_add_rms_norm).

    `residual` takes the sum in place unless `sum_out` is given, rounded to its type; the norm reads the sum as
    it is stored.  `w1` is 1 + w in f32.  `out_dtype` (x's type by default): bf16, f32, or float8_e4m3fn with one
    f32 scale per row (out * scale is the value).  Returns (out, scales), scales None unless out is e4m3."""
    dev = _device_of(x, "x")
    if stream is not None or dev != _current_device():
        with _on(stream, dev):
            return add_rms_norm(x, w1, eps, residual=residual, sum_out=sum_out, out=out, out_dtype=out_dtype,
                                scales=scales)
    xc, xs = _rows(x, "x", _FLOATS, dev)
    shape = x.shape
    n, hidden = shape
    w1p = None if w1 is None else _values(w1, "w1", hidden, dev)
    if out is None:
        out = torch.empty(shape, dtype=out_dtype or x.dtype, device=x.device)
    elif out_dtype is not None and out.dtype != out_dtype:
        raise ValueError("out and out_dtype disagree")
    oc, os_ = _rows(out, "out", _CODES, dev)
    if out.shape != shape:
        raise ValueError("out must have x's shape")
    rp = sp = None
    rc = rs = ss = 0
    if residual is not None:
        rc, rs = _rows(residual, "residual", _FLOATS, dev)
        rp = sp = residual.data_ptr()
        ss = rs
        if residual.shape != shape:
            raise ValueError("residual must have x's shape")
        if sum_out is not None:
            sc, ss = _rows(sum_out, "sum_out", _FLOATS, dev)
            sp = sum_out.data_ptr()
            if sc != rc or sum_out.shape != shape:
                raise ValueError("sum_out must have residual's type and shape")
    elif sum_out is not None:
        raise ValueError("sum_out without a residual")
    scp = None
    if oc == L.MTN_DTYPE_E4M3:
        if scales is None:
            scales = torch.empty(n, dtype=torch.float32, device=x.device)
        scp = _values(scales, "scales", n, dev)
    elif scales is not None:
        raise ValueError("scales go with an e4m3 output only")
    if n:
        st = L.lib().mtn_add_rms_norm(x.data_ptr(), xc, xs, rp, rs, sp, ss, rc, w1p, eps, n, hidden, out.data_ptr(), oc,
                                      os_, scp, _stream_of(dev))
        if st:
            L.check(st)
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
        dev = _device_of(weight, "weight")
        code, row = _rows(weight, "weight", _FLOATS, dev)
        with _on(stream, dev):
            w = cls(*weight.shape, group, weight.device)
            L.check(L.lib().mtn_w4_quantize(weight.data_ptr(), code, row, w.n, w.k, group, w.packed.data_ptr(),
                                            w.scales.data_ptr(), _stream_of(dev)))
        return w

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor, group: int = 128, stream=None) -> "W4Weight":
        """Pack int8 codes [n, k] (-8..7) and bf16 scales [n, ceil(k / group)]."""
        dev = _device_of(codes, "codes")
        _, code_row = _rows(codes, "codes", {torch.int8: 0}, dev)
        _, scale_row = _rows(scales, "scales", {torch.bfloat16: 0}, dev)
        with _on(stream, dev):
            w = cls(*codes.shape, group, codes.device)
            if scales.shape != (w.n, -(-w.k // group)):
                raise ValueError("scales must be [n, ceil(k / group)]")
            L.check(L.lib().mtn_w4_pack(codes.data_ptr(), code_row, scales.data_ptr(), scale_row, w.n, w.k, group,
                                        w.packed.data_ptr(), w.scales.data_ptr(), _stream_of(dev)))
        return w

    def dequantize(self, dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None,
                   stream=None) -> torch.Tensor:
        """The values code * scale, row-major [n, k] in f32 (exact) or bf16."""
        dev = self.packed.get_device()
        with _on(stream, dev):
            if out is None:
                out = torch.empty((self.n, self.k), dtype=dtype, device=self.device)
            code, row = _rows(out, "out", _FLOATS, dev)
            if out.shape != (self.n, self.k):
                raise ValueError("out must be [n, k]")
            L.check(L.lib().mtn_w4_dequantize(self.packed.data_ptr(), self.scales.data_ptr(), self.n, self.k, self.group,
                                              out.data_ptr(), code, row, _stream_of(dev)))
        return out


def w4_matvec(x: torch.Tensor, weight: W4Weight, *, x_scales: torch.Tensor | None = None,
              out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None, stream=None) -> torch.Tensor:
    """x [m, k] times the transposed 4-bit weight: [m, n] in bf16 or f32 (mtn_w4_matvec), sums in f32.

    x: bf16, f32, or float8_e4m3fn with `x_scales`, one f32 per row (add_rms_norm's e4m3 output).  `out_dtype`
    defaults to x's type, or bf16 for e4m3.  Meant for the few rows of a decode step: the weights are read at
    least once per 16 rows, and more often where so many rows do not fit in shared memory (16 f32 rows of 18944);
    for a prompt's many rows dequantise and use a matrix product.  The order of the sums goes by the number of
    rows."""
    dev = _device_of(x, "x")
    if stream is not None or dev != _current_device():
        with _on(stream, dev):
            return w4_matvec(x, weight, x_scales=x_scales, out=out, out_dtype=out_dtype)
    xc, xs = _rows(x, "x", _CODES, dev)
    m, k = x.shape
    if k != weight.k:
        raise ValueError(f"x has {k} columns, the weight {weight.k}")
    if (xc == L.MTN_DTYPE_E4M3) != (x_scales is not None):
        raise ValueError("x_scales go with float8_e4m3fn rows, and only with them")
    xsp = None if x_scales is None else _values(x_scales, "x_scales", m, dev)
    if out is None:
        out = torch.empty((m, weight.n), device=x.device,
                          dtype=out_dtype or (x.dtype if x_scales is None else torch.bfloat16))
    elif out_dtype is not None and out.dtype != out_dtype:
        raise ValueError("out and out_dtype disagree")
    oc, os_ = _rows(out, "out", _FLOATS, dev)
    if out.shape != (m, weight.n):
        raise ValueError("out must be [rows, n]")
    if weight.packed.get_device() != dev:
        raise ValueError(f"the weight is on {weight.device}, x on {x.device}")
    if m:
        st = L.lib().mtn_w4_matvec(x.data_ptr(), xc, xs, xsp, m, weight.packed.data_ptr(), weight.scales.data_ptr(),
                                   weight.n, k, weight.group, out.data_ptr(), oc, os_, _stream_of(dev))
        if st:
            L.check(st)
    return out
