"""The dense entry points refuse bad arguments before they launch anything (CPU: no pointer is dereferenced)."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from mitten_b200 import _lib, dense

FAKE = [C.c_void_p(0x100000 * (i + 1)) for i in range(6)]


def _norm(x=FAKE[0], x_dtype=_lib.MTN_DTYPE_BF16, x_stride=64, residual=FAKE[1], res_stride=64, sum_=FAKE[2],
          sum_stride=64, res_dtype=_lib.MTN_DTYPE_BF16, w1=None, eps=1e-6, n=2, hidden=64, out=FAKE[3],
          out_dtype=_lib.MTN_DTYPE_BF16, out_stride=64, scales=None):
    return _lib.lib().mtn_add_rms_norm(x, x_dtype, x_stride, residual, res_stride, sum_, sum_stride, res_dtype, w1, eps,
                                       n, hidden, out, out_dtype, out_stride, scales, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(n=-1), b"bad row count"),
    (dict(hidden=0), b"hidden 0"),
    (dict(hidden=32769, x_stride=40000, out_stride=40000, res_stride=40000, sum_stride=40000), b"hidden 32769"),
    (dict(x_dtype=_lib.MTN_DTYPE_E4M3), b"bad x dtype"),
    (dict(res_dtype=9), b"bad residual dtype"),
    (dict(out_dtype=9), b"bad out dtype"),
    (dict(eps=-1.0), b"eps"),
    (dict(eps=float("nan")), b"eps"),
    (dict(x=None), b"null pointer"),
    (dict(out=None), b"null pointer"),
    (dict(sum_=None), b"come together"),
    (dict(residual=None), b"come together"),
    (dict(scales=FAKE[4]), b"scales go with"),
    (dict(out_dtype=_lib.MTN_DTYPE_E4M3), b"scales go with"),
    (dict(out=FAKE[0]), b"overlap"),
    (dict(sum_=FAKE[0]), b"overlap"),
    (dict(x_stride=63), b"strides"),
    (dict(out_stride=63), b"strides"),
    (dict(sum_stride=63), b"strides"),
    (dict(x=C.c_void_p(0x100001)), b"not aligned"),
    (dict(out=C.c_void_p(0x400002), out_dtype=_lib.MTN_DTYPE_F32), b"not aligned"),
    (dict(w1=C.c_void_p(0x500002)), b"not aligned"),
])
def test_norm_refuses(kw, msg):
    assert _norm(**kw) == _lib.MTN_EINVAL
    assert msg in _lib.lib().mtn_last_error()


def test_norm_without_rows_is_nothing_to_do():
    assert _norm(n=0) == _lib.MTN_OK


def test_norm_wrapper_refuses_cpu_tensors():
    with pytest.raises(ValueError, match="CUDA tensor"):
        dense.add_rms_norm(torch.zeros(2, 64))


def _matvec(x=FAKE[0], x_dtype=_lib.MTN_DTYPE_BF16, x_stride=128, xs=None, m=2, packed=FAKE[1], scales=FAKE[2], n=32,
            k=128, group=64, out=FAKE[3], out_dtype=_lib.MTN_DTYPE_F32, out_stride=32):
    return _lib.lib().mtn_w4_matvec(x, x_dtype, x_stride, xs, m, packed, scales, n, k, group, out, out_dtype, out_stride,
                                    None)


@pytest.mark.parametrize("kw,msg", [
    (dict(n=0), b"out of range"), (dict(k=0), b"out of range"), (dict(k=65537, x_stride=70000), b"out of range"),
    (dict(group=48), b"group 48"), (dict(m=-1), b"row count"), (dict(m=65536), b"row count"),
    (dict(x_dtype=7), b"bad x dtype"), (dict(out_dtype=_lib.MTN_DTYPE_E4M3), b"bad out dtype"),
    (dict(x=None), b"null pointer"), (dict(packed=None), b"null pointer"), (dict(out=None), b"null pointer"),
    (dict(x_dtype=_lib.MTN_DTYPE_E4M3), b"x_scales"), (dict(xs=FAKE[4]), b"x_scales"),
    (dict(x_stride=127), b"strides"), (dict(out_stride=31), b"strides"),
    (dict(packed=C.c_void_p(0x100008)), b"aligned"), (dict(scales=C.c_void_p(0x100004)), b"aligned"),
    (dict(out=FAKE[0]), b"overlaps"),
    (dict(x=C.c_void_p(0x100001)), b"not aligned"), (dict(out=C.c_void_p(0x400002)), b"not aligned"),
])
def test_w4_matvec_refuses(kw, msg):
    assert _matvec(**kw) == _lib.MTN_EINVAL
    assert msg in _lib.lib().mtn_last_error()


def test_w4_matvec_without_rows_is_nothing_to_do():
    assert _matvec(m=0) == _lib.MTN_OK


def test_w4_sizes():
    lib = _lib.lib()
    assert lib.mtn_w4_packed_bytes(16, 128) == 1024 and lib.mtn_w4_packed_bytes(17, 129) == 32 * 256 // 2
    assert lib.mtn_w4_scales_bytes(16, 128, 32) == 16 * 4 * 2 and lib.mtn_w4_scales_bytes(17, 129, 128) == 32 * 2 * 2
    for bad in ((0, 128), (16, 0), (16, 65537), (-1, 5)):
        assert lib.mtn_w4_packed_bytes(*bad) == 0
    assert lib.mtn_w4_scales_bytes(16, 128, 16) == 0
    # [152064, 65536] needs offsets beyond 32 bits
    assert lib.mtn_w4_packed_bytes(152064, 65536) == 152064 * 32768


@pytest.mark.parametrize("call,msg", [
    (lambda lib: lib.mtn_w4_quantize(None, 0, 64, 4, 64, 64, FAKE[0], FAKE[1], None), b"null"),
    (lambda lib: lib.mtn_w4_quantize(FAKE[2], 2, 64, 4, 64, 64, FAKE[0], FAKE[1], None), b"dtype"),
    (lambda lib: lib.mtn_w4_quantize(FAKE[2], 0, 63, 4, 64, 64, FAKE[0], FAKE[1], None), b"stride"),
    (lambda lib: lib.mtn_w4_quantize(FAKE[2], 0, 64, 4, 64, 64, C.c_void_p(8), FAKE[1], None), b"aligned"),
    (lambda lib: lib.mtn_w4_pack(FAKE[2], 64, FAKE[3], 0, 4, 64, 64, FAKE[0], FAKE[1], None), b"stride"),
    (lambda lib: lib.mtn_w4_pack(FAKE[2], 64, None, 1, 4, 64, 64, FAKE[0], FAKE[1], None), b"null"),
    (lambda lib: lib.mtn_w4_dequantize(FAKE[0], FAKE[1], 4, 64, 64, None, 0, 64, None), b"null"),
    (lambda lib: lib.mtn_w4_dequantize(FAKE[0], FAKE[1], 4, 64, 64, FAKE[2], 2, 64, None), b"dtype"),
    (lambda lib: lib.mtn_w4_dequantize(FAKE[0], FAKE[1], 4, 64, 63, FAKE[2], 0, 64, None), b"group"),
])
def test_w4_layout_calls_refuse(call, msg):
    assert call(_lib.lib()) == _lib.MTN_EINVAL
    assert msg in _lib.lib().mtn_last_error()


@pytest.mark.parametrize("call", [
    lambda lib: lib.mtn_w4_quantize(C.c_void_p(0x300002), _lib.MTN_DTYPE_F32, 64, 4, 64, 64, FAKE[0], FAKE[1], None),
    lambda lib: lib.mtn_w4_quantize(C.c_void_p(0x300001), _lib.MTN_DTYPE_BF16, 64, 4, 64, 64, FAKE[0], FAKE[1], None),
    lambda lib: lib.mtn_w4_pack(FAKE[2], 64, C.c_void_p(0x400001), 1, 4, 64, 64, FAKE[0], FAKE[1], None),
    lambda lib: lib.mtn_w4_dequantize(FAKE[0], FAKE[1], 4, 64, 64, C.c_void_p(0x300002), _lib.MTN_DTYPE_F32, 64, None),
    lambda lib: lib.mtn_w4_dequantize(FAKE[0], FAKE[1], 4, 64, 64, C.c_void_p(0x300001), _lib.MTN_DTYPE_BF16, 64, None),
])
def test_w4_layout_calls_refuse_pointers_between_elements(call):
    assert call(_lib.lib()) == _lib.MTN_EINVAL
    assert b"not aligned" in _lib.lib().mtn_last_error()


@pytest.mark.parametrize("kw", [dict(sum_stride=128), dict(res_stride=128)])
def test_norm_in_place_needs_equal_strides(kw):
    # row 1 of the sum would be row 2 of the residual, which another CTA may not have read yet
    assert _norm(sum_=FAKE[1], n=3, **kw) == _lib.MTN_EINVAL
    assert b"equal strides" in _lib.lib().mtn_last_error()
