"""add_rms_norm (mtn_add_rms_norm) against the formula in 64 bits.

Tolerances, from the arithmetic (u = 2^-24, f32's half step):
  sum   one f32 addition and one rounding: bit-equal to the same two steps in torch;
  y     the sum of squares adds positive terms, so whatever the order over at least 32 threads its relative error
        is at most (hidden / 32 + 40) u; the root halves it, and the mean, the root, the reciprocal and the two
        products round at most 6 times more: (hidden / 64 + 26) u, plus half a step of the output's type;
  e4m3  the code is y / scale with half a step of 2^-4 relative, or half of the smallest step (2^-9) near zero,
        in units of the scale; y's own error and the two roundings of the division and the scale come on top.
"""
from __future__ import annotations

import pytest
import torch

from mitten_b200 import dense, paged

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BF, F32, E4 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _inputs(n, hidden, xd, rd, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, hidden, generator=g, device="cuda").to(xd)
    r = None if rd is None else (3.0 * torch.randn(n, hidden, generator=g, device="cuda")).to(rd)
    w1 = 1.0 + 0.3 * torch.randn(hidden, generator=g, device="cuda")
    return x, r, w1


def _check(x, r, w1, eps, total, out, scales):
    hidden = x.shape[1]
    if r is not None:
        want = (x.float() + r.float()).to(r.dtype)
        assert torch.equal(total, want)
        s = want.double()
    else:
        s = x.double()
    y = s / torch.sqrt(s.square().mean(1, keepdim=True) + eps)
    if w1 is not None:
        y = y * w1.double()
    rel = (hidden / 64 + 26) * U
    if out.dtype == E4:
        scale = torch.clamp(y.abs().amax(1) / 448.0, min=2.0 ** -100)
        assert ((scales.double() - scale).abs() <= scale * (rel + 2 * U)).all()
        got = out.double() * scales.double()[:, None]
        tol = y.abs() * (2.0 ** -4 * (1 + 4 * rel) + rel + 4 * U) + scale[:, None] * (2.0 ** -10 * (1 + 4 * rel) + 2 * U)
        assert ((got - y).abs() <= tol).all()
    else:
        half = torch.finfo(out.dtype).eps / 2
        assert ((out.double() - y).abs() <= y.abs() * (rel + half * (1 + rel))).all()


SHAPES = [(1, 1), (3, 2), (1, 896), (7, 33), (5, 1000), (64, 3584), (9, 2049), (33, 64), (130, 257), (2, 16384),
          (3, 18944), (1, 32768), (400, 1024), (300, 1032)]


@pytest.mark.parametrize("n,hidden", SHAPES)
@pytest.mark.parametrize("xd,rd,od", [(BF, BF, BF), (BF, BF, E4), (F32, F32, F32), (F32, BF, BF), (BF, F32, F32),
                                      (F32, F32, E4), (BF, None, BF), (F32, None, E4), (BF, None, F32)])
def test_norm_matches_the_formula(cuda_device, n, hidden, xd, rd, od):
    x, r, w1 = _inputs(n, hidden, xd, rd, n + hidden)
    keep = None if r is None else r.clone()
    total = None if r is None else torch.empty_like(r)
    out, scales = dense.add_rms_norm(x, w1, 1e-6, residual=r, sum_out=total, out_dtype=od)
    _check(x, keep, w1, 1e-6, total, out, scales)
    if r is not None:
        assert torch.equal(r, keep)  # the residual itself is left alone when the sum goes elsewhere
        got, sc2 = dense.add_rms_norm(x, w1, 1e-6, residual=r, out_dtype=od)  # in place
        assert torch.equal(r, total) and torch.equal(got.view(torch.uint8), out.view(torch.uint8))
        assert scales is None or torch.equal(sc2, scales)


@pytest.mark.parametrize("hidden,pad,off", [(896, 8, 0), (896, 3, 1), (128, 1, 5), (3584, 16, 8), (2051, 7, 2),
                                            (1024, 4, 4)])
@pytest.mark.parametrize("xd,od", [(BF, BF), (F32, F32), (BF, E4)])
def test_strided_and_unaligned_rows(cuda_device, hidden, pad, off, xd, od):
    n = 11
    big = torch.randn(n, hidden + pad + off, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    xb, rb = big.to(xd), (2.0 * big.flip(1)).to(BF)
    x, r = xb[:, off:off + hidden], rb[:, off:off + hidden]
    keep_r, sentinel = r.clone(), rb.clone()
    ob = torch.full((n, hidden + pad + off), 7.0, device="cuda").to(od)
    out = ob[:, off:off + hidden]
    _, scales = dense.add_rms_norm(x, None, 1e-5, residual=r, out=out)
    _check(x, keep_r, None, 1e-5, r, out, scales)
    # what lies beside the rows stays as it was
    side = torch.ones(hidden + pad + off, dtype=torch.bool, device="cuda")
    side[off:off + hidden] = False
    assert torch.equal(rb[:, side], sentinel[:, side])
    assert (ob.float()[:, side] == 7.0).all()


def test_empty_zero_and_non_finite_rows(cuda_device):
    assert dense.add_rms_norm(torch.empty(0, 64, device="cuda"))[0].shape == (0, 64)
    for hidden in (64, 3584):
        x = torch.randn(6, hidden, device="cuda")
        x[1] = 0.0
        x[2, 5] = float("nan")
        x[3, 7] = float("inf")
        x[4] *= 1e-30
        for od in (F32, BF, E4):
            out, scales = dense.add_rms_norm(x, None, 1e-6, out_dtype=od)
            o = out.float() if scales is None else out.float() * scales[:, None]
            assert (o[1] == 0).all()
            assert torch.isnan(o[2]).all()
            assert torch.isnan(o[3, 7])
            for row in (0, 4, 5):
                assert torch.isfinite(o[row]).all()
                _check(x[row:row + 1], None, None, 1e-6, None, out[row:row + 1],
                       None if scales is None else scales[row:row + 1])
            if scales is not None:
                assert scales[1].item() == 2.0 ** -100 and torch.isnan(scales[2]) and torch.isnan(scales[3])


def test_other_stream_and_captured_replay(cuda_device):
    x, r, w1 = _inputs(17, 3584, BF, BF, 3)
    want, wsc = dense.add_rms_norm(x, w1, residual=r.clone(), out_dtype=E4)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    r1 = r.clone()
    s.wait_stream(torch.cuda.current_stream())
    got, sc = dense.add_rms_norm(x, w1, residual=r1, out_dtype=E4, stream=s)
    s.synchronize()
    assert torch.equal(got.view(torch.uint8), want.view(torch.uint8)) and torch.equal(sc, wsc)
    r2, out, sco = r.clone(), torch.empty_like(want), torch.empty_like(wsc)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dense.add_rms_norm(x, w1, residual=r2, out=out, scales=sco)
    x.copy_(x.flip(0))
    want, wsc = dense.add_rms_norm(x, w1, residual=r.clone(), out_dtype=E4)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out.view(torch.uint8), want.view(torch.uint8)) and torch.equal(sco, wsc)


def test_results_on_another_stream_are_not_written_by_work_still_queued(cuda_device):
    # memory freed with a fill still queued on the current stream must not become a result on another one
    x, _, w1 = _inputs(64, 1024, F32, None, 5)
    want = dense.add_rms_norm(x, w1)[0]
    w = dense.W4Weight.from_float(torch.randn(1024, 1024, device="cuda"), 128)
    values, y = w.dequantize(), dense.w4_matvec(x, w)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for call, ref in ((lambda: dense.add_rms_norm(x, w1, stream=s)[0], want), (lambda: w.dequantize(stream=s), values),
                      (lambda: dense.w4_matvec(x, w, stream=s), y)):
        freed = torch.empty_like(ref)
        torch.cuda._sleep(20_000_000)
        freed.fill_(7.0)
        del freed
        got = call()
        torch.cuda.synchronize()
        assert torch.equal(got, ref)


def test_wrapper_refuses(cuda_device):
    x = torch.zeros(4, 64, device="cuda")
    bad = [dict(w1=torch.ones(63, device="cuda")), dict(w1=torch.ones(64, device="cuda", dtype=BF)),
           dict(w1=torch.ones(64)), dict(residual=torch.zeros(4, 63, device="cuda")),
           dict(residual=torch.zeros(4, 64, device="cuda").half()), dict(sum_out=x),
           dict(out=torch.zeros(4, 64, device="cuda").half()), dict(out=torch.zeros(5, 64, device="cuda")),
           dict(out=torch.zeros(4, 64, device="cuda"), out_dtype=BF), dict(scales=torch.zeros(4, device="cuda")),
           dict(out_dtype=E4, scales=torch.zeros(3, device="cuda")), dict(residual=torch.zeros(64, 4, device="cuda").T)]
    for kw in bad:
        with pytest.raises(ValueError):
            dense.add_rms_norm(x, **kw)
    with pytest.raises(ValueError):
        dense.add_rms_norm(torch.zeros(64, device="cuda"))
    with pytest.raises(ValueError):  # rows that share memory
        dense.add_rms_norm(torch.zeros(64, device="cuda").expand(4, 64))
    assert paged.device_error(0) == (0, 0)


@pytest.mark.parametrize("hidden", [256, 259, 2048, 2055])
@pytest.mark.parametrize("xd", [BF, F32])
def test_e4m3_codes_are_those_of_the_quotient(cuda_device, hidden, xd):
    """Rows of signs with eps 0 have y = w1, exactly, and with a scale s of 16 bits w1 = 448 s and w1 = t s are exact
    for every t halfway between two codes: y / s is t without rounding, and the code is the even neighbour's."""
    codes = torch.arange(0x7f, dtype=torch.uint8).view(E4).float()  # every finite value from 0 on
    half = (codes[:-1] + codes[1:]) / 2
    want = half.to(E4).float()
    g = torch.Generator().manual_seed(hidden)
    sign = torch.randint(0, 2, (3, hidden), generator=g).float() * 2 - 1
    at = torch.arange(hidden - 1) % len(half)
    for s in torch.randint(1 << 15, 1 << 16, (40,), generator=g).tolist():
        s *= 2.0 ** -20
        w1 = torch.cat([torch.tensor([448.0]), half[at]]) * s
        out, scales = dense.add_rms_norm(sign.to(xd).cuda(), w1.cuda(), 0.0, out_dtype=E4)
        assert (scales == s).all()
        assert torch.equal(out.float().cpu(), sign * torch.cat([torch.tensor([448.0]), want[at]]))


@pytest.mark.parametrize("hidden", [256, 259, 2048])
def test_e4m3_rows_of_infinite_values(cuda_device, hidden):
    x = torch.ones(2, hidden, device="cuda")
    x[1] = -1.0
    w1 = torch.rand(hidden, device="cuda") + 0.5
    w1[3] = float("inf")
    out, scales = dense.add_rms_norm(x, w1, 0.0, out_dtype=E4)
    assert (scales == float("inf")).all()  # the quotients: 0, and NaN for infinity over infinity
    o = out.float()
    assert o[:, 3].isnan().all() and (o[:, :3] == 0).all() and (o[:, 4:] == 0).all()
