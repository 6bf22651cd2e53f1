"""Products with 4-bit weights (mtn_w4_*) against the formula in 64 bits.

Exact cases: small integers in x, one power of two as every scale, and sums below 2^24 leave nothing to round, so
the result has to be bit-equal at every size.  f32 rows with one non-zero element of 24 significant bits and codes
that are powers of two likewise.

General cases, u = 2^-24: products of x (each a sum of at most three bf16 parts) with a code are exact; the sums run
in f32 over at least 16 elements at a time, each addition off by at most 2 u of the running sum of magnitudes
S = sum |x q s| (a tensor core may cut instead of rounding), then one product with the scale and at most 64 joins of
partial sums: |error| <= 4 (k / 16 + 64) u S, plus half a step of the output's type.
"""
from __future__ import annotations

import pytest
import torch

from mitten_b200 import _lib, dense, paged

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BF, F32, E4 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _codes(n, k, g):
    return torch.randint(-8, 8, (n, k), generator=g, device="cuda", dtype=torch.int8)


def _values(codes, scales, group):
    return codes.double() * scales.double().repeat_interleave(group, 1)[:, :codes.shape[1]]


SIZES = [(1, 1), (16, 128), (17, 129), (3, 31), (64, 64), (100, 1000), (512, 3584), (1, 3584), (2047, 96),
         (4873, 1000), (896, 896), (33, 18944), (8, 65536), (5000, 130), (128, 4864)]
ROWS = [1, 2, 5, 8, 9, 16, 17, 33]


@pytest.mark.parametrize("n,k", SIZES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("xd", [BF, F32, E4])
def test_integers_are_exact(cuda_device, n, k, group, xd):
    g = _gen(n * 7 + k + group)
    codes = _codes(n, k, g)
    scales = torch.full((n, -(-k // group)), 2.0 ** -5, device="cuda", dtype=BF)
    w = dense.W4Weight.from_codes(codes, scales, group)
    for m in ROWS:
        x = torch.randint(-4, 5, (m, k), generator=g, device="cuda").float()
        xs = None if xd != E4 else 2.0 ** torch.randint(-3, 4, (m,), generator=g, device="cuda").float()
        got = dense.w4_matvec(x.to(xd), w, x_scales=xs, out_dtype=F32)
        want = (x.double() @ codes.double().T) * 2.0 ** -5
        if xs is not None:
            want = want * xs.double()[:, None]
        assert torch.equal(got.double(), want), (m, (got.double() - want).abs().max())


@pytest.mark.parametrize("n,k,group", [(50, 300, 32), (512, 3584, 128), (77, 896, 64)])
def test_f32_rows_keep_all_their_bits(cuda_device, n, k, group):
    g = _gen(n)
    codes = torch.tensor([-8, -4, -2, -1, 1, 2, 4], dtype=torch.int8, device="cuda")[
        torch.randint(0, 7, (n, k), generator=g, device="cuda")]
    scales = (2.0 ** torch.randint(-6, 3, (n, -(-k // group)), generator=g, device="cuda").float()).to(BF)
    w = dense.W4Weight.from_codes(codes, scales, group)
    m = 7
    val = torch.randn(m, generator=g, device="cuda") * 10.0 ** torch.randint(-8, 9, (m,), generator=g, device="cuda").float()
    at = torch.randint(0, k, (m,), generator=g, device="cuda")
    at[0], at[1] = 0, k - 1
    x = torch.zeros(m, k, device="cuda")
    x[torch.arange(m, device="cuda"), at] = val
    got = dense.w4_matvec(x, w)
    want = val.double()[:, None] * _values(codes, scales, group).T[at]
    assert torch.equal(got.double(), want)


@pytest.mark.parametrize("n,k", [(1, 5), (512, 3584), (4873, 1000), (3584, 18944), (300, 4736), (18944, 896)])
@pytest.mark.parametrize("group,xd,od", [(32, F32, F32), (64, BF, F32), (128, BF, BF), (128, E4, BF), (64, E4, F32),
                                         (32, BF, BF), (128, F32, F32)])
def test_general_values(cuda_device, n, k, group, xd, od):
    g = _gen(n + k)
    codes = _codes(n, k, g)
    scales = (0.01 * (0.2 + torch.rand(n, -(-k // group), generator=g, device="cuda"))).to(BF)
    w = dense.W4Weight.from_codes(codes, scales, group)
    val = _values(codes, scales, group)
    for m in (1, 3, 8, 14, 20):
        x = torch.randn(m, k, generator=g, device="cuda")
        xs = x.abs().amax(1) / 448.0 if xd == E4 else None
        x = (x if xs is None else x / xs[:, None]).to(xd)
        got = dense.w4_matvec(x, w, x_scales=xs, out_dtype=od)
        xv = x.double() if xs is None else x.double() * xs.double()[:, None]
        want, mag = xv @ val.T, xv.abs() @ val.abs().T
        half = torch.finfo(od).eps / 2
        tol = 4 * (k / 16 + 64) * U * mag
        tol = tol + half * (want.abs() + tol)
        assert ((got.double() - want).abs() <= tol).all(), ((got.double() - want).abs() / tol).max()


# More than one pass of rows: slices of k over 1 to 8 CTAs, groups of every size, each of the row types.
@pytest.mark.parametrize("n,k", [(32768, 128), (3584, 1280), (2056, 2048), (18950, 256), (128, 32768), (37888, 384),
                                 (64, 65536), (70, 65536), (4099, 1024)])
@pytest.mark.parametrize("group,xd", [(32, BF), (64, E4), (128, F32), (128, BF), (32, F32), (64, BF), (32, E4)])
def test_more_than_sixteen_rows(cuda_device, n, k, group, xd):
    g = _gen(n + k + group)
    codes = _codes(n, k, g)
    scales = (0.01 * (0.2 + torch.rand(n, k // group, generator=g, device="cuda"))).to(BF)
    w = dense.W4Weight.from_codes(codes, scales, group)
    val = _values(codes, scales, group)
    ones = dense.W4Weight.from_codes(codes, torch.full_like(scales, 2.0 ** -5), group)
    for m in (17, 31, 32, 33, 70):
        big = torch.randn(m, k + 16, generator=g, device="cuda")
        xs = big.abs().amax(1) / 448.0 if xd == E4 else None
        x = (big if xs is None else big / xs[:, None]).to(xd)[:, 16:]  # rows with a stride
        out = torch.full((m + 1, n + 3), 7.0, device="cuda")
        dense.w4_matvec(x, w, x_scales=xs, out=out[:m, :n])
        assert (out[m] == 7).all() and (out[:, n:] == 7).all()
        xv = x.double() if xs is None else x.double() * xs.double()[:, None]
        want, mag = xv @ val.T, xv.abs() @ val.abs().T
        tol = 4 * (k / 16 + 64) * U * mag
        tol = tol + U * (want.abs() + tol)
        got = out[:m, :n].double()
        assert ((got - want).abs() <= tol).all(), (m, ((got - want).abs() / tol).max())
        again = dense.w4_matvec(x, w, x_scales=xs, out_dtype=F32)
        assert torch.equal(again, out[:m, :n])
        xi = torch.randint(-2, 3, (m, k), generator=g, device="cuda").float()  # sums of these are exact
        one = None if xd != E4 else torch.ones(m, device="cuda")
        got = dense.w4_matvec(xi.to(xd), ones, x_scales=one, out_dtype=F32)
        assert torch.equal(got.double(), (xi.double() @ codes.double().T) * 2.0 ** -5)
    assert paged.device_error(0) == (0, 0)


def test_more_than_sixteen_rows_with_values_that_are_none(cuda_device):
    g = _gen(3)
    codes, scales = _codes(4096, 1024, g), torch.full((4096, 8), 0.5, device="cuda", dtype=BF)
    scales[5, 2], scales[300, 0] = float("nan"), float("inf")
    codes[:, 700] = 3
    w = dense.W4Weight.from_codes(codes, scales, 128)
    x = torch.randn(20, 1024, generator=g, device="cuda").to(BF)
    want = dense.w4_matvec(x, w)
    x[3, 700], x[9, 700] = float("nan"), float("inf")
    got = dense.w4_matvec(x, w)
    other = [r for r in range(20) if r not in (3, 9)]
    assert torch.equal(got[other].nan_to_num(7, 8, 9), want[other].nan_to_num(7, 8, 9))
    assert got[:, 5].isnan().all() and got[3].isnan().all()
    fine = [c for c in range(4096) if c not in (5, 300)]
    assert (got[9][fine] == float("inf")).all() and not got[other][:, fine].isnan().any()
    # captured and replayed, behind and before a norm
    h, out = torch.empty_like(x[:, :1024]), torch.empty(20, 4096, device="cuda", dtype=BF)
    x = torch.randn(20, 1024, generator=g, device="cuda").to(BF)
    scales.fill_(0.5)
    w = dense.W4Weight.from_codes(codes, scales, 128)
    graph = torch.cuda.CUDAGraph()
    dense.add_rms_norm(x, out=h)
    want = dense.w4_matvec(h, w)
    want2 = dense.add_rms_norm(want)[0]
    h.zero_()
    res = torch.empty_like(want2)
    with torch.cuda.graph(graph):
        for _ in range(3):
            dense.add_rms_norm(x, out=h)
            dense.w4_matvec(h, w, out=out)
            dense.add_rms_norm(out, out=res)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(res, want2)


def test_same_result_every_time_and_for_rows_alone(cuda_device):
    g = _gen(9)
    codes, scales = _codes(1000, 3584, g), torch.rand(1000, 28, generator=g, device="cuda").to(BF)
    w = dense.W4Weight.from_codes(codes, scales, 128)
    x = torch.randn(8, 3584, generator=g, device="cuda").to(BF)
    first = dense.w4_matvec(x, w, out_dtype=F32)
    for _ in range(5):
        assert torch.equal(dense.w4_matvec(x, w, out_dtype=F32), first)


@pytest.mark.parametrize("n,k,group", [(64, 256, 128), (17, 130, 32), (300, 1000, 64), (1, 7, 128)])
@pytest.mark.parametrize("wd", [BF, F32])
def test_quantize_round_trip(cuda_device, n, k, group, wd):
    g = _gen(k)
    weight = torch.randn(n, k, generator=g, device="cuda").to(wd)
    weight[0] = 0.0
    w = dense.W4Weight.from_float(weight, group)
    val = w.dequantize(F32).double()
    ng = -(-k // group)
    pad = torch.zeros(n, ng * group, device="cuda", dtype=torch.float64)
    pad[:, :k] = weight.double()
    amax = pad.view(n, ng, group).abs().amax(2)
    # the scale is bf16(f32(max / 7)): half a step of each type
    s = (amax.float() / 7.0).to(BF).double().repeat_interleave(group, 1)[:, :k]
    # the code is the nearest one, off by at most half a scale; the f32 division adds an u of up to 8 codes
    assert ((val - weight.double()).abs() <= s * (0.5 + 8 * U + 7 * 2.0 ** -8)).all()
    assert (val[0] == 0).all()
    code = torch.where(s > 0, val / torch.where(s > 0, s, 1.0), 0.0)
    assert torch.equal(code, code.round()) and (code.abs() <= 8).all()
    assert torch.equal(w.dequantize(BF), w.dequantize(F32).to(BF))
    # packing those codes gives the same weights
    scales = (amax.float() / 7.0).to(BF)
    w2 = dense.W4Weight.from_codes(code.to(torch.int8), scales, group)
    assert torch.equal(w2.packed, w.packed) and torch.equal(w2.scales.view(torch.int16), w.scales.view(torch.int16))
    # and the product goes by them
    x = torch.randint(-2, 3, (3, k), generator=g, device="cuda").float()
    got, want = dense.w4_matvec(x, w).double(), x.double() @ val.T
    assert ((got - want).abs() <= 4 * (k / 16 + 64) * U * (x.double().abs() @ val.abs().T)).all()


def test_from_codes_clamps_and_takes_strides(cuda_device):
    big = torch.randint(-128, 128, (40, 200), device="cuda", dtype=torch.int8)
    sc = torch.rand(40, 9, device="cuda").to(BF)
    w = dense.W4Weight.from_codes(big[:, 3:163], sc[:, 1:6], 32)
    want = _values(big[:, 3:163].clamp(-8, 7), sc[:, 1:6], 32)
    assert torch.equal(w.dequantize().double(), want)
    out = torch.full((40, 170), 5.0, device="cuda")
    w.dequantize(out=out[:, 4:164])
    assert torch.equal(out[:, 4:164].double(), want) and (out[:, :4] == 5).all() and (out[:, 164:] == 5).all()


def test_non_finite_weights_and_rows(cuda_device):
    weight = torch.randn(32, 256, device="cuda")
    weight[3, 200] = float("inf")
    weight[5, 10] = float("nan")
    w = dense.W4Weight.from_float(weight, 64)
    x = torch.ones(4, 256, device="cuda")
    x[1, 7] = float("inf")
    x[2, 9] = float("nan")
    x[3, 11] = 3.4e38  # rounds to infinity in bf16, is finite in f32
    y = dense.w4_matvec(x, w)
    assert torch.isnan(y[:, 3]).all() and torch.isnan(y[:, 5]).all()
    ok = [j for j in range(32) if j not in (3, 5)]
    assert torch.isfinite(y[0, ok]).all() and torch.isnan(y[2]).all()
    val = w.dequantize()
    inf = x[1, 7] * val[:, 7]  # infinity times the weight's sign, or NaN for a weight of 0
    assert torch.equal(torch.isnan(y[1, ok]), torch.isnan(inf[ok]))
    keep = [j for j in ok if not torch.isnan(inf[j])]
    assert torch.equal(y[1, keep], inf[keep])
    want = x[3].double() @ val.double().T
    for j in ok:
        if abs(want[j].item()) < 3.4e38 and abs(val[j, 11].item()) < 0.9:
            assert torch.isfinite(y[3, j])


def test_strides_streams_and_replay(cuda_device):
    g = _gen(4)
    w = dense.W4Weight.from_float(torch.randn(130, 520, generator=g, device="cuda"), 64)
    xb = torch.randn(6, 700, generator=g, device="cuda")
    for xd, off in ((F32, 1), (F32, 4), (BF, 3), (BF, 8)):
        x = xb.to(xd)[:, off:off + 520]
        ob = torch.full((6, 200), 9.0, device="cuda")
        dense.w4_matvec(x, w, out=ob[:, 7:137])
        assert torch.equal(ob[:, 7:137], dense.w4_matvec(x.contiguous(), w, out_dtype=F32))
        assert (ob[:, :7] == 9).all() and (ob[:, 137:] == 9).all()
    x = xb[:, :520].contiguous()
    want = dense.w4_matvec(x, w)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = dense.w4_matvec(x, w, stream=s)
    s.synchronize()
    assert torch.equal(got, want)
    out, xi = torch.empty_like(want), x.clone()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        dense.w4_matvec(xi, w, out=out)
    xi.copy_(x.flip(0))
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want.flip(0))
    assert dense.w4_matvec(x[:0], w).shape == (0, 130)


def test_wrapper_refuses(cuda_device):
    w = dense.W4Weight.from_float(torch.randn(16, 64, device="cuda"), 64)
    x = torch.randn(2, 64, device="cuda")
    for args, kw in [((x[:, :63], w), {}), ((x.half(), w), {}), ((x.to(E4), w), {}), ((x[0], w), {}),
                     ((x.to(E4), w), dict(x_scales=torch.ones(3, device="cuda"))),
                     ((x, w), dict(x_scales=torch.ones(2, device="cuda"))),
                     ((x, w), dict(out=torch.empty(2, 17, device="cuda"))),
                     ((x, w), dict(out=torch.empty(2, 16, device="cuda"), out_dtype=BF)),
                     ((x, w), dict(out_dtype=torch.float16)), ((x.cpu(), w), {}),
                     ((x.T.contiguous().T, w), {})]:
        with pytest.raises((ValueError, KeyError)):
            dense.w4_matvec(*args, **kw)
    with pytest.raises(ValueError):
        dense.W4Weight.from_float(torch.randn(16, 64, device="cuda"), 48)
    with pytest.raises(ValueError):
        dense.W4Weight.from_codes(torch.zeros(4, 64, dtype=torch.int8, device="cuda"), torch.zeros(4, 2, device="cuda").to(BF), 64)
    with pytest.raises(_lib.MittenError):
        dense.w4_matvec(torch.zeros(70000, 64, device="cuda"), w)
    assert paged.device_error(0) == (0, 0)
