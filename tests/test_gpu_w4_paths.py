"""The forms of mtn_w4_matvec that only large matrices reach: two row units a step for few rows, and several rounds of
row units within a split of k.  Small integers and scales of 2^-5 leave nothing to round, so results are exact.

The choices are restated from csrc/w4.cu, with its constants, so that a change there cannot leave these forms untested
without a test that says so."""
from __future__ import annotations

import re
from pathlib import Path

import pytest
import torch

from mitten_b200 import dense, paged

pytestmark = pytest.mark.gpu
BF, F32, E4 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
SOURCE = (Path(__file__).resolve().parents[1] / "mitten_b200" / "csrc" / "w4.cu").read_text()


def _constant(name: str) -> int:
    factors = re.search(rf"constexpr \w+ {name} = ([\d* ]+);", SOURCE).group(1)
    out = 1
    for f in factors.split("*"):
        out *= int(f)
    return out


def _steps(n, k):
    return -(-n // 16), -(-k // 128)  # row units, steps of 128 k


def _rounds(m, n, k, group, parts, sms):
    """The fewest rounds of a cluster over every split of k that fits and any number of resident clusters."""
    units, ks = _steps(n, k)
    units = -(-units // 2)  # more than 8 rows: two units a step
    warps = _constant("kMvWarps")
    ring, slot = warps * 2 * 2 * (1024 + 32 * (128 // group)), 16 * 2 * 16 * 4
    least = None
    for s in (1, 2, 4, 8):
        x = -(-parts * m * (-(-ks // s) * 128 + _constant("kXPad")) * 2 // 128) * 128
        if x + ring + (warps + (_constant("kMinUnits") if s > 1 else 0)) * slot > _constant("kSmemMax"):
            continue
        room = min((_constant("kSmemMax") - x - ring) // slot - warps, ring // slot)
        rounds = 1 if s == 1 else -(-(-(-units // (sms // s))) // room)
        least = rounds if least is None else min(least, rounds)
    return least


def _check(m, n, k, group, xd, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(-8, 8, (n, k), generator=g, device="cuda", dtype=torch.int8)
    w = dense.W4Weight.from_codes(codes, torch.full((n, -(-k // group)), 2.0 ** -5, device="cuda", dtype=BF), group)
    val = codes.double()
    top = 256 if xd == F32 and k < 4096 else 4  # two of an f32 row's three parts; sums stay below 2^24
    for rows in m:
        x = torch.randint(-top - 1, top + 2, (rows, k), generator=g, device="cuda").float()
        xs = None if xd != E4 else 2.0 ** torch.randint(-3, 4, (rows,), generator=g, device="cuda").float()
        out = torch.full((rows + 1, n + 5), 7.0, device="cuda")
        dense.w4_matvec(x.to(xd), w, x_scales=xs, out=out[:rows, :n])
        want = (x.double() @ val.T) * 2.0 ** -5
        if xs is not None:
            want = want * xs.double()[:, None]
        assert torch.equal(out[:rows, :n].double(), want), rows
        assert (out[rows] == 7).all() and (out[:, n:] == 7).all()
    assert paged.device_error(0) == (0, 0)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("xd", [BF, E4])
def test_few_rows_of_a_vocabulary_sized_matrix(cuda_device, group, xd):
    n, k = 43329, 3584  # an odd number of row units, the last with one row
    units, ks = _steps(n, k)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert units % 2 == 1 and units * ks >= _constant("kSteps2") * _constant("kMvWarps") * sms
    _check((1, 5, 8), n, k, group, xd, group)


@pytest.mark.parametrize("m,n,k,group,xd", [(16, 18944, 18944, 128, BF), (16, 18944, 18944, 32, E4),
                                            (16, 75001, 3584, 64, F32), (16, 75001, 3584, 128, F32)])
def test_rounds_within_a_split_of_k(cuda_device, m, n, k, group, xd):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert _rounds(m, n, k, group, 3 if xd == F32 else 1, sms) > 1
    _check((m, m - 1), n, k, group, xd, n)


def test_a_row_alone_and_in_a_batch(cuda_device):
    """The split of k, and with it the order of the sums, goes by the number of rows: a row alone agrees with the same
    row in a batch within both sums' bounds, 4 (k / 16 + 64) u of the magnitudes' sum each."""
    g = torch.Generator(device="cuda").manual_seed(9)
    n, k = 1000, 3584
    codes = torch.randint(-8, 8, (n, k), generator=g, device="cuda", dtype=torch.int8)
    scales = torch.rand(n, 28, generator=g, device="cuda").to(BF)
    w = dense.W4Weight.from_codes(codes, scales, 128)
    val = codes.double() * scales.double().repeat_interleave(128, 1)
    for xd in (BF, F32):
        x = torch.randn(16, k, generator=g, device="cuda").to(xd)
        tol = 8 * (k / 16 + 64) * 2.0 ** -24 * (x.double().abs() @ val.abs().T)
        for rows in (8, 16):
            batch = dense.w4_matvec(x[:rows], w, out_dtype=F32).double()
            for i in (0, rows - 1):
                alone = dense.w4_matvec(x[i:i + 1], w, out_dtype=F32).double()
                assert ((alone[0] - batch[i]).abs() <= tol[i]).all(), (xd, rows, i)
