"""process_logits (mtn_process_logits) against the rules applied one operation after the other on the CPU: in f32
with every operation rounded, where the kernel has to agree bit for bit, and in 64 bits, where its at most five
roundings (quotient or product, frequency product, three sums) are each off by half a step of the largest value
that meets them.  Greedy tokens have to be those of argmax_rows on the processed rows."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from mitten_b200 import _lib, paged

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _case(rng, rows, vocab, hist, bias, mask, frequent=0.5):
    """Host lists of the rules of each row."""
    c = {"hist": None, "bias": None, "mask": None}
    if hist is not None:
        lens = rng.integers(0, hist + 1, rows)
        lens[-1] = hist
        toks = [np.where(rng.random(n) < frequent, rng.integers(0, min(vocab, 5), n), rng.integers(0, vocab, n))
                for n in lens]
        c["hist"] = [t.astype(np.int32) for t in toks]
        c["prompt"] = np.array([rng.integers(0, n + 1) for n in lens], np.int32)
        c["rep"] = rng.uniform(0.7, 1.6, rows).astype(np.float32)
        c["pres"] = rng.uniform(-0.5, 1.0, rows).astype(np.float32)
        c["freq"] = rng.uniform(-0.2, 0.5, rows).astype(np.float32)
    if bias is not None:
        lens = rng.integers(0, bias + 1, rows)
        c["bias"] = [(rng.integers(0, vocab, n).astype(np.int32), rng.standard_normal(n).astype(np.float32) * 5)
                     for n in lens]
        for t, v in c["bias"]:
            if len(t) > 2:
                t[-1] = t[0]  # listed twice
                v[1] = -np.inf
    if mask is not None:
        allow = rng.random((mask, vocab)) < np.linspace(0.0, 1.0, mask)[:, None]
        c["mask"], c["mask_rows"] = allow, rng.integers(-1, mask, rows).astype(np.int32)
    return c


def _pack(allow):
    n, vocab = allow.shape
    words = -(-vocab // 32)
    b = np.zeros((n, words * 32), np.uint8)
    b[:, :vocab] = allow
    return np.packbits(b, axis=1, bitorder="little").view(np.int32).reshape(n, words)


def _csr(lists, dtype):
    ptr = np.concatenate([[0], np.cumsum([len(x) for x in lists])]).astype(np.int32)
    return torch.from_numpy(ptr).cuda(), torch.from_numpy(np.concatenate(lists).astype(dtype)).cuda()


def _rules(c):
    kw = {}
    if c["hist"] is not None:
        kw["hist_indptr"], kw["hist_tokens"] = _csr(c["hist"], np.int32)
        for a, b in (("prompt_lens", "prompt"), ("repetition", "rep"), ("presence", "pres"), ("frequency", "freq")):
            kw[a] = torch.from_numpy(c[b]).cuda()
    if c["bias"] is not None:
        kw["bias_indptr"], kw["bias_tokens"] = _csr([t for t, _ in c["bias"]], np.int32)
        kw["bias_values"] = _csr([v for _, v in c["bias"]], np.float32)[1]
    if c["mask"] is not None:
        kw["mask"] = torch.from_numpy(_pack(c["mask"])).cuda()
        kw["mask_rows"] = torch.from_numpy(c["mask_rows"]).cuda()
    return paged.LogitsRules(**kw)


def _want(x, c, dtype):
    """The rules in `dtype`, and the largest magnitude an operation met per element."""
    x = x.astype(dtype).copy()
    big = np.abs(x)
    with np.errstate(invalid="ignore"):
        for r in range(x.shape[0]):
            row = x[r]
            if c["hist"] is not None:
                h = c["hist"][r]
                seen = np.zeros(row.size, bool)
                seen[h] = True
                made = np.bincount(h[c["prompt"][r]:], minlength=row.size).astype(dtype)
                rep, fr, pr = (dtype(c[k][r]) for k in ("rep", "freq", "pres"))
                row = np.where(seen, np.where(row > 0, row / rep, row * rep), row)
                big[r] = np.fmax(big[r], np.abs(row))
                row = np.where(seen, row - fr * made, row)
                row = np.where(made > 0, row - pr, row)
                big[r] = np.fmax(big[r], np.abs(row)) + np.abs(fr * made) + abs(pr)
            if c["bias"] is not None:
                add = np.zeros(row.size, dtype)
                has = np.zeros(row.size, bool)
                for t, v in zip(*c["bias"][r]):
                    add[t], has[t] = v, True
                row = np.where(has, row + add, row)
                big[r] = big[r] + np.where(np.isfinite(add), np.abs(add), 0)
            if c["mask"] is not None and c["mask_rows"][r] >= 0:
                row = np.where(c["mask"][c["mask_rows"][r]], row, dtype(-np.inf))
            x[r] = row
    return x, big


def _check(x, c, rules, in_place=False):
    lg = x.cuda()
    xf = x.float().numpy()
    out, tok = paged.process_logits(lg, rules, out=lg if in_place else None, greedy=True)
    got = out.cpu().numpy()
    want, _ = _want(xf, c, np.float32)
    assert np.array_equal(got, want, equal_nan=True)
    w64, big = _want(xf, c, np.float64)
    # Half a step holds for results within f32's range: -max * 1.5 rounds to -inf in f32 (the step-by-step f32
    # comparison above covers those), so only elements whose operations all stay within it are measured.
    fin = np.isfinite(w64) & (big * (1 + 8 * U) <= np.finfo(np.float32).max)
    assert (np.abs(got[fin] - w64[fin]) <= 6 * U * big[fin] * 2).all()
    assert np.array_equal(tok.cpu().numpy(), paged.argmax_rows(out.contiguous()).cpu().numpy())
    best = [int(np.argmax(np.where(np.isnan(r), -np.inf, r))) if np.any(r > -np.inf) else 0 for r in want]
    assert tok.cpu().numpy().tolist() == best


@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 31), (3, 1000), (2, 4097), (5, 8192), (4, 8193), (2, 50001),
                                        (1, 151936), (7, 32768), (37, 16385)])
@pytest.mark.parametrize("hist,bias,mask", [(200, None, None), (None, 20, None), (None, None, 4), (300, 40, 5),
                                            (0, 0, 1), (5000, None, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rules_match(cuda_device, rows, vocab, hist, bias, mask, dtype):
    rng = np.random.default_rng(rows * 1000 + vocab)
    c = _case(rng, rows, vocab, hist, bias, mask)
    x = torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32) * 3).to(dtype)
    _check(x, c, _rules(c))
    if dtype == torch.float32:
        _check(x, c, _rules(c), in_place=True)
    assert paged.device_error(0) == (0, 0)


@pytest.mark.parametrize("vocab", [300, 20000])
def test_values_that_do_not_compare(cuda_device, vocab):
    rng = np.random.default_rng(vocab)
    c = _case(rng, 8, vocab, 100, 10, 3)
    c["mask_rows"][:] = [0, 1, 2, -1, 0, 1, 2, -1]
    x = rng.standard_normal((8, vocab)).astype(np.float32)
    x[:, ::7], x[:, 3::11], x[:, 5::13] = np.nan, -np.inf, np.inf
    x[4] = -np.inf
    x[5] = np.nan
    x[6] = np.finfo(np.float32).min
    x[7] = np.where(np.arange(vocab) % 2, -0.0, 0.0)
    c["hist"][7] = np.zeros(0, np.int32)
    c["prompt"][7] = 0
    c["bias"][7] = (np.zeros(0, np.int32), np.zeros(0, np.float32))
    _check(torch.from_numpy(x), c, _rules(c))


def test_ties_go_to_the_lowest_index(cuda_device):
    x = torch.zeros(3, 40000)
    x[0, [9000, 30000, 39999]] = 2.0
    x[1] = 1.0
    x[2, 20000] = -1.0
    x[2, :20000] = -2.0
    x[2, 20001:] = -1.0
    _, tok = paged.process_logits(x.cuda(), paged.LogitsRules(), greedy=True)
    assert tok.tolist() == [9000, 0, 20000]


@pytest.mark.filterwarnings("ignore::RuntimeWarning")
@pytest.mark.parametrize("kind", ["distinct", "repeats"])
@pytest.mark.parametrize("n", [500, 16384, 16385, 40000])
def test_long_histories(cuda_device, kind, n):
    """Histories of many steps of the sorting kernel: all different, and few that repeat."""
    rng = np.random.default_rng(n)
    vocab = 150001
    c = _case(rng, 3, vocab, 50, 40, 2)
    pick = rng.choice(7, n) * 1000 if kind == "repeats" else rng.permutation(vocab)[:n]
    c["hist"][1] = pick.astype(np.int32)
    c["prompt"][1] = len(pick) // 3
    _check(torch.from_numpy(rng.standard_normal((3, vocab)).astype(np.float32) * 3), c, _rules(c))
    assert paged.device_error(0) == (0, 0)


def test_vocabulary_of_more_chunks_than_buckets(cuda_device):
    rng = np.random.default_rng(6)
    vocab = 40_000_003
    c = _case(rng, 1, vocab, 3000, 100, None)
    x = torch.randn(1, vocab)
    x[0, 39_999_999] = 50.0
    _check(x, c, _rules(c))


@pytest.mark.parametrize("off,pad", [(0, 3), (1, 0), (2, 5), (3, 1), (4, 4), (5, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_rows(cuda_device, off, pad, dtype):
    rng = np.random.default_rng(off)
    rows, vocab = 5, 12345
    c = _case(rng, rows, vocab, 64, 8, 2)
    xb = torch.randn(rows, off + vocab + pad, device="cuda").to(dtype)
    ob = torch.full((rows, 2 * off + vocab + 7), 4.0, device="cuda")
    out = ob[:, 2 * off:2 * off + vocab]
    paged.process_logits(xb[:, off:off + vocab], _rules(c), out=out)
    want, _ = _want(xb[:, off:off + vocab].float().cpu().numpy(), c, np.float32)
    assert np.array_equal(out.cpu().numpy(), want)
    assert (ob[:, :2 * off] == 4).all() and (ob[:, 2 * off + vocab:] == 4).all()


def test_bad_entries_are_skipped_and_reported(cuda_device):
    x = torch.randn(3, 1000, device="cuda")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    f32 = lambda *v: torch.tensor(v, dtype=torch.float32, device="cuda")  # noqa: E731
    cases = [
        (dict(hist_indptr=i32(0, 1, 3, 4), hist_tokens=i32(5, -1, 7, 1000), repetition=f32(2, 2, 2)), {(0, 5), (1, 7)}),
        (dict(hist_indptr=i32(0, 1, 9, 4), hist_tokens=i32(5, 6, 7, 8), repetition=f32(2, 2, 2)), {(0, 5)}),
        (dict(bias_indptr=i32(0, 1, 2, 3), bias_tokens=i32(3, 1 << 30, 4), bias_values=f32(1, 1, 1)), {(0, 3), (2, 4)}),
        (dict(bias_indptr=i32(-1, 1, 2, 3), bias_tokens=i32(3, 2, 4), bias_values=f32(1, 1, 1)), {(1, 2), (2, 4)}),
        (dict(mask=torch.full((2, 32), -1, dtype=torch.int32, device="cuda"), mask_rows=i32(0, 2, -2)), set()),
    ]
    for kw, changed in cases:
        out, _ = paged.process_logits(x, paged.LogitsRules(**kw))
        diff = {tuple(p) for p in torch.nonzero(out != x).tolist()}
        assert diff == changed, kw
        assert paged.device_error(0)[0] == 7
    assert paged.device_error(0) == (0, 0)


def test_rows_that_share_entries_read_only_their_list(cuda_device):
    # rows 0 and 2 of an index pointer that falls share entries 50..99: their values are undefined, but what they
    # add is a bias of the list, and row 3 is as it should be
    n = 100
    indptr = torch.tensor([0, n, n // 2, n, n + 1], dtype=torch.int32, device="cuda")
    tokens = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    store = torch.full((4 * n,), float("nan"), device="cuda")
    store[:n + 1] = 1.0
    x = torch.zeros(4, 1000, device="cuda")
    rules = paged.LogitsRules(bias_indptr=indptr, bias_tokens=tokens, bias_values=store[:n + 1])
    for _ in range(20):
        out, _ = paged.process_logits(x, rules)
        assert paged.device_error(0)[0] == 7
        assert ((out == 0) | (out == 1)).all() and not out[1].any()
        assert out[3].nonzero().tolist() == [[n]]


def test_streams_replay_and_shared_workspace(cuda_device):
    rng = np.random.default_rng(2)
    c = _case(rng, 6, 30000, 100, 10, 3)
    rules = _rules(c)
    x = torch.randn(6, 30000, device="cuda")
    want, wt = paged.process_logits(x, rules, greedy=True)
    torch.cuda.synchronize()
    ws = paged.logits_workspace(6, "cuda")
    s = torch.cuda.Stream()
    for _ in range(3):  # calls that follow one another share a workspace, and it is left zeroed
        got, t = paged.process_logits(x, rules, greedy=True, workspace=ws, stream=s)
    s.synchronize()
    assert torch.equal(got, want) and torch.equal(t, wt) and not ws.any()
    out, tok, xi = torch.empty_like(want), torch.empty_like(wt), x.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        paged.process_logits(xi, rules, out=out, tokens=tok, workspace=ws)
    xi.copy_(x.neg())
    rules._keep["repetition"].fill_(1.25)  # the rules' contents may change between replays
    want, wt = paged.process_logits(xi, rules, greedy=True)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(tok, wt)


def test_a_workspace_made_for_the_call_is_zeroed_on_its_stream(cuda_device):
    x = torch.randn(8, 5000, device="cuda")
    rules = paged.LogitsRules(mask=torch.full((8, 157), -1, dtype=torch.int32, device="cuda"))
    want = paged.argmax_rows(x)
    s = torch.cuda.Stream()
    dirty = [torch.full((512,), 255, dtype=torch.uint8, device="cuda") for _ in range(8)]
    with torch.cuda.stream(s):
        dirty += [torch.full((512,), 255, dtype=torch.uint8, device="cuda") for _ in range(8)]
    torch.cuda.synchronize()
    del dirty
    torch.cuda._sleep(20_000_000)  # the current stream is busy: nothing of the call waits for it
    out, tokens = paged.process_logits(x, rules, greedy=True, stream=s)
    s.synchronize()
    with torch.cuda.stream(s):
        assert torch.equal(tokens, want) and torch.equal(out, x)


def test_wrapper_refuses(cuda_device):
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    f32 = lambda *v: torch.tensor(v, dtype=torch.float32, device="cuda")  # noqa: E731
    x = torch.zeros(2, 100, device="cuda")
    for kw in [dict(hist_tokens=i32(1)), dict(hist_indptr=i32(0, 0, 0)), dict(repetition=f32(1, 1)),
               dict(bias_indptr=i32(0, 0, 0), bias_tokens=i32()), dict(mask_rows=i32(0, 0)),
               dict(bias_indptr=i32(0, 0, 1), bias_tokens=i32(1), bias_values=f32(1, 2)),
               dict(hist_indptr=i32(0, 0, 0).long(), hist_tokens=i32()),
               dict(hist_indptr=i32(0, 0, 0), hist_tokens=i32(), repetition=f32(1, 1, 1)),
               dict(hist_indptr=i32(0, 0, 0).cpu(), hist_tokens=i32().cpu()), dict(mask=i32(1, 2, 3, 4)),
               dict(hist_indptr=i32(0, 0, 0), hist_tokens=i32().cpu())]:
        with pytest.raises(ValueError):
            paged.LogitsRules(**kw)
    rules = paged.LogitsRules(hist_indptr=i32(0, 0, 0), hist_tokens=i32())
    for args, kw in [((x.half(), rules), {}), ((x[:1], rules), {}), ((x[0], rules), {}), ((x.cpu(), rules), {}),
                     ((x, rules), dict(out=torch.zeros(2, 99, device="cuda"))),
                     ((x, rules), dict(out=torch.zeros(2, 100, device="cuda").to(torch.bfloat16))),
                     ((x, rules), dict(tokens=i32(0))), ((x, rules), dict(tokens=i32(0, 0).long())),
                     ((x, paged.LogitsRules(mask=i32(1, 2, 3).view(1, 3), mask_rows=i32(0, 0))), {}),
                     ((x, paged.LogitsRules(mask=torch.zeros(1, 4, dtype=torch.int32, device="cuda"))), {})]:
        with pytest.raises(ValueError):
            paged.process_logits(*args, **kw)
    with pytest.raises(_lib.MittenError):  # overlapping rows
        paged.process_logits(torch.zeros(150, device="cuda").as_strided((2, 100), (50, 1)), rules)
    with pytest.raises(_lib.MittenError):  # too small a workspace
        paged.process_logits(x, rules, greedy=True, workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"))
    # no rows and no rules
    assert paged.process_logits(x[:0], paged.LogitsRules(), greedy=True)[1].numel() == 0
