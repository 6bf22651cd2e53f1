"""The decode step's operators together: chained, in the model with 4-bit matrices, and in the engine with token rules.

The 4-bit model is held to the numpy oracle on weights that quantise to themselves (a group's largest value is 7
times its scale, so quantising the dequantised weights gives the same codes and scales): what remains is f32
summation order, as for the model with plain weights, and the same bounds apply."""
from __future__ import annotations

import dataclasses

import numpy as np
import pytest
import torch

from mitten_b200 import dense, host, model as M, paged
from oracle import model_ref as R
from tests.test_gpu_logits import _want
from tests.test_gpu_model import LOGIT_TOL_SMALL, shape_of

pytestmark = pytest.mark.gpu


def _quantised(weights, group):
    """Every matrix replaced by its 4-bit values; norms and biases as they are."""
    out = {}
    for k, v in weights.items():
        if v.ndim == 2:
            v = dense.W4Weight.from_float(torch.from_numpy(v).cuda(), group).dequantize().cpu().numpy()
        out[k] = v
    return out


def _engine(cfg, weights, prompts, steps, graphs, **kw):
    model = M.QwenPagedModel(shape_of(cfg), weights, 256, 16, **kw)
    sched = host.Scheduler(256, 16, max_prefill_tokens_per_iter=512, max_decode_batch_size=8,
                           eos_token_ids=(cfg.vocab,))
    for rid, p in enumerate(prompts):
        sched.add_request(rid, p.astype(np.uint32), temperature=0.0, max_new_tokens=steps)
    return M.Engine(model, sched, cuda_graphs=graphs), sched


@pytest.mark.parametrize("kind,group", [("qwen", 64), ("qwen", 128), ("gemma", 32)])
def test_w4_model_matches_the_oracle(cuda_device, kind, group):
    if kind == "qwen":
        cfg = R.QwenShape(hidden=256, layers=3, hq=14, hkv=2, head_dim=64, inter=512, vocab=4096)
    else:
        cfg = dataclasses.replace(R.GEMMA_2B, hidden=512, layers=2, inter=1000, vocab=5001)
    w = _quantised(R.random_weights(cfg, seed=group), group)
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, cfg.vocab, n).astype(np.int64) for n in (40, 17, 130, 5)]
    steps = 12
    want = R.generate(R.RefModel(cfg, w, kv_round=True), prompts, steps)
    for graphs in (False, True):
        eng, sched = _engine(cfg, w, prompts, steps, graphs, w4_group=group)
        eng.run()
        assert [sched.request_output(r) for r in range(len(prompts))] == want
    # the logits themselves, on the first prompt
    eng, sched = _engine(cfg, w, prompts[:1], steps, False, w4_group=group)
    ref = R.RefModel(cfg, w, kv_round=True)
    got = eng.model.forward(sched.schedule()).cpu().numpy()[0]
    assert np.abs(got - ref.forward(0, prompts[0], np.arange(len(prompts[0])))).max() <= LOGIT_TOL_SMALL
    assert paged.device_error(0) == (0, 0)


def test_e4m3_rows_between_norms_and_matrices(cuda_device, monkeypatch):
    """act_e4m3 in an f32 model against the same model with both operators replaced by plain torch.  The two sides'
    values differ by f32 roundings (about 1e-6 relative), so a code of half a step 2^-4 comes out differently for
    about 2e-5 of the 6e4 elements that the norms write here; one such element moves its row by at most 2^-3 of a
    256th of its square, 1 % of its length."""
    cfg = R.QwenShape(hidden=256, layers=2, hq=14, hkv=2, head_dim=64, inter=512, vocab=4096)
    w = R.random_weights(cfg, seed=5)
    rng = np.random.default_rng(6)
    prompts = [rng.integers(0, cfg.vocab, n).astype(np.int64) for n in (30, 9, 6)]

    def logits():
        eng, sched = _engine(cfg, w, prompts, 4, False, w4_group=64, act_e4m3=True)
        out = []
        while sched.num_active():
            b = sched.schedule()
            lg = eng.model.forward(b)
            out.append(lg)
            sched.process_tokens((np.arange(b.n_reqs) * 7 + len(out)).astype(np.uint32))  # the same tokens for both
        return out

    def norm(x, w1, eps, residual=None, out_dtype=None):
        if residual is not None:
            residual += x
            x = residual
        y = x / torch.sqrt(x.square().mean(1, keepdim=True) + eps) * w1
        if out_dtype != torch.float8_e4m3fn:
            return y, None
        scale = (y.abs().amax(1) / 448.0).clamp(min=2.0 ** -100)
        return (y / scale[:, None]).clamp(-448, 448).to(out_dtype), scale

    def matvec(x, weight, x_scales=None, out_dtype=None):
        x = x.float() if x_scales is None else x.float() * x_scales[:, None]
        return (x @ weight.dequantize().T).to(out_dtype)

    got = logits()
    monkeypatch.setattr(M.dense, "add_rms_norm", norm)
    monkeypatch.setattr(M.dense, "w4_matvec", matvec)
    want = logits()
    assert len(got) == len(want) > 2
    for a, b in zip(got, want):
        assert ((a - b).norm() <= 1e-2 * b.norm()), ((a - b).norm() / b.norm())


def test_operators_chained(cuda_device):
    """x + residual -> norm in e4m3 -> 4-bit head -> rules -> greedy token, captured once and replayed on new rows,
    against 64 bits: e4m3 rounds each element by half a step (2^-4, or 2^-10 of the scale near zero), which bounds
    every logit by the sum of those against the weights' magnitudes."""
    g = torch.Generator(device="cuda").manual_seed(3)
    n, hidden, vocab, group = 5, 896, 5003, 64
    r = torch.randn(n, hidden, generator=g, device="cuda").to(torch.bfloat16)
    w1 = 1.0 + 0.1 * torch.randn(hidden, generator=g, device="cuda")
    head = dense.W4Weight.from_float(0.05 * torch.randn(vocab, hidden, generator=g, device="cuda"), group)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    rules = paged.LogitsRules(hist_indptr=i32([0, 2, 2, 5, 6, 6]), hist_tokens=i32([1, 2, 3, 3, 4, 5000]),
                              prompt_lens=i32([1, 0, 1, 0, 0]), repetition=torch.full((n,), 1.5, device="cuda"),
                              mask=torch.full((1, 157), 0x7ffffffe, dtype=torch.int32, device="cuda"),
                              mask_rows=i32([0, -1, 0, 0, -1]))
    x = torch.zeros(n, hidden, dtype=torch.bfloat16, device="cuda")
    total, h, hs = torch.empty_like(r), torch.empty(n, hidden, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(n, device="cuda")
    lg, tok, ws = torch.empty(n, vocab, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda"), paged.logits_workspace(n, "cuda")

    def step():
        dense.add_rms_norm(x, w1, 1e-6, residual=r, sum_out=total, out=h, scales=hs)
        dense.w4_matvec(h, head, x_scales=hs, out=lg)
        paged.process_logits(lg, rules, out=lg, tokens=tok, workspace=ws)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        x.copy_(torch.randn(n, hidden, generator=g, device="cuda"))
        for _ in range(4):
            graph.replay()
        torch.cuda.synchronize()
        s = (x.float() + r.float()).to(torch.bfloat16).double()
        y = s / torch.sqrt(s.square().mean(1, keepdim=True) + 1e-6) * w1.double()
        val = head.dequantize().double()
        raw = y @ val.T
        scale = y.abs().amax(1, keepdim=True) / 448.0
        err = (y.abs() * 2.0 ** -4 + scale * 2.0 ** -10) @ val.abs().T * 1.01 + 1e-4
        want = raw.clone()
        for row, toks in enumerate([[1, 2], [], [3, 3, 4], [5000], []]):
            for t in set(toks):
                want[row, t] = raw[row, t] / 1.5 if raw[row, t] > 0 else raw[row, t] * 1.5
        blocked = torch.zeros(n, vocab, dtype=torch.bool, device="cuda")
        ids = torch.arange(vocab, device="cuda")
        blocked[[0, 2, 3]] = (ids % 32 == 0) | (ids % 32 == 31)
        assert (lg[blocked] == -float("inf")).all()
        assert ((lg.double() - want).abs() <= 1.5 * err)[~blocked].all()
        assert torch.equal(tok, paged.argmax_rows(lg))
        assert torch.equal(total.double(), s)


def test_engine_applies_token_rules(cuda_device):
    """The engine's tokens against a loop that takes the model's logits to the host and applies each request's rules
    there; rows without rules, a prompt in chunks, greedy and hot rows, and a request whose mask leaves nothing."""
    cfg = R.QwenShape(hidden=256, layers=2, hq=14, hkv=2, head_dim=64, inter=512, vocab=4096)
    w = R.random_weights(cfg, seed=11)
    rng = np.random.default_rng(12)
    prompts = [rng.integers(0, cfg.vocab, n).astype(np.int64) for n in (20, 45, 7, 31)]
    odd = np.arange(cfg.vocab) % 2 == 1

    def allowed(out):  # odd tokens, then nothing, then everything
        return odd if len(out) < 4 else np.zeros(cfg.vocab, bool) if len(out) == 4 else None

    rules = {0: M.TokenRules(repetition=1.3, presence=0.4, frequency=0.2),
             1: M.TokenRules(bias={5: 4.0, 9: -float("inf"), int(prompts[1][3]): 2.5}, repetition=0.8),
             3: M.TokenRules(allowed=allowed, frequency=1.0)}

    def fresh():
        model = M.QwenPagedModel(shape_of(cfg), w, 256, 16, w4_group=64)
        sched = host.Scheduler(256, 16, max_prefill_tokens_per_iter=48, max_decode_batch_size=8,
                               eos_token_ids=(cfg.vocab,))
        for rid, p in enumerate(prompts):
            sched.add_request(rid, p.astype(np.uint32), temperature=0.0, max_new_tokens=10)
        return model, sched

    model, sched = fresh()
    while sched.num_active():
        b = sched.schedule()
        lg = model.forward(b).cpu().numpy()
        tok = []
        for i, rid in enumerate(map(int, b.req_ids)):
            row = lg[i:i + 1]
            if rid in rules:
                r, out = rules[rid], sched.request_output(rid)
                allow = r.allowed(out) if r.allowed else None
                c = {"hist": [np.concatenate([prompts[rid], np.array(out, np.int64)]).astype(np.int32)],
                     "prompt": [len(prompts[rid])], "rep": [np.float32(r.repetition)], "pres": [np.float32(r.presence)],
                     "freq": [np.float32(r.frequency)],
                     "bias": [(list(r.bias), np.array(list(r.bias.values()), np.float32))] if r.bias else None,
                     "mask": None if allow is None else allow[None], "mask_rows": [0]}
                row, _ = _want(row, c, np.float32)
            tok.append(int(np.argmax(row[0])) if np.any(row[0] > -np.inf) else 0)
        sched.process_tokens(np.array(tok, np.uint32))
    want = [sched.request_output(r) for r in range(4)]
    assert want[3][4] == 0 and all(t % 2 for t in want[3][:4])
    for graphs in (False, True):
        model, sched = fresh()
        eng = M.Engine(model, sched, cuda_graphs=graphs)
        for rid, r in rules.items():
            eng.set_rules(rid, prompts[rid], r)
        eng.run()
        assert [sched.request_output(r) for r in range(4)] == want
        assert not eng._rules  # forgotten once their requests have ended
    # without rules the requests' tokens are others, so they had an effect
    model, sched = fresh()
    M.Engine(model, sched, cuda_graphs=False).run()
    assert [sched.request_output(r) for r in (0, 1, 3)] != [want[r] for r in (0, 1, 3)]
    assert sched.request_output(2) == want[2]


def test_engine_rules_refusals_and_failures(cuda_device):
    cfg = R.QwenShape(hidden=256, layers=1, hq=14, hkv=2, head_dim=64, inter=512, vocab=1000)
    model = M.QwenPagedModel(shape_of(cfg), R.random_weights(cfg, seed=1), 64, 16)
    sched = host.Scheduler(64, 16, eos_token_ids=(cfg.vocab,))
    eng = M.Engine(model, sched, cuda_graphs=False)
    for bad in (M.TokenRules(repetition=0.0), M.TokenRules(repetition=float("nan")), M.TokenRules(presence=float("inf")),
                M.TokenRules(bias={1000: 1.0}), M.TokenRules(bias={-1: 1.0}), M.TokenRules(bias={1: float("nan")})):
        with pytest.raises(ValueError):
            eng.set_rules(0, [1, 2], bad)
    with pytest.raises(ValueError):
        eng.set_rules(0, [1, 1000], M.TokenRules())
    with pytest.raises(ValueError):
        M.QwenPagedModel(shape_of(cfg), R.random_weights(cfg, seed=1), 64, 16, act_e4m3=True)
    # a mask of the wrong size aborts the batch, and the engine goes on with the next request
    sched.add_request(0, np.arange(5, dtype=np.uint32), max_new_tokens=3)
    eng.set_rules(0, np.arange(5), M.TokenRules(allowed=lambda out: np.ones(999, bool)))
    with pytest.raises(RuntimeError):
        eng.step()
    assert not eng._rules
    sched.add_request(1, np.arange(5, dtype=np.uint32), max_new_tokens=3)
    eng.run()
    assert len(sched.request_output(1)) == 3


def test_temperature_rows_sample_the_processed_logits(cuda_device):
    cfg = R.QwenShape(hidden=256, layers=1, hq=14, hkv=2, head_dim=64, inter=512, vocab=1000)
    model = M.QwenPagedModel(shape_of(cfg), R.random_weights(cfg, seed=1), 64, 16)
    sched = host.Scheduler(64, 16, eos_token_ids=(cfg.vocab,))
    eng = M.Engine(model, sched, cuda_graphs=True)
    only = np.zeros(cfg.vocab, bool)
    only[[17, 400]] = True
    for rid, t in enumerate((0.0, 0.9, 1.4)):
        sched.add_request(rid, np.arange(5 + rid, dtype=np.uint32), temperature=t, max_new_tokens=6)
        eng.set_rules(rid, np.arange(5 + rid), M.TokenRules(allowed=lambda out: only))
    eng.run()
    for rid in range(3):
        out = sched.request_output(rid)
        assert len(out) == 6 and set(out) <= {17, 400}


def _sampled(cfg, model, rules, temperature, steps=4):
    sched = host.Scheduler(64, 16, eos_token_ids=(cfg.vocab,))
    eng = M.Engine(model, sched, cuda_graphs=False)
    sched.add_request(0, np.arange(7, dtype=np.uint32), temperature=temperature, max_new_tokens=steps)
    if rules is not None:
        eng.set_rules(0, np.arange(7), rules)
    eng.run()
    return sched.request_output(0)


def test_sampling_with_rules_keeps_to_them(cuda_device, monkeypatch):
    cfg = R.QwenShape(hidden=256, layers=1, hq=14, hkv=2, head_dim=64, inter=512, vocab=1000)
    model = M.QwenPagedModel(shape_of(cfg), R.random_weights(cfg, seed=1), 64, 16)
    # neutral rules change nothing
    assert _sampled(cfg, model, M.TokenRules(), 0.9) == _sampled(cfg, model, None, 0.9)
    # exp(x / t) overflows f32 with the bias, and vanishes with the mask and the negative one
    assert _sampled(cfg, model, M.TokenRules(bias={33: 100.0}), 0.5) == [33] * 4
    only = np.zeros(cfg.vocab, bool)
    only[[17, 400]] = True
    out = _sampled(cfg, model, M.TokenRules(bias={17: -200.0, 400: -200.0}, allowed=lambda o: only), 0.5)
    assert set(out) <= {17, 400}
    # nothing allowed: the greedy token of such a row
    assert _sampled(cfg, model, M.TokenRules(allowed=lambda o: np.zeros(cfg.vocab, bool)), 0.9) == [0] * 4
    # a random number of 0, or no running sum that reaches it: the sampler's first and last tokens
    for forbidden in (0, cfg.vocab - 1):
        monkeypatch.setattr(M.paged, "sample_rows", lambda x, t, workspace=None, f=forbidden: torch.full(
            (x.shape[0],), f, dtype=torch.int32, device=x.device))
        out = _sampled(cfg, model, M.TokenRules(allowed=lambda o: only), 0.9)
        assert len(out) == 4 and set(out) <= {17, 400}
    with pytest.raises(ValueError):
        M.Engine(model, host.Scheduler(64, 16, eos_token_ids=(cfg.vocab,))).set_rules(
            0, [1], M.TokenRules(bias={1: float("inf")}))


@pytest.mark.parametrize("act_e4m3", [False, True])
def test_head_of_many_rows_keeps_f32_logits(cuda_device, act_e4m3):
    """A bf16 model's head above the row limit of the matrix-vector product.  Scales that are powers of two leave
    the dequantised weights exact in bf16, as bf16 and e4m3 rows are: what is left to round are the f32 sums, each
    of their k additions by at most 2 u of the magnitudes' sum (a tensor core may cut), and one product."""
    cfg = R.QwenShape(hidden=256, layers=1, hq=14, hkv=2, head_dim=64, inter=512, vocab=5003)
    model = M.QwenPagedModel(shape_of(cfg), R.random_weights(cfg, seed=3), 64, 16, dtype=torch.bfloat16, w4_group=64,
                             act_e4m3=act_e4m3)
    g = torch.Generator(device="cuda").manual_seed(5)
    codes = torch.randint(-8, 8, (cfg.vocab, cfg.hidden), generator=g, device="cuda", dtype=torch.int8)
    scales = 2.0 ** torch.randint(-8, -3, (cfg.vocab, 4), generator=g, device="cuda").float()
    model.q4["head"] = dense.W4Weight.from_codes(codes, scales.to(torch.bfloat16), 64)
    for rows in (M.W4_MATVEC_ROWS[torch.bfloat16], M.W4_MATVEC_ROWS[torch.bfloat16] + 1, 200):
        x = torch.randn(rows, cfg.hidden, generator=g, device="cuda")
        xs = x.abs().amax(1) / 448.0 if act_e4m3 else None
        x = (x / xs[:, None]).to(torch.float8_e4m3fn) if act_e4m3 else x.to(torch.bfloat16)
        got = model._linear4("head", x, xs, out_dtype=torch.float32)
        assert got.dtype == torch.float32 and got.is_contiguous()
        xv = x.double() if xs is None else x.double() * xs.double()[:, None]
        val = codes.double() * scales.double().repeat_interleave(64, 1)
        want, mag = xv @ val.T, xv.abs() @ val.abs().T
        u = 2.0 ** -24
        assert ((got.double() - want).abs() <= 2 * cfg.hidden * u * mag + 2 * u * want.abs()).all(), rows


def test_w4_model_without_the_fused_prologue(cuda_device):
    """q, k and v as strided parts of one product, through torch's norms, RoPE and a separate append."""
    cfg = R.QwenShape(hidden=256, layers=3, hq=14, hkv=2, head_dim=64, inter=512, vocab=4096)
    w = _quantised(R.random_weights(cfg, seed=64), 64)
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, cfg.vocab, n).astype(np.int64) for n in (40, 17, 130, 5)]
    want = R.generate(R.RefModel(cfg, w, kv_round=True), prompts, 8)
    for graphs in (False, True):
        eng, sched = _engine(cfg, w, prompts, 8, graphs, w4_group=64, fused_prologue=False)
        eng.run()
        assert [sched.request_output(r) for r in range(len(prompts))] == want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act_e4m3", [False, True])
@pytest.mark.parametrize("lens", [(30, 9, 6), (150, 40, 7)])
def test_w4_model_in_each_type_and_for_many_rows(cuda_device, monkeypatch, dtype, act_e4m3, lens):
    """The model against itself with its norms and its 4-bit products replaced by plain torch in f32, rounded to the
    model's type where the model rounds; 45 rows go through the matrix-vector product, 197 through dequantised
    matrices.  f32: a code of e4m3 comes out differently for about 2e-5 of the elements and then moves its row by 1 %
    of its length at most; two such may meet in a row.  bf16: two layers and the head round about 24 times, each by at
    most 2^-8 of a row's length.  With e4m3 rows a value off by 2^-8 gets another code, 2^-4 off, in one case of 16 at
    most: a quarter of 2^-4 for each of 5 norms."""
    cfg = R.QwenShape(hidden=256, layers=2, hq=14, hkv=2, head_dim=64, inter=512, vocab=4096)
    w = R.random_weights(cfg, seed=5)
    rng = np.random.default_rng(6)
    prompts = [rng.integers(0, cfg.vocab, n).astype(np.int64) for n in lens]

    def logits():
        eng, sched = _engine(cfg, w, prompts, 4, False, w4_group=64, act_e4m3=act_e4m3, dtype=dtype)
        out = []
        while sched.num_active():
            b = sched.schedule()
            out.append(eng.model.forward(b))
            sched.process_tokens((np.arange(b.n_reqs) * 7 + len(out)).astype(np.uint32))  # the same tokens for both
        return out

    def norm(x, w1, eps, residual=None, out_dtype=None):
        if residual is not None:
            residual.copy_(residual.float() + x.float())
            x = residual
        x = x.float()
        y = x / torch.sqrt(x.square().mean(1, keepdim=True) + eps) * w1
        if out_dtype != torch.float8_e4m3fn:
            return y.to(out_dtype), None
        scale = (y.abs().amax(1) / 448.0).clamp(min=2.0 ** -100)
        return (y / scale[:, None]).clamp(-448, 448).to(out_dtype), scale

    def linear(model, name, x, scales=None, out_dtype=None):
        x = x.float() if scales is None else x.float() * scales[:, None]
        return (x @ model.q4[name].dequantize().T).to(out_dtype or model.dt)

    got = logits()
    monkeypatch.setattr(M.dense, "add_rms_norm", norm)
    monkeypatch.setattr(M.QwenPagedModel, "_linear4", linear)
    want = logits()
    tol = 2e-2 if dtype == torch.float32 else 24 * 2.0 ** -8 + (5 * 2.0 ** -6 if act_e4m3 else 0.0)
    assert len(got) == len(want) > 2
    for a, b in zip(got, want):
        assert a.dtype == torch.float32
        assert ((a - b).norm() <= tol * b.norm()), ((a - b).norm() / b.norm())


def test_graphs_of_many_rows_share_the_dequantised_matrices(cuda_device):
    """A decode graph of more rows than the matrix-vector product takes dequantises matrices: graphs of other batch
    sizes must not each keep a copy.  The head is 105 MB in bf16, a graph's own logits are 21 MB."""
    cfg = R.QwenShape(hidden=512, layers=1, hq=14, hkv=2, head_dim=64, inter=512, vocab=102400)
    rng = np.random.default_rng(2)
    head = cfg.vocab * cfg.hidden * 2
    first, n = M.W4_MATVEC_ROWS[torch.bfloat16] + 1, 6
    model = M.QwenPagedModel(shape_of(cfg), R.random_weights(cfg, seed=2), 256, 16, dtype=torch.bfloat16, w4_group=64)
    prompts = [rng.integers(0, cfg.vocab, 5).astype(np.uint32) for _ in range(first + n)]

    def tokens(size):
        sched = host.Scheduler(256, 16, max_prefill_tokens_per_iter=512, max_decode_batch_size=64, eos_token_ids=(cfg.vocab,))
        for r in range(size):
            sched.add_request(r, prompts[r], max_new_tokens=4)
        M.Engine(model, sched).run()
        return [sched.request_output(r) for r in range(size)]

    def held():
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        return torch.cuda.memory_reserved()

    want = tokens(first)
    before = held()
    for i in range(1, n + 1):
        assert tokens(first + i)[:first] == want
    assert held() - before < n * head
    assert tokens(first) == want  # the first graph again, replayed from its first decode step on
