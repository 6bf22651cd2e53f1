"""Cases for the operators of the decode step around attention.

  norm    residual addition + RMSNorm, output bf16 / f32, or e4m3 with one scale per row
  w4      matrix-vector products with 4-bit weights and group scales, for the few rows of a decode step
  logits  penalties for repeated tokens, biases and grammar masks on logits rows, with the greedy token

`run` computes them as elementary torch operations in 32 bits, or, where `own` is set, through the
package's entry points on the same inputs.
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}
BYTES = {"bf16": 2, "f32": 4, "e4m3": 1}
EPS = 1e-6
E4M3_MAX = 448.0
MIN_SCALE = 2.0 ** -100  # a row of zeros keeps a finite, non-zero scale


def listed():
    return [
        # one decoding request of a 0.5B-shaped f32 model: pure launch latency
        {"name": "norm_token", "op": "norm", "rows": 1, "hidden": 896, "x": "f32", "res": "f32", "out": "f32"},
        # 64 decoding requests of a 7B-shaped bf16 model, the row handed on in 8 bits
        {"name": "norm_decode", "op": "norm", "rows": 64, "hidden": 3584, "x": "bf16", "res": "bf16", "out": "e4m3"},
        # a prompt iteration of the same model: bound by memory
        {"name": "norm_prompt", "op": "norm", "rows": 16384, "hidden": 3584, "x": "bf16", "res": "bf16", "out": "e4m3"},
        # k/v projection of one request: the smallest matrix of a 7B-shaped layer
        {"name": "w4_kv_token", "op": "w4", "rows": 1, "n": 512, "k": 3584, "group": 128, "x": "bf16", "out": "bf16"},
        # gate or up projection of one request: the bulk of a decode step's weights
        {"name": "w4_up_token", "op": "w4", "rows": 1, "n": 18944, "k": 3584, "group": 128, "x": "bf16", "out": "bf16"},
        # the same for a batch of 8, fed by the norm's 8-bit rows
        {"name": "w4_up_batch", "op": "w4", "rows": 8, "n": 18944, "k": 3584, "group": 128, "x": "e4m3", "out": "bf16"},
        # down projection for a batch of 8: long rows, few outputs
        {"name": "w4_down_batch", "op": "w4", "rows": 8, "n": 3584, "k": 18944, "group": 128, "x": "bf16", "out": "bf16"},
        # the vocabulary's matrix for a batch of 16: the largest of a step
        {"name": "w4_head_batch", "op": "w4", "rows": 16, "n": 152064, "k": 3584, "group": 64, "x": "bf16", "out": "f32"},
        # odd sizes in f32, a last group that is not full
        {"name": "w4_odd_f32", "op": "w4", "rows": 5, "n": 4873, "k": 1000, "group": 32, "x": "f32", "out": "f32"},
        # one request with penalties only: latency
        {"name": "logits_token", "op": "logits", "rows": 1, "vocab": 151936, "history": 160, "bias": 0, "mask": False,
         "x": "f32"},
        # a serving batch with everything on
        {"name": "logits_batch", "op": "logits", "rows": 64, "vocab": 152064, "history": 4096, "bias": 64, "mask": True,
         "x": "f32"},
        # the largest vocabulary, long histories, bf16 logits
        {"name": "logits_wide", "op": "logits", "rows": 128, "vocab": 256000, "history": 16384, "bias": 16,
         "mask": True, "x": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "w4", "logits"])
    if op == "norm":
        hidden = _log(rng, 64, 8192)
        if rng.random() < 0.5:
            hidden = max(64, hidden // 64 * 64)
        # no more bytes than norm_prompt has, at up to 16 bytes an element
        rows = _log(rng, 1, min(16384, 16384 * 3584 * 7 // (16 * hidden)))
        return {"op": "norm", "rows": rows, "hidden": hidden, "x": rng.choice(["bf16", "f32"]),
                "res": rng.choice(["bf16", "f32", "none"]), "out": rng.choice(["bf16", "f32", "e4m3"])}
    if op == "w4":
        k = _log(rng, 64, 18944)
        if rng.random() < 0.7:
            k = max(64, k // 128 * 128)
        n = _log(rng, 64, 152064)
        n = min(n, 152064 * 3584 // (4 * k))
        return {"op": "w4", "rows": rng.choice([1, 2, 3, 4, 5, 7, 8, 11, 13, 16, 17, 24, 29, 32]), "n": n, "k": k,
                "group": rng.choice([32, 64, 128]), "x": rng.choice(["bf16", "f32", "e4m3"]),
                "out": rng.choice(["bf16", "f32"])}
    vocab = _log(rng, 1000, 256000)
    # no more bytes than logits_wide has, at up to 8 bytes an element
    rows = _log(rng, 1, min(128, 128 * 256000 * 5 // (8 * vocab)))
    history = 0 if rng.random() < 0.25 else _log(rng, 16, 16384)
    return {"op": "logits", "rows": rows, "vocab": vocab, "history": history, "bias": rng.choice([0, _log(rng, 1, 300)]),
            "mask": history == 0 or rng.random() < 0.6, "x": rng.choice(["bf16", "f32"])}


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def _prepare_norm(c, g):
    rows, hidden = c["rows"], c["hidden"]
    # a few channels carry values far above the others, as residual streams of trained models do
    chan = torch.where(_rand(g, hidden) < 0.01, 20.0, 1.0)
    st = {"x": (_randn(g, rows, hidden) * 0.5).to(DT[c["x"]]), "w1": 1.0 + 0.2 * _randn(g, hidden), "res": None,
          "sum": None}
    if c["res"] != "none":
        st["res"] = (_randn(g, rows, hidden) * chan).to(DT[c["res"]])
        st["sum"] = torch.empty_like(st["res"])
    st["out"] = torch.empty(rows, hidden, dtype=DT[c["out"]], device="cuda")
    st["scales"] = torch.empty(rows, device="cuda") if c["out"] == "e4m3" else None
    return st


def _prepare_w4(c, g):
    rows, n, k, group = c["rows"], c["n"], c["k"], c["group"]
    codes = torch.empty(n, k, dtype=torch.int8, device="cuda")
    codes.copy_((_randn(g, n, k) * 2.5).round_().clamp_(-8, 7))
    scales = (0.008 * (0.5 + _rand(g, n, -(-k // group)))).to(torch.bfloat16)
    x = _randn(g, rows, k) * torch.where(_rand(g, k) < 0.01, 8.0, 1.0)
    st = {"codes": codes, "scales": scales, "group": group, "xs": None,
          "out": torch.empty(rows, n, dtype=DT[c["out"]], device="cuda")}
    if c["x"] == "e4m3":
        st["xs"] = x.abs().amax(1) / E4M3_MAX
        st["x"] = (x / st["xs"][:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    else:
        st["x"] = x.to(DT[c["x"]])
    if own:
        from mitten_b200 import dense

        # the layout a serving program keeps its weights in
        st["weight"] = dense.W4Weight.from_codes(codes, scales, group)
    return st


def _ragged(g, rows, most):
    """Row lengths between 0 and `most` (the last one `most`) as an index pointer, and row r's number for each entry."""
    lens = (_rand(g, rows) * (most + 1)).long().clamp_(max=most)
    lens[-1] = most
    ptr = torch.zeros(rows + 1, dtype=torch.int32, device="cuda")
    ptr[1:] = lens.cumsum(0)
    return ptr, lens, torch.repeat_interleave(torch.arange(rows, device="cuda"), lens)


def _prepare_logits(c, g):
    rows, vocab = c["rows"], c["vocab"]
    st = {"logits": (_randn(g, rows, vocab) * 3.0).to(DT[c["x"]]), "hist": None, "bias": None, "mask": None,
          "out": torch.empty(rows, vocab, device="cuda"),
          "tokens": torch.empty(rows, dtype=torch.int32, device="cuda")}
    if c["history"]:
        # texts repeat their frequent tokens; a part of each history is the prompt
        ptr, lens, row = _ragged(g, rows, c["history"])
        st["hist"] = {"ptr": ptr, "row": row, "tokens": (_rand(g, row.numel()).pow(3) * vocab).int().clamp_(max=vocab - 1),
                      "prompt": (lens * _rand(g, rows)).int(), "rep": 1.0 + 0.5 * _rand(g, rows),
                      "presence": 0.6 * _rand(g, rows), "frequency": 0.4 * _rand(g, rows)}
    if c["bias"]:
        ptr, _, row = _ragged(g, rows, c["bias"])
        st["bias"] = {"ptr": ptr, "row": row, "tokens": (_rand(g, row.numel()) * vocab).int().clamp_(max=vocab - 1),
                      "values": 4.0 * _randn(g, row.numel())}
    if c["mask"]:
        # one bit per token; grammar states allow from nothing through a handful to nearly everything, and
        # requests share them; some requests have none
        states = max(2, rows // 2)
        words = -(-vocab // 32)
        share = _rand(g, states, 1).pow(2)
        bits = torch.empty(states, words, 32, dtype=torch.bool, device="cuda")
        bits.copy_((_rand(g, states, words * 32) < share).view(states, words, 32))
        bits[0] = False
        val = (bits.long() << torch.arange(32, device="cuda")).sum(2)
        st["mask"] = {"bits": torch.where(val >= 2 ** 31, val - 2 ** 32, val).int(),
                      "rows": (_rand(g, rows) * (states + 1)).int().clamp_(max=states) - 1}
    if own:
        from mitten_b200 import paged

        h, b, m = st["hist"], st["bias"], st["mask"]
        st["rules"] = paged.LogitsRules(
            **({} if h is None else {"hist_indptr": h["ptr"], "hist_tokens": h["tokens"], "prompt_lens": h["prompt"],
                                     "repetition": h["rep"], "presence": h["presence"], "frequency": h["frequency"]}),
            **({} if b is None else {"bias_indptr": b["ptr"], "bias_tokens": b["tokens"], "bias_values": b["values"]}),
            **({} if m is None else {"mask": m["bits"], "mask_rows": m["rows"]}))
        st["workspace"] = paged.logits_workspace(rows, "cuda")
    return st


def prepare(case, seed):
    g = _gen(seed)
    st = {"norm": _prepare_norm, "w4": _prepare_w4, "logits": _prepare_logits}[case["op"]](case, g)
    st["case"] = case
    return st


# ------------------------------------------------------------------ the plain forms

def _plain_norm(st):
    s = st["x"].float()
    total = None
    if st["res"] is not None:
        total = (s + st["res"].float()).to(st["res"].dtype)  # the norm reads the sum as it is stored
        s = total.float()
    y = s / torch.sqrt((s * s).mean(1, keepdim=True) + EPS) * st["w1"]
    if st["scales"] is None:
        return {"sum": total, "y": y.to(st["out"].dtype)}
    scale = (y.abs().amax(1) / E4M3_MAX).clamp(min=MIN_SCALE)
    return {"sum": total, "y": (y / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), "scales": scale}


def _plain_w4(st):
    k = st["codes"].shape[1]
    w = st["codes"].float() * st["scales"].float().repeat_interleave(st["group"], 1)[:, :k]
    x = st["x"].float()
    if st["xs"] is not None:
        x = x * st["xs"][:, None]
    return {"y": (x @ w.T).to(st["out"].dtype)}


def _plain_logits(st):
    x = st["logits"].float()
    rows, vocab = x.shape
    h, b, m = st["hist"], st["bias"], st["mask"]
    if h is not None:
        flat = h["row"] * vocab + h["tokens"]
        at = torch.arange(flat.numel(), device=x.device) - h["ptr"][:-1].long()[h["row"]]
        seen = torch.zeros(rows * vocab, dtype=torch.int32, device=x.device).index_fill_(0, flat, 1).view(rows, vocab) > 0
        made = torch.zeros(rows * vocab, dtype=torch.int32, device=x.device).index_add_(
            0, flat, (at >= h["prompt"].long()[h["row"]]).int()).view(rows, vocab)
        rep = h["rep"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
        x = x - h["frequency"][:, None] * made.float()
        x = x - torch.where(made > 0, h["presence"][:, None], 0.0)
    if b is not None:
        # a token listed twice: its last entry counts
        flat = b["row"] * vocab + b["tokens"]
        last = torch.zeros(rows * vocab, dtype=torch.int32, device=x.device).scatter_reduce_(
            0, flat, torch.arange(1, flat.numel() + 1, dtype=torch.int32, device=x.device), "amax").view(rows, vocab).long()
        x = x + torch.cat([torch.zeros(1, device=x.device), b["values"]])[last]
    if m is not None:
        v = torch.arange(vocab, device=x.device)
        bits = (m["bits"][m["rows"].long().clamp(min=0)][:, v >> 5] >> (v & 31)) & 1
        x = torch.where((bits == 0) & (m["rows"] >= 0)[:, None], -math.inf, x)
    # the first strict maximum; a row of nothing but -inf gives 0
    top = x.amax(1, keepdim=True)
    first = torch.where(x == top, torch.arange(vocab, device=x.device), vocab).amin(1)
    return {"logits": x, "tokens": first.int()}


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"norm": _plain_norm, "w4": _plain_w4, "logits": _plain_logits}[op](state)
    if op == "logits":
        from mitten_b200 import paged

        out, tokens = paged.process_logits(state["logits"], state["rules"], out=state["out"], tokens=state["tokens"],
                                           workspace=state["workspace"])
        return {"logits": out, "tokens": tokens}
    from mitten_b200 import dense

    if op == "norm":
        y, scales = dense.add_rms_norm(state["x"], state["w1"], EPS, residual=state["res"], sum_out=state["sum"],
                                       out=state["out"], scales=state["scales"])
        if scales is None:
            return {"sum": state["sum"], "y": y}
        return {"sum": state["sum"], "y": y, "scales": scales}
    return {"y": dense.w4_matvec(state["x"], state["weight"], x_scales=state["xs"], out=state["out"])}


# ------------------------------------------------------------------ in 64 bits, from the definitions

def _exact_norm(st):
    v = st["x"].double()
    total = None
    if st["res"] is not None:
        total = v + st["res"].double()
        v = total.to(st["res"].dtype).double()
    rms = (v.square().sum(1) / v.shape[1] + EPS).sqrt()
    y = v / rms[:, None] * st["w1"].double()[None, :]
    if st["scales"] is None:
        return {"sum": total, "y": y}
    scale = torch.maximum(y.abs().max(1).values / E4M3_MAX, torch.tensor(MIN_SCALE, dtype=torch.float64, device=y.device))
    return {"sum": total, "y": y / scale[:, None], "scales": scale}


def _exact_w4(st):
    x = st["x"].to(torch.float64)
    if st["xs"] is not None:
        x = x * st["xs"].double()[:, None]
    codes, scales, group = st["codes"], st["scales"].double(), st["group"]
    y = torch.zeros(x.shape[0], codes.shape[0], dtype=torch.float64, device=x.device)
    for j in range(scales.shape[1]):
        part = slice(j * group, min((j + 1) * group, codes.shape[1]))
        y += (x[:, part] @ codes[:, part].double().T) * scales[:, j]
    return {"y": y}


def _exact_logits(st):
    x = st["logits"].double()
    vocab = x.shape[1]
    h, b, m = st["hist"], st["bias"], st["mask"]
    ptr = None if h is None else h["ptr"].tolist()
    bptr = None if b is None else b["ptr"].tolist()
    allowed = None if m is None else m["rows"].tolist()
    for r in range(x.shape[0]):
        row = x[r]
        if h is not None:
            mine = h["tokens"][ptr[r]:ptr[r + 1]].long()
            made = torch.bincount(mine[int(h["prompt"][r]):], minlength=vocab).double()
            seen = torch.bincount(mine, minlength=vocab) > 0
            rep = h["rep"][r].double()
            row = torch.where(seen & (row > 0), row / rep, torch.where(seen, row * rep, row))
            row = row - h["frequency"][r].double() * made - h["presence"][r].double() * (made > 0)
        if b is not None:
            add = dict(zip(b["tokens"][bptr[r]:bptr[r + 1]].tolist(), b["values"][bptr[r]:bptr[r + 1]].tolist()))
            if add:
                at = torch.tensor(list(add), device=x.device)
                row = row.index_add(0, at, torch.tensor(list(add.values()), dtype=torch.float64, device=x.device))
        if m is not None and allowed[r] >= 0:
            bits = (m["bits"][allowed[r]][:, None] >> torch.arange(32, device=x.device)) & 1
            row = row.masked_fill(bits.reshape(-1)[:vocab] == 0, -math.inf)
        x[r] = row
    return {"logits": x, "tokens": None}


def exact(case, seed):
    st = prepare(case, seed)
    return {"norm": _exact_norm, "w4": _exact_w4, "logits": _exact_logits}[case["op"]](st)


def work(case):
    if case["op"] == "norm":
        n = case["rows"] * case["hidden"]
        per = BYTES[case["x"]] + BYTES[case["out"]] + (0 if case["res"] == "none" else 2 * BYTES[case["res"]])
        return {"bytes": n * per + 4 * case["hidden"] + (4 * case["rows"] if case["out"] == "e4m3" else 0), "flops": 6 * n}
    if case["op"] == "w4":
        m, n, k = case["rows"], case["n"], case["k"]
        weights = n * k // 2 + 2 * n * -(-k // case["group"])
        rows = m * k * BYTES[case["x"]] + m * n * BYTES[case["out"]] + (4 * m if case["x"] == "e4m3" else 0)
        return {"bytes": weights + rows, "flops": 2 * m * n * k}
    m, v = case["rows"], case["vocab"]
    n = m * v * (BYTES[case["x"]] + 4) + 4 * m
    n += 4 * m * case["history"] // 2 + 8 * m * case["bias"] // 2 + (max(2, m // 2) * -(-v // 32) * 4 if case["mask"] else 0)
    return {"bytes": n, "flops": 4 * m * v}
