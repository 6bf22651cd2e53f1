"""The engine's token rules on the host: what set_rules refuses, and whose rules a step applies (CPU: stand-ins for
the model and the kernels, nothing launched)."""
from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from mitten_b200 import _lib, host, model as M

VOCAB = 64


def _engine(pages=64, page_size=16, **kw):
    sched = host.Scheduler(pages, page_size, eos_token_ids=(VOCAB,), **kw)
    model = SimpleNamespace(s=SimpleNamespace(vocab=VOCAB), dev=SimpleNamespace(index=0),
                            forward=lambda b: torch.zeros(b.n_reqs, VOCAB))
    return M.Engine(model, sched, cuda_graphs=False), sched


@pytest.fixture
def applied(monkeypatch):
    """The rules of every step that applied some, as its keyword arguments; every row's token is 1."""
    calls = []

    def rules(**kw):
        calls.append({k: v.tolist() for k, v in kw.items()})

    def pick(logits, *args, **kw):
        return torch.ones(len(logits), dtype=torch.int32)

    monkeypatch.setattr(M.paged, "LogitsRules", rules)
    monkeypatch.setattr(M.paged, "process_logits", lambda logits, *a, **kw: (logits, pick(logits)))
    monkeypatch.setattr(M.paged, "argmax_rows", pick)
    monkeypatch.setattr(M.paged, "device_error", lambda dev: (0, 0))
    return calls


@pytest.mark.parametrize("rules", [
    M.TokenRules(repetition=1e-46), M.TokenRules(repetition=1e39), M.TokenRules(repetition=1e-39),
    M.TokenRules(repetition=-1.0), M.TokenRules(presence=1e39), M.TokenRules(presence=float("nan")),
    M.TokenRules(frequency=-1e39), M.TokenRules(bias={3: 1e39}), M.TokenRules(bias={3: float("inf")}),
    M.TokenRules(bias={3: 1.0, 4: float("nan")}),
])
def test_values_are_held_to_their_f32_form(rules):
    """1e-46 is 0 in f32 and 1e39 infinite: a division by 0, or infinity times 0 occurrences."""
    eng, _ = _engine()
    with pytest.raises(ValueError):
        eng.set_rules(0, [1, 2], rules)
    assert not eng._rules


@pytest.mark.parametrize("rules", [
    M.TokenRules(repetition=1e-38), M.TokenRules(repetition=3e38), M.TokenRules(presence=-3e38, frequency=3e38),
    M.TokenRules(bias={3: 3e38, 4: -float("inf"), 5: -1e39}),
])
def test_values_within_f32_are_taken(rules):
    eng, _ = _engine()
    eng.set_rules(0, np.arange(3), rules)
    assert 0 in eng._rules


def test_rules_end_with_an_exported_request(applied):
    eng, sched = _engine()
    sched.add_request(7, np.arange(5, dtype=np.uint32), max_new_tokens=8)
    eng.set_rules(7, np.arange(5), M.TokenRules(presence=1.0))
    eng.step()
    assert len(applied) == 1
    h = sched.export_request(7)
    assert not eng._rules
    # another request under the same id, as a handoff from elsewhere brings it
    sched.import_request(7, [9, 9, 9], h["outputs"], 3, 0.0, 8)
    eng.step()
    assert len(applied) == 1
    # its own rules, given after the import, do apply
    eng.set_rules(7, [9, 9, 9], M.TokenRules(presence=1.0))
    eng.step()
    assert len(applied) == 2 and applied[1]["hist_tokens"] == [9, 9, 9] + h["outputs"] + [1]


def test_rules_end_with_a_request_that_no_batch_holds(applied):
    """A request that finds no page for its next token is aborted as the batch is made, and is not part of it."""
    eng, sched = _engine(pages=4, page_size=4)
    for rid, n in ((0, 4), (1, 12)):
        sched.add_request(rid, np.arange(n, dtype=np.uint32) + 20 * rid, max_new_tokens=8)
        eng.set_rules(rid, np.arange(n) + 20 * rid, M.TokenRules(presence=1.0))
    while sched.num_active():
        eng.step()
        for rid in (0, 1):
            live = sched.request_info(rid)["state"] not in (_lib.MTN_REQ_DONE, _lib.MTN_REQ_ABORTED)
            assert (rid in eng._rules) == live
    assert _lib.MTN_REQ_ABORTED in [sched.request_info(r)["state"] for r in (0, 1)]


def test_rules_given_before_their_request_is_queued_are_kept(applied):
    eng, sched = _engine()
    eng.set_rules(3, [1, 2], M.TokenRules(presence=1.0))
    sched.add_request(0, np.arange(2, dtype=np.uint32), max_new_tokens=1)
    eng.step()
    sched.add_request(3, np.array([1, 2], np.uint32), max_new_tokens=2)
    eng.run()
    assert len(applied) == 2 and not eng._rules


def test_allowed_is_asked_once_for_every_token(applied):
    """A prompt in chunks of 16: the rows of its unfinished chunks give no token."""
    eng, sched = _engine(max_prefill_tokens_per_iter=16)
    asked = {0: [], 1: [], 2: []}

    def allowed(rid):
        return lambda out: asked[rid].append(list(out))

    def queue(rid, prompt):
        eng.set_rules(rid, prompt, M.TokenRules(allowed=allowed(rid), presence=1.0))

    sched.add_request(0, np.arange(40, dtype=np.uint32), max_new_tokens=6)
    queue(0, np.arange(40))
    eng.step()
    eng.step()
    assert asked[0] == [] and all(a["hist_tokens"] == [] for a in applied)
    eng.step()
    assert asked[0] == [[]] and applied[-1]["hist_tokens"] == list(range(40))
    # a fork's prompt is its parent's and the suffix; its chunks run beside the parent's tokens
    sched.fork(0, 1, np.arange(20, dtype=np.uint32), max_new_tokens=3)
    queue(1, np.concatenate([np.arange(40), np.arange(20)]))
    eng.run()
    assert asked[0] == [[1] * i for i in range(6)] and asked[1] == [[1] * i for i in range(3)]
    # an imported request has its prompt behind it
    sched.import_request(2, np.arange(5), [1, 1], 6, 0.0, 4)
    queue(2, np.arange(5))
    eng.run()
    assert asked[2] == [[1, 1], [1, 1, 1]]


def test_a_step_looks_only_at_its_own_requests(applied, monkeypatch):
    """Rules of queued requests cost a step nothing: their state is not asked for."""
    eng, sched = _engine(max_prefill_tokens_per_iter=4)
    for rid in range(50):
        sched.add_request(rid, np.arange(4, dtype=np.uint32), max_new_tokens=2)
        eng.set_rules(rid, np.arange(4), M.TokenRules(presence=1.0))
    asked = []
    info = sched.request_info
    monkeypatch.setattr(sched, "request_info", lambda r: asked.append(r) or info(r))
    eng.step()
    assert set(asked) == {0}
    eng.run()
    assert not eng._rules and all(len(sched.request_output(r)) == 2 for r in range(50))
