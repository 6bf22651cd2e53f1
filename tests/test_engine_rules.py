"""The engine's token rules on the host: what set_rules refuses (CPU: a stand-in for the model, nothing launched)."""
from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest

from mitten_b200 import host, model as M

VOCAB = 64


def _engine(**kw):
    sched = host.Scheduler(64, 16, eos_token_ids=(VOCAB,), **kw)
    return M.Engine(SimpleNamespace(s=SimpleNamespace(vocab=VOCAB)), sched, cuda_graphs=False), sched


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
