"""mtn_process_logits refuses bad arguments before it launches anything (CPU: no pointer is dereferenced)."""
from __future__ import annotations

import ctypes as C

import pytest

from mitten_b200 import _lib

P = [0x100000 * (i + 1) for i in range(8)]


def _call(rules=None, no_rules=False, logits=P[0], dtype=_lib.MTN_DTYPE_F32, stride=100, n=2, vocab=100, out=P[1],
          out_stride=100, tokens=None, ws=None, ws_bytes=0, scratch=P[5], scratch_bytes=1 << 20):
    r = _lib.LogitsRules(**(rules or {}))
    return _lib.lib().mtn_process_logits(logits, dtype, stride, n, vocab, None if no_rules else C.byref(r), out,
                                         out_stride, tokens, ws, ws_bytes, scratch, scratch_bytes, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(n=-1), b"bad sizes"), (dict(vocab=0), b"bad sizes"), (dict(dtype=_lib.MTN_DTYPE_E4M3), b"bad dtype"),
    (dict(logits=None), b"null"), (dict(out=None), b"null"), (dict(no_rules=True), b"null"),
    (dict(logits=P[0] + 2), b"not aligned"), (dict(out=P[1] + 2), b"not aligned"),
    (dict(stride=99), b"strides"), (dict(out_stride=99), b"strides"),
    (dict(out=P[0], dtype=_lib.MTN_DTYPE_BF16), b"in place"), (dict(out=P[0], out_stride=128), b"in place"),
    (dict(rules=dict(n_hist=-1)), b"list sizes"), (dict(rules=dict(hist_indptr=P[2], n_hist=3)), b"hist_tokens"),
    (dict(rules=dict(presence=P[2])), b"without a history"), (dict(rules=dict(prompt_lens=P[2])), b"without a history"),
    (dict(rules=dict(bias_indptr=P[2], bias_tokens=P[3], n_bias=3)), b"bias_values"),
    (dict(rules=dict(mask=P[2], mask_stride=3, n_masks=2)), b"shorter than the vocabulary"),
    (dict(rules=dict(mask=P[2], mask_stride=4, n_masks=1)), b"fewer mask rows"),
    (dict(rules=dict(mask_rows=P[2])), b"without a mask"),
    (dict(tokens=P[3]), b"workspace"), (dict(tokens=P[3], ws=P[4], ws_bytes=31), b"workspace"),
    (dict(tokens=P[3], ws=P[4] + 4, ws_bytes=64), b"aligned"),
    (dict(vocab=2 ** 31 - 1, stride=2 ** 31, out_stride=2 ** 31), b"bad sizes"),
    (dict(n=2 ** 31 - 1, vocab=2 ** 30, stride=2 ** 31, out_stride=2 ** 31), b"batch too large"),
    (dict(rules=dict(hist_indptr=P[2], hist_tokens=P[3], n_hist=10), scratch=None), b"aligned scratch"),
    (dict(rules=dict(hist_indptr=P[2], hist_tokens=P[3], n_hist=10), scratch_bytes=127), b"aligned scratch"),
    (dict(rules=dict(hist_indptr=P[2], hist_tokens=P[3], n_hist=10), scratch=P[5] + 4), b"aligned scratch"),
])
def test_refuses(kw, msg):
    assert _call(**kw) == _lib.MTN_EINVAL
    assert msg in _lib.lib().mtn_last_error(), _lib.lib().mtn_last_error()


def test_nothing_to_do():
    assert _call(n=0) == _lib.MTN_OK
    assert _lib.lib().mtn_process_logits_workspace_bytes(5) == 80


_HIST = dict(hist_indptr=P[2], hist_tokens=P[3], n_hist=10)
_BIAS = dict(bias_indptr=P[2], bias_tokens=P[3], bias_values=P[4], n_bias=10)
_MASK = dict(mask=P[2], mask_stride=4, n_masks=2, mask_rows=P[3])


@pytest.mark.parametrize("rules,field", [
    (_HIST, "hist_indptr"), (_HIST, "hist_tokens"), (dict(_HIST, prompt_lens=P[6]), "prompt_lens"),
    (dict(_HIST, repetition=P[6]), "repetition"), (dict(_HIST, presence=P[6]), "presence"),
    (dict(_HIST, frequency=P[6]), "frequency"), (_BIAS, "bias_indptr"), (_BIAS, "bias_tokens"),
    (_BIAS, "bias_values"), (_MASK, "mask"), (_MASK, "mask_rows"),
])
@pytest.mark.parametrize("off", [1, 2])
def test_refuses_rules_between_elements(rules, field, off):
    assert _call(rules=dict(rules, **{field: rules[field] + off})) == _lib.MTN_EINVAL
    assert b"not aligned" in _lib.lib().mtn_last_error()


def test_refuses_tokens_between_elements():
    assert _call(tokens=P[3] + 2, ws=P[4], ws_bytes=64) == _lib.MTN_EINVAL
    assert b"not aligned" in _lib.lib().mtn_last_error()
