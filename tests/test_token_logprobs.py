"""Log probabilities, entropy and alternatives: refusals, which need no GPU."""

import pytest
import torch as t

from aiproj_amd import _native
from aiproj_amd.kernals.token_logprobs import token_logprobs


@pytest.mark.parametrize("logits,tokens,top", [
    (t.zeros(3), t.zeros(3, dtype=t.int64), 0),                              # not rows
    (t.zeros(3, 4), t.zeros(2, dtype=t.int64), 0),                           # another count of tokens
    (t.zeros(3, 4), t.zeros(3, 1, dtype=t.int64), 0),
    (t.zeros(3, 4, dtype=t.float64), t.zeros(3, dtype=t.int64), 0),
    (t.zeros(3, 4), t.zeros(3), 0),                                          # tokens that are no indices
    (t.zeros(3, 0), t.zeros(3, dtype=t.int64), 0),
    (t.zeros(4, 3).T, t.zeros(3, dtype=t.int64), 0),                         # columns apart
    (t.zeros(3, 4), t.zeros(3, dtype=t.int64), 5),                           # more than V
    (t.zeros(3, 100), t.zeros(3, dtype=t.int64), 65),
    (t.zeros(3, 100), t.zeros(3, dtype=t.int64), -1),
    (t.zeros(3, 100), t.zeros(3, dtype=t.int64), True),
])
def test_refused_arguments(logits, tokens, top):
    with pytest.raises(ValueError):
        token_logprobs(logits, tokens, top)


def test_host_tensors_are_refused():
    with pytest.raises(RuntimeError):
        token_logprobs(t.zeros(3, 4), t.zeros(3, dtype=t.int64))


def test_argument_codes():
    fn = _native.lib().kvfp8_token_logprobs
    back = _native.lib().kvfp8_token_logprobs_backward
    some = 4096      # an address that a refused call does not look at

    def call(dtype=_native.F32, rows=2, vocab=8, tok=_native.I64, top=0, logits=some, stats=some, tops=some):
        return fn(logits, dtype, vocab, rows, vocab, some, tok, top, some, some, stats, tops, tops, None)

    assert call(dtype=_native.E4M3FN) == -1 and call(tok=_native.F32) == -1
    assert call(rows=-1) == -2 and call(vocab=0) == -2 and call(top=9) == -2 and call(top=-1) == -2
    assert call(vocab=1 << 30) == -6 and call(vocab=100, top=65) == -6
    assert call(logits=None) == -4 and call(top=1, tops=None) == -4
    assert call(logits=some + 2) == -3 and call(dtype=_native.BF16, logits=some + 1) == -3 and call(stats=some + 4) == -3
    assert call(rows=0) == 0
    assert back(some, _native.F32, 8, 2, 8, some, _native.I64, some, some, some, some, None, None) == -4
    assert back(some, _native.F32, 8, 2, 8, some, _native.I64, some, some, some, some, some + 2, None) == -3
    assert back(some, _native.F32, 8, 2, 8, some, _native.F16, some, some, some, some, some, None) == -1
    assert back(some, _native.F32, 8, 0, 8, some, _native.I64, some, some, None, None, some, None) == 0
