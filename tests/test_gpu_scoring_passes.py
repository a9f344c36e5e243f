"""Scores of more continuations than one pass holds."""

import pytest
import torch as t

from aiproj_amd.inference import scoring
from tests.test_gpu_shared_prefix_model import ATOL, RTOL, SMALL, _tokens, _whole_logits, model  # noqa: F401

pytestmark = pytest.mark.gpu


class Watched:
    """A model that keeps the number of tokens of its calls."""

    def __init__(self, model):
        self.model, self.cfg, self.embed, self.rows = model, model.cfg, model.embed, []

    def __call__(self, tokens, meta, caches):
        self.rows.append(tokens.shape[0])
        return self.model(tokens, meta, caches)


@pytest.mark.parametrize("cache_dtype", [t.bfloat16, t.float8_e4m3fn])
def test_passes_score_like_one(model, cache_dtype, monkeypatch):  # noqa: F811
    """The same continuations in one pass and in several; a bf16 cache also against whole sequences."""
    lengths = [5, 1, 17, 2, 40, 33, 1, 1, 9]
    prompt, continuations = _tokens(50, seed=6), [_tokens(n, seed=7 + i) for i, n in enumerate(lengths)]
    one = scoring.score_continuations(model, prompt, continuations, top=3, cache_dtype=cache_dtype)
    monkeypatch.setattr(scoring, "_PASS_TOKENS", 24)
    watched = Watched(model)
    got = scoring.score_continuations(watched, prompt, continuations, top=3, cache_dtype=cache_dtype)
    assert watched.rows == [50, 23, 2, 40, 33, 11]
    whole = _whole_logits(model, [t.cat([prompt, c]) for c in continuations])
    for g, o, c, logits in zip(got, one, continuations, whole):
        rows = logits[len(prompt) - 1:-1].double()
        slack = 2 * (ATOL + RTOL * rows.abs().amax(-1))
        # Logits of one model through products of other shapes, in both.
        assert bool(((g.logprobs - o.logprobs).abs() <= 2 * slack).all()) and g.top_tokens.shape == (len(c), 3)
        if cache_dtype == t.bfloat16:
            want = t.log_softmax(rows, -1).gather(1, c[:, None])[:, 0]
            assert bool(((g.logprobs.double() - want).abs() <= slack).all())


def test_a_pass_is_bounded(model):  # noqa: F811
    prompt, continuations = _tokens(20, seed=1), [_tokens(60, seed=2)] * 600
    watched = Watched(model)
    got = scoring.score_continuations(watched, prompt, continuations)
    assert len(watched.rows) == 4 and max(watched.rows) <= 1 << 14
    assert len(got) == 600 and all(g.logprobs.shape == (60,) for g in got)
    # Equal continuations: the same products in the first two passes, which have the same shape.
    assert t.equal(got[0].logprobs, got[273].logprobs)
