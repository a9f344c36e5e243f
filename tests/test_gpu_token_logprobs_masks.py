"""Log probabilities of rows whose masked entries hold the type's lowest value or another large finite one."""

import pytest
import torch as t

from aiproj_amd.kernals.token_logprobs import token_logprobs
from tests.test_gpu_token_logprobs import DTYPES, HALF, _check_forward, _grad_64, _logits, _slack, _want

pytestmark = pytest.mark.gpu

# Vocabularies of one, several and all waves of a workgroup with entries, and one past what registers hold.
VOCABS = [512, 9000, 32000, 140000]


def _masked(vocab, dtype, value):
    """Rows with a few entries left: the first, the last, some of one wave, every 700th; none left; few masked."""
    logits = _logits(6, vocab, dtype, seed=3)
    masked = t.ones(6, vocab, dtype=t.bool, device="cuda")
    masked[0, :5] = False
    masked[1, -3:] = False
    masked[2, 300:310] = False
    masked[3, ::700] = False
    masked[5] = False
    masked[5, 40:60] = True
    logits[masked] = value
    return logits, t.tensor([2, vocab - 1, 304, 0, 7, 100], device="cuda")


def _values(dtype):
    low = t.finfo(dtype).min
    return [low] if dtype == t.float16 else [low, -1e36]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_masks_of_large_finite_values(dtype, vocab):
    for value in _values(dtype):
        logits, tokens = _masked(vocab, dtype, value)
        for top in (0, 3):
            got = _check_forward(logits, tokens, top)
            assert bool(got.entropy.isfinite().all())


@pytest.mark.parametrize("trains", ["logprobs", "entropy", "both"])
@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_behind_masks_of_large_finite_values(dtype, vocab, trains):
    """Bounds as for the gradients of rows without masks: masked entries have p = 0 and a gradient of 0."""
    gen = t.Generator(device="cuda").manual_seed(5)
    for value in _values(dtype):
        logits, tokens = _masked(vocab, dtype, value)
        logits.requires_grad_(True)
        g, h = (t.randn(6, generator=gen, device="cuda") for _ in range(2))
        got = token_logprobs(logits, tokens)
        if trains == "logprobs":
            h = 0 * h
            grad, = t.autograd.grad(got.logprobs, logits, g)
        elif trains == "entropy":
            g = 0 * g
            grad, = t.autograd.grad(got.entropy, logits, h)
        else:
            grad, = t.autograd.grad((got.logprobs, got.entropy), logits, (g, h))
        want = _grad_64(logits, tokens, g, h)
        logp, _, entropy = _want(logits, tokens)
        p = logp.exp()
        far = t.where(p > 0, logp.abs(), 0.0)
        size = p * (g.abs()[:, None] + h.abs()[:, None] * (far + entropy[:, None]))
        size += g.abs()[:, None] * (t.arange(vocab, device="cuda") == tokens[:, None])
        slack = size * (_slack(logits, logp)[:, None] * 4 + 2.0 ** -22 * (1 + far))
        tiny = t.finfo(dtype).tiny * t.finfo(dtype).eps / 2
        assert bool(((grad.double() - want).abs() <= HALF[dtype] * 1.01 * want.abs() + slack + tiny).all())


@pytest.mark.parametrize("left", [0, 1, 10, 63])
@pytest.mark.parametrize("value", [-1e4, -7.5, -0.3, 0.0, 1.7])
@pytest.mark.parametrize("dtype", DTYPES)
def test_alternatives_of_rows_with_fewer_entries_than_asked_for(dtype, value, left):
    """More entries of one value than the list holds, which follow those above it by index; some of the rest lie below it."""
    for vocab in (2000, 9000, 32000, 140000):
        logits = t.full((3, vocab), value, device="cuda", dtype=dtype)
        gen = t.Generator(device="cuda").manual_seed(left)
        for row, at in enumerate((0, vocab // 2, vocab - left - 7)):
            logits[row, at:at + left] = value + 1 + t.rand(left, generator=gen, device="cuda").to(dtype)
            logits[row, at + left:at + left + 5] = value - 1
        for top in (20, 64):
            _check_forward(logits, t.tensor([0, 1, vocab - 1], device="cuda"), top)
