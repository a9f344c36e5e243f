"""Log probabilities under transforms, modes and traces, which addresses would hide the operation from (on the CPU: such
calls take PyTorch operations)."""

import pytest
import torch as t
from torch.autograd import forward_ad
from torch.utils._python_dispatch import TorchDispatchMode

from aiproj_amd import _native
from aiproj_amd.kernals.token_logprobs import token_logprobs

ROWS, VOCAB = 6, 200


@pytest.fixture(autouse=True)
def any_device(monkeypatch):
    monkeypatch.setattr(_native, "require_gpu", lambda *x, what: x[0].device)


def _inputs(seed=0):
    """Rows without masks, without a target, masked by -inf and by the lowest value, of -inf alone."""
    gen = t.Generator().manual_seed(seed)
    x = 3 * t.randn(ROWS, VOCAB, generator=gen)
    x[2, 50:] = -t.inf
    x[3, 50:] = t.finfo(t.float32).min
    x[4] = -t.inf
    return x, t.tensor([7, -1, 3, 49, 5, VOCAB - 1]), t.randn(ROWS, VOCAB, generator=gen)


def _derivatives(x, tokens):
    """Log probabilities, entropies and their derivatives [T, V] in the logits, in float64."""
    x = x.double()
    logp = t.log_softmax(x, -1)
    empty = (x == -t.inf).all(-1)
    logp[empty] = -t.inf
    p = logp.exp()
    plogp = t.where(p > 0, p * logp, 0.0)
    entropy = -plogp.sum(-1)
    inside = (tokens >= 0) & (tokens < x.shape[1])
    given = logp.gather(1, tokens.clamp(0, x.shape[1] - 1)[:, None])[:, 0]
    hit = (tokens[:, None] == t.arange(x.shape[1])).double()
    d_given = t.where(inside & ~empty, 1.0, 0.0)[:, None] * (hit - p)
    return t.where(inside, given, 0.0), entropy, d_given, -(plogp + p * entropy[:, None])


# float32 sums of V terms, each p, ln p and product with a few roundings; values and derivatives are below 64 here.
TOL = dict(rtol=0, atol=64 * (VOCAB + 20) * 2.0 ** -24)


def _close(got, want):
    t.testing.assert_close(got.double(), want, **TOL)


def test_forward_mode():
    x, tokens, tangent = _inputs()
    given, entropy, d_given, d_entropy = _derivatives(x, tokens)
    with forward_ad.dual_level():
        got = token_logprobs(forward_ad.make_dual(x, tangent), tokens, 3)
        parts = [forward_ad.unpack_dual(y) for y in got]
        _close(parts[0].primal, given)
        _close(parts[1].primal, entropy)
        _close(parts[0].tangent, (d_given * tangent).sum(-1))
        _close(parts[1].tangent, (d_entropy * tangent).sum(-1))
        assert parts[2].tangent is None or bool((parts[2].tangent == 0).all())
        order = t.sort(x, dim=-1, descending=True, stable=True).indices[:, :3]
        assert t.equal(parts[3].primal, order)


def test_func_transforms():
    x, tokens, tangent = _inputs()
    given, entropy, d_given, d_entropy = _derivatives(x, tokens)
    _, tangents = t.func.jvp(lambda y: token_logprobs(y, tokens)[:2], (x,), (tangent,))
    _close(tangents[0], (d_given * tangent).sum(-1))
    _close(tangents[1], (d_entropy * tangent).sum(-1))
    weights = t.randn(2, ROWS, generator=t.Generator().manual_seed(1))
    weights[0, 4] = 0.0          # a log probability of -inf

    def loss(y):
        got = token_logprobs(y, tokens)
        kept = t.where(got.logprobs.isfinite(), got.logprobs, 0.0)
        return (kept * weights[0] + got.entropy * weights[1]).sum()

    want = weights[0][:, None] * d_given + weights[1][:, None] * d_entropy
    _close(t.func.grad(loss)(x), want)
    _close(t.autograd.forward_ad.unpack_dual(t.func.grad(loss)(x)).primal, want)
    # A derivative of the gradient: forward over reverse, against central differences of the float64 gradient.
    _, second = t.func.jvp(t.func.grad(loss), (x,), (tangent,))
    step = 2.0 ** -10
    ends = [_derivatives(x.double() + s * step * tangent.double(), tokens) for s in (1, -1)]
    slope = sum(s * (weights[0][:, None] * e[2] + weights[1][:, None] * e[3]) for s, e in zip((1, -1), ends)) / (2 * step)
    # Differences are off by step^2 / 6 times third derivatives, below 64 times |tangent|^3 of at most 4^3 here.
    t.testing.assert_close(second.double(), slope, rtol=0, atol=TOL["atol"] * 16 + step ** 2 / 6 * 64 * 64)


def test_vmap():
    pairs = [_inputs(seed)[:2] for seed in range(3)]
    x, tokens = (t.stack(y) for y in zip(*pairs))
    got = t.func.vmap(lambda a, b: token_logprobs(a, b, 2))(x, tokens)
    for i in range(3):
        given, entropy, _, _ = _derivatives(x[i], tokens[i])
        _close(got[0][i], given)
        _close(got[1][i], entropy)
        assert t.equal(got[3][i], t.sort(x[i], dim=-1, descending=True, stable=True).indices[:, :2])


def test_traces_and_modes():
    x, tokens, _ = _inputs()
    traced = t.jit.trace(lambda a, b: tuple(token_logprobs(a, b, 2)), (x, tokens),
                         check_trace=False)      # the check calls the function untraced, which needs a GPU
    other, others, _ = _inputs(1)
    given, entropy, _, _ = _derivatives(other, others)
    got = traced(other, others)
    _close(got[0], given)
    _close(got[1], entropy)

    compiled = t.compile(lambda a, b: tuple(token_logprobs(a, b, 2)), backend="eager", fullgraph=True)
    got = compiled(other, others)
    _close(got[0], given)
    _close(got[1], entropy)

    class Seen(TorchDispatchMode):
        count = 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            Seen.count += func is t.ops.aten.exp.default
            return func(*args, **(kwargs or {}))

    with Seen():
        token_logprobs(x, tokens)
    assert Seen.count == 1


@pytest.mark.parametrize("row", [[t.nan, 1.0, 2.0], [t.inf, 1.0, -t.inf]])
def test_nan_and_infinity(row):
    with forward_ad.dual_level():
        x = t.tensor([row])
        got = token_logprobs(forward_ad.make_dual(x, t.ones_like(x)), t.tensor([1]), 1)
        assert bool(got.entropy.isnan().all()) and bool(got.logprobs.isnan().all()) and got.top_tokens.tolist() == [[0]]


def test_refusals_come_first():
    with forward_ad.dual_level():
        x = forward_ad.make_dual(t.zeros(3, 4), t.ones(3, 4))
        with pytest.raises(ValueError):
            token_logprobs(x, t.zeros(2, dtype=t.int64))
        with pytest.raises(ValueError):
            token_logprobs(x, t.zeros(3, dtype=t.int64), 5)
