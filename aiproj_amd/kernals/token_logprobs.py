"""Log probabilities of given tokens, with entropy and top alternatives, and their gradient.

`token_logprobs(logits, tokens, top=0) -> TokenLogprobs(logprobs, entropy, top_logprobs, top_tokens)`:

* logits [T, V] (float32, float16 or bfloat16; rows of unit element stride, any row stride),
  tokens [T] int32/int64, both on one GPU; `top` 0 to 64, at most V.
* `logprobs` [T] float32: ln p of each row's token under the row's softmax. A token outside
  [0, V) marks a row without a target: 0, and no gradient.
* `entropy` [T] float32: -sum p ln p in nats.
* `top_logprobs` [T, top] float32 and `top_tokens` [T, top] int64: the most probable tokens in
  falling order, equal logits by rising index. They carry no gradient.
* Logits of -inf have probability 0. A row of -inf alone has log probabilities of -inf, entropy 0
  and gradient 0. A row with NaN or +inf gives NaN (its alternatives count NaN as the largest).

Sums are float32, one launch of the HIP kernel `token_logprobs_kernel` (C ABI
`kvfp8_token_logprobs`), nothing is synchronized with the host and no [T, V] copy is made. Where
gradients are wanted, `logprobs` and `entropy` are differentiable in the logits: one launch of
`token_logprobs_grad_kernel` (`kvfp8_token_logprobs_backward`) reads the logits again and writes the
gradient in their type. Calls that a transform, mode or trace looks at (forward-mode derivatives, vmap,
`torch.func`, `torch.jit.trace`, `torch.compile`), and gradients that one looks at (`is_grads_batched`), take
PyTorch operations in float32, which have derivatives of every kind and order. The kernels' backward is
differentiable once.

The reference has no counterpart: its sampler takes the argmax of the logits.
"""

from __future__ import annotations

from typing import NamedTuple

import torch as t

from aiproj_amd import _native

_DTYPES = (t.float32, t.float16, t.bfloat16)
MAX_TOP = 64


class TokenLogprobs(NamedTuple):
    logprobs: t.Tensor        # [T] float32
    entropy: t.Tensor         # [T] float32
    top_logprobs: t.Tensor    # [T, top] float32
    top_tokens: t.Tensor      # [T, top] int64


def _check(logits: t.Tensor, tokens: t.Tensor, top: int) -> t.device:
    if logits.ndim != 2 or tokens.ndim != 1 or tokens.shape[0] != logits.shape[0]:
        raise ValueError("token_logprobs: logits [T, V] and tokens [T]")
    if logits.dtype not in _DTYPES:
        raise ValueError(f"token_logprobs: unsupported logits dtype {logits.dtype}")
    if tokens.dtype not in (t.int32, t.int64):
        raise ValueError("token_logprobs: tokens must be int32 or int64")
    if logits.shape[1] == 0:
        raise ValueError("token_logprobs: rows without entries")
    if logits.stride(1) != 1 and logits.shape[1] > 1:
        raise ValueError("token_logprobs: rows need unit element stride")
    if isinstance(top, bool) or not isinstance(top, int) or not 0 <= top <= min(MAX_TOP, logits.shape[1]):
        raise ValueError(f"token_logprobs: top must be an int from 0 to {MAX_TOP} and at most V")
    return _native.require_gpu(logits, tokens, what="token_logprobs")


def _forward(logits: t.Tensor, tokens: t.Tensor, top: int, for_backward: bool = False):
    """(logprobs, entropy, top_logprobs, top_tokens, stats [T, 2] for the backward or None)."""
    device = _check(logits, tokens, top)
    rows, vocab = logits.shape
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    logprobs = t.empty(rows, dtype=t.float32, device=device)
    entropy = t.empty_like(logprobs)
    stats = t.empty((rows, 2), dtype=t.float32, device=device) if for_backward else None
    top_logprobs = t.empty((rows, top), dtype=t.float32, device=device)
    top_tokens = t.empty((rows, top), dtype=t.int64, device=device)
    if rows:
        rc = _native.fn("kvfp8_token_logprobs")(
            logits.data_ptr(), _native.dtype_code(logits.dtype), logits.stride(0), rows, vocab,
            tokens.data_ptr(), _native.dtype_code(tokens.dtype), top, logprobs.data_ptr(), entropy.data_ptr(),
            _native.ptr(stats), top_logprobs.data_ptr(), top_tokens.data_ptr(), _native.stream_handle(device))
        _native.check(rc, "kvfp8_token_logprobs")
    return logprobs, entropy, top_logprobs, top_tokens, stats


def _plain_forward(logits, tokens, top):
    """(logprobs, entropy, top_logprobs, top_tokens) as PyTorch operations in float32."""
    x = logits.float()
    m = x.detach().amax(-1, keepdim=True)
    empty = m == -t.inf                                  # every entry is -inf
    d = x - t.where(empty, 0.0, m)
    e = t.exp(d)
    total = t.where(empty, 1.0, e.sum(-1, keepdim=True))
    log_s = t.log(total)
    # Below -200 e^d is 0, and d is kept finite for the product.
    entropy = t.where(empty, 0.0, log_s - (e * d.clamp(min=-200.0)).sum(-1, keepdim=True) / total)[:, 0]
    inside = (tokens >= 0) & (tokens < x.shape[1])
    given = d.gather(1, t.where(inside, tokens, 0).long()[:, None]) - log_s
    logprobs = t.where(inside, t.where(empty, -t.inf, given)[:, 0], 0.0)
    values, order = t.sort(x.detach() + 0.0, dim=-1, descending=True, stable=True)
    top_logprobs = t.where(empty, -t.inf, values[:, :top] - m - log_s.detach())
    return logprobs, entropy, top_logprobs, order[:, :top]


def _plain_backward(logits, tokens, entropy, stats, grad_logprobs, grad_entropy):
    """The gradient as PyTorch operations in float32."""
    vocab = logits.shape[1]
    logp = logits.float() - stats[:, :1] - stats[:, 1:]
    p = t.exp(logp)
    grad = t.zeros_like(p)
    if grad_logprobs is not None:
        inside = (tokens >= 0) & (tokens < vocab)
        hit = (tokens.unsqueeze(1) == t.arange(vocab, device=logits.device)).float()
        grad = grad + t.where(inside, grad_logprobs, 0.0).unsqueeze(1) * (hit - p)
    if grad_entropy is not None:
        grad = grad - grad_entropy.unsqueeze(1) * p * (logp.clamp(min=-200.0) + entropy.unsqueeze(1))
    return t.where(stats[:, 1:] == -t.inf, 0.0, grad).to(logits.dtype)


class TokenLogprobsFunction(t.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top):
        logprobs, entropy, top_logprobs, top_tokens, stats = _forward(logits, tokens, top, True)
        ctx.mark_non_differentiable(top_logprobs, top_tokens)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, tokens, entropy, stats)
        return logprobs, entropy, top_logprobs, top_tokens

    @staticmethod
    @t.autograd.function.once_differentiable
    def backward(ctx, grad_logprobs, grad_entropy, *_):
        logits, tokens, entropy, stats = ctx.saved_tensors
        grads = [g for g in (grad_logprobs, grad_entropy) if g is not None]
        if not grads:
            return None, None, None
        if not _native.is_plain(logits, tokens, entropy, stats, *grads):
            return _plain_backward(logits, tokens, entropy, stats, grad_logprobs, grad_entropy), None, None
        grad = t.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        if grad.numel():
            tokens = tokens.contiguous()
            grad_logprobs, grad_entropy = (None if g is None else g.contiguous() for g in (grad_logprobs, grad_entropy))
            rc = _native.fn("kvfp8_token_logprobs_backward")(
                logits.data_ptr(), _native.dtype_code(logits.dtype), logits.stride(0), logits.shape[0], logits.shape[1],
                tokens.data_ptr(), _native.dtype_code(tokens.dtype), entropy.data_ptr(), stats.data_ptr(),
                _native.ptr(grad_logprobs), _native.ptr(grad_entropy), grad.data_ptr(), _native.stream_handle(logits.device))
            _native.check(rc, "kvfp8_token_logprobs_backward")
        return grad, None, None


def token_logprobs(logits: t.Tensor, tokens: t.Tensor, top: int = 0) -> TokenLogprobs:
    if not _native.is_plain(logits, tokens):
        _check(logits, tokens, top)
        return TokenLogprobs(*_plain_forward(logits, tokens, top))
    if t.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobs(*TokenLogprobsFunction.apply(logits, tokens, top))
    return TokenLogprobs(*_forward(logits, tokens, top)[:4])
