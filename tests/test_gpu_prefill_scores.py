"""Prompt attention at scores of any size, against float64."""

import math

import pytest
import torch as t

from aiproj_amd.kernals.flash_attention import flash_attention_forward

pytestmark = pytest.mark.gpu

BF16, F16 = t.bfloat16, t.float16
HALF = {x: t.finfo(x).eps / 2 for x in (BF16, F16)}


def _attend(q, k, v):
    """(output, lse) and (softmax(q k^T / sqrt(D)) v, softmax |v|) in float64, one causal sequence."""
    n, hq, d = q.shape
    cu = t.tensor([0, n], dtype=t.int32, device="cuda")
    got = flash_attention_forward(q, k, v, cu, n, 1 / math.sqrt(d))
    kk, vv = (x.double().repeat_interleave(hq // k.shape[1], 1).transpose(0, 1).contiguous() for x in (k, v))
    scores = t.matmul(q.double().transpose(0, 1).contiguous(), kk.transpose(1, 2).contiguous()) / math.sqrt(d)
    p = t.softmax(scores.masked_fill(t.ones(n, n, device="cuda").triu(1).bool(), -math.inf), -1)
    return got, (t.matmul(p, vv).transpose(0, 1), t.matmul(p, vv.abs()).transpose(0, 1))


def _equal_keys(dtype, hq, hkv, d, size, top):
    """Keys 0, 97, .. are one, which lies at `top` along the first dim, far from the others; q is `size` there and 0 elsewhere. Equal
    keys have equal scores in whatever block they fall: all of the weight, in equal parts, 1 each before the division. What is left is
    a half step for each of them in the sums, 64 for the rescalings, the weight's in the product and the output's."""
    n, gen = 700, t.Generator(device="cpu").manual_seed(d)
    k, v = t.randn(n, hkv, d, generator=gen).clamp(-3, 3), t.randn(n, hkv, d, generator=gen)
    best = t.randn(hkv, d, generator=gen).clamp(-3, 3)
    best[:, 0] = top
    k[::97] = best
    q = t.zeros(n, hq, d)
    q[..., 0] = size
    (out, lse), (want, weight) = _attend(*(x.to(dtype).cuda() for x in (q, k, v)))
    assert bool(out.isfinite().all()) and bool(lse.isfinite().all())
    bound = HALF[dtype] * want.abs() + (HALF[dtype] + (64 + 8) * 2.0 ** -24) * weight + (2.0 ** -25 if dtype == F16 else 0.0)
    assert bool(((out.double() - want).abs() <= bound).all()), float(((out.double() - want).abs() - bound).max())


FORMS = [(8, 2, 64), (16, 4, 128), (32, 8, 128), (4, 4, 80), (6, 2, 112)]


@pytest.mark.parametrize("size", [1e4, 1e6, 1e8, 3e9, 1e10, 1e12, 1e30])
@pytest.mark.parametrize("form", FORMS)
def test_equal_keys_share_the_weight_at_any_size(form, size):
    _equal_keys(BF16, *form, size, 8.0)


@pytest.mark.parametrize("size,top", [(1e4, 8.0), (6e4, 8.0), (6e4, 1e3), (6e4, 6e4)])
@pytest.mark.parametrize("form", FORMS)
def test_equal_keys_of_float16(form, size, top):
    """With an outlier channel of 6e4 in queries and keys scores are 4e8."""
    _equal_keys(F16, *form, size, top)


def test_scores_a_step_past_what_the_reference_allows():
    """A reference at which 2^8 more rounds to 2^16 more: the weights of the scores there are past float16's largest number. Keys 0,
    128, .. have a score of 134601552 (base 2), keys 64, 192, .. the next float32, 16 above it."""
    n, d, gen = 250, 64, t.Generator(device="cpu").manual_seed(1)
    k, v, q = t.zeros(n, 2, d), t.randn(n, 2, d, generator=gen).clamp(-3, 3), t.zeros(n, 8, d)
    k[::64, :, 0] = 13016.0
    k[64::128, :, 1] = 1.0
    q[..., 0], q[..., 1] = 57344.0, 64.0
    (out, _), (want, weight) = _attend(*(x.to(F16).cuda() for x in (q, k, v)))
    # The scores are 8 apart (base e), their float32 values 11: the lower ones weigh e^-8 or e^-11, of values up to 3 that are not the
    # higher ones'. The others are roundings.
    bound = HALF[F16] * want.abs() + (HALF[F16] + 2.0 ** -12) * weight + 2.0 ** -25 + 2 * 3 * math.exp(-8)
    assert bool(out.isfinite().all()) and bool(((out.double() - want).abs() <= bound).all())
