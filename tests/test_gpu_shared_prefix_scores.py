"""Shared prefixes behind blocks of 256 rows: scores at the borders of the weights' types."""

import math

import pytest
import torch as t

from aiproj_amd.kernals.shared_prefix_attention import shared_prefix_decode_attention
from tests import shared_prefix_cases as cases
from tests.test_gpu_shared_prefix import F16, HALF, LARGE
from tests.test_gpu_shared_prefix_wide import _softmax_64

pytestmark = pytest.mark.gpu


def test_scores_a_step_past_what_the_reference_allows():
    """A reference at which 2^8 more rounds to 2^16 more: the weights of the scores there are past float16's largest number. Tokens 0,
    128, .. of the prefix have a score of 134601552 (base 2), tokens 64, 192, .. the next float32, 16 above it."""
    hq, hkv, d, _, _, page = LARGE[6]
    own, prefix, gen = [1] * 90, 2560, t.Generator(device="cpu").manual_seed(1)
    c = cases.case(own, [prefix], [90], hq, hkv, d, F16, F16, page)
    for slot, n in [(int(c.prefix.slots[0]), prefix), *zip(c.ctx.cache_slots.tolist(), own)]:
        k, v, token = t.zeros(n, hkv, d), t.randn(n, hkv, d, generator=gen).clamp(-3, 3), t.arange(n)
        if n == prefix:
            k[::64, :, 0] = 13016.0
            k[64::128, :, 1] = 1.0
        c.cache.append_kv(c.table[slot].long().cpu()[token // page].cuda(), (token % page).cuda(), k.cuda(), v.cuda())
    c.q = t.zeros_like(c.q)
    c.q[..., 0], c.q[..., 1] = 57344.0, 64.0
    got = shared_prefix_decode_attention(c.q, c.cache, c.ctx, c.prefix)
    want, weight = _softmax_64(c)
    # The scores are 8 apart (base e), their float32 values 11: the lower ones weigh e^-8 or e^-11, of values up to 3 that are not the
    # higher ones'. The others are roundings.
    bound = HALF[F16] * want.abs() + (HALF[F16] + 2.0 ** -12) * weight + 2.0 ** -25 + 2 * 3 * math.exp(-8)
    assert bool(got.isfinite().all()) and bool(((got.double() - want).abs() <= bound).all())
