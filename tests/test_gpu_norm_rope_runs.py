"""Normed and rotated heads with rows enough for runs of four heads a group, whose last run is short: forward, cache write, gradients."""

import pytest
import torch as t

from aiproj_amd.kernals.norm_rope import norm_rope, norm_rope_append
from tests import norm_rope_cases as cases
from tests.test_gpu_norm_rope import BF16, F16, F32, FP8, _cache, _case, _check_cache, _check_grads, _check_rows, _leaves

pytestmark = pytest.mark.gpu

# (rows, q heads, KV heads, head size, type, weights, tables): rows x heads x lanes of a row are 2^19 and more, so that 256 CUs are full.
FORMS = [(7000, 6, 2, 64, F16, F32, F32), (3000, 9, 1, 128, BF16, BF16, F32), (1500, 5, 3, 256, BF16, F32, F16),
         (1000, 5, 2, 512, F16, F16, F32), (3000, 7, 2, 80, BF16, F16, F32), (4000, 2, 4, 128, F16, None, F32)]
IDS = ["-".join(str(x).replace("torch.", "") for x in f) for f in FORMS]


def test_forms_take_runs_of_four():
    for n, hq, hkv, d, *_ in FORMS:
        lanes = max(8, 1 << (d // 8 - 1).bit_length())
        assert n * (hq + 2 * hkv) * lanes >= t.cuda.get_device_properties(0).multi_processor_count * 8 * 256 and (hq % 4 or hkv % 4)


@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_forward_against_float64(form):
    s = _case(form)
    _check_rows(s, *norm_rope(*cases.args(s)))


@pytest.mark.parametrize("cache_dtype", [FP8, BF16])
@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_append_against_float64(form, cache_dtype):
    s = _case(form)
    cache, blocks, offsets = _cache(s, cache_dtype)
    packed = norm_rope_append(*cases.args(s), cache, blocks, offsets, packed=True)
    assert all(t.equal(a, b) for a, b in zip(packed, norm_rope(*cases.args(s))))
    _check_cache(s, cache, blocks, offsets)
    again, blocks, offsets = _cache(s, cache_dtype)
    assert t.equal(norm_rope_append(*cases.args(s), again, blocks, offsets), packed[0])
    _check_cache(s, again, blocks, offsets)


@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_gradients_against_float64(form):
    s = _case(form)
    leaves = _leaves(s)
    got = t.autograd.grad(norm_rope(*cases.args(s)), leaves, s.grads)
    _check_grads(s, s.grads, list(got))
    again = t.autograd.grad(norm_rope(*cases.args(s)), leaves, s.grads)
    assert all(t.equal(a, b) for a, b in zip(got, again))
