"""Workspaces of drafted trees: what they hold, and that a call stays inside."""

import random

import pytest
import torch as t

from aiproj_amd import _native
from aiproj_amd.kernals import draft_tree
from aiproj_amd.kernals.draft_tree import tree_attention
from tests import draft_tree_cases as cases
from tests.test_gpu_tree_attention import BF16, F16, F32, FP8, _check


def _bytes(*sizes):
    return _native.lib().kvfp8_tree_attention_workspace_bytes(*sizes)


@pytest.mark.parametrize("kv", [_native.E4M3FN, _native.BF16])
def test_size_has_a_limit(kv):
    """Sequences that one workgroup reads leave no states, and of the others' there are at most two for every place: a large batch of
    large trees needs no more than a middle-sized one, less than 64 MB on a device of 256 CUs."""
    large = _bytes(255, 256, 64, 8, 128, 16, kv)
    assert 0 < large == _bytes(32, 256, 64, 8, 128, 16, kv) == _bytes(4000, 8, 64, 8, 128, 16, kv) < 64 * 2 ** 20
    assert _bytes(1, 4, 8, 2, 64, 16, kv) < large


@pytest.mark.gpu
@pytest.mark.parametrize("q_dtype,cache_dtype", [(BF16, FP8), (F32, FP8), (F16, F16)])
@pytest.mark.parametrize("batch", [40, 150])
def test_calls_stay_inside(q_dtype, cache_dtype, batch, monkeypatch):
    """Long sequences, which are cut, among short ones, whose items leave nothing in the workspace. The bytes behind it stay."""
    rng = random.Random(batch)
    held = [rng.randint(0, 100) for _ in range(batch)]
    held[1], held[batch // 2], held[-1] = 6000, 9000, 3000
    c = cases.case(held, [rng.randint(1, 40) for _ in range(batch)], 32, 8, 64, q_dtype, cache_dtype)
    held_back = {}

    def workspace(device, stream, nbytes):
        whole = t.full((nbytes + 2 ** 20,), 0x5A, dtype=t.uint8, device=device)
        held_back["tail"] = whole[nbytes:]
        return whole[:nbytes]

    monkeypatch.setattr(draft_tree, "_workspace", workspace)
    got = tree_attention(c.q, c.cache, c.ctx, c.tree)
    assert bool((held_back["tail"] == 0x5A).all())
    _check(c, got)
