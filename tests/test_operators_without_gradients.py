"""Operators without derivatives refuse tensors that ask for them: checked before anything touches a device."""

import pytest
import torch as t
from torch.autograd import forward_ad

from aiproj_amd.kernals.draft_tree import append_tree_attention, tree_attention
from aiproj_amd.kernals.norm_rope import norm_rope_append
from tests import norm_rope_cases as cases
from tests.test_draft_tree import _case
from tests.test_norm_rope import Cache


def _calls():
    """(name of the call, what it is given, the call)"""
    c, s = _case(), cases.rows(4, 2, 1, 16, t.float32, t.float32, device="cpu")
    given = dict(q=c.q, ks=t.zeros(3, 2, 64, dtype=t.bfloat16), vs=t.zeros(3, 2, 64, dtype=t.bfloat16))
    rows = dict(qkv=s.qkv, cos=s.cos, sin=s.sin, q_weight=s.q_weight, k_weight=s.k_weight)
    places = t.zeros(4, dtype=t.int64)
    return [("tree_attention", dict(q=c.q), lambda g: tree_attention(g["q"], c.cache, c.ctx, c.tree)),
            ("append_tree_attention", given, lambda g: append_tree_attention(g["q"], g["ks"], g["vs"], c.cache, c.ctx, c.tree)),
            ("norm_rope_append", rows, lambda g: norm_rope_append(g["qkv"], s.positions, g["cos"], g["sin"], 2, 1, g["q_weight"],
                                                                  g["k_weight"], 1e-5, Cache(), places, places))]


CASES = [(i, name) for i, (_, given, _) in enumerate(_calls()) for name in given]


@pytest.mark.parametrize("i,name", CASES)
def test_tensors_that_require_gradients(i, name):
    what, given, call = _calls()[i]
    given[name].requires_grad_(True)
    with pytest.raises(ValueError, match=f"{what}: no gradients"):
        call(given)


@pytest.mark.parametrize("i,name", CASES)
def test_dual_tensors(i, name):
    what, given, call = _calls()[i]
    with forward_ad.dual_level():
        given[name] = forward_ad.make_dual(given[name], t.ones_like(given[name]))
        with t.no_grad(), pytest.raises(ValueError, match=f"{what}: no forward-mode"):
            call(given)


@pytest.mark.parametrize("i", [0, 2])
def test_what_is_asked_of_no_derivative_goes_on(i):
    """On the CPU that is the refusal of its device."""
    what, given, call = _calls()[i]
    with pytest.raises(RuntimeError, match="GPU"):
        call(given)
    for x in given.values():
        x.requires_grad_(True)
    with t.no_grad(), pytest.raises(RuntimeError, match="GPU"):
        call(given)
    with forward_ad.dual_level(), t.no_grad(), pytest.raises(RuntimeError, match="GPU"):
        call(given)
