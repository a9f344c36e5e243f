"""The prompt form whose prefix kernel joins out and lse itself, and whose last row blocks are split, at every head size and
cache type that blocks of 256 rows take."""

import pytest
import torch as t

from aiproj_amd import _native
from tests import shared_prefix_cases as cases
from tests import test_gpu_shared_prefix as base
from tests.test_gpu_shared_prefix import BF16, F16, FP8

pytestmark = pytest.mark.gpu

# (q heads, KV heads, head size, q type, cache type, page): two q heads a KV head, so that pairs and rows differ.
FORMS = [(64, 32, 64, F16, FP8, 16), (64, 32, 80, BF16, FP8, 16), (64, 32, 96, F16, FP8, 64), (64, 32, 112, BF16, FP8, 16),
         (64, 32, 128, BF16, FP8, 32), (64, 32, 128, F16, FP8, 16), (64, 32, 64, BF16, BF16, 16), (64, 32, 128, F16, F16, 16),
         (64, 32, 128, BF16, BF16, 128)]
# (own lengths, prefixes, group sizes, sequences before the first group). Row blocks are counted as (pairs + 255 groups) /
# 256, for each of the 32 KV heads. No splits from 172 of 256 CUs' worth of them on, and those past 256 (32 an XCD at once)
# are split: 6 to 8 blocks are joined in place, 9 and more have an end.
PROMPTS = {
    "in place, one": ([300, 1, 250, 349], [2300], [4], 0),                                  # 1800 pairs: 8 blocks
    "in place, uneven": ([100, 150, 7, 120, 0, 60], [2300, 0, 20, 300], [2, 1, 1, 1], 1),   # 874 pairs: 7 blocks
    "end, one": ([300, 1, 250, 549], [2300], [4], 0),                                       # 2200 pairs: 9 blocks
    "end, uneven": ([100, 300, 7, 300, 0, 290], [2300, 0, 20, 300], [2, 1, 1, 1], 1),       # 1994 pairs: 11 blocks
    "end, many": ([70 - (i % 3) for i in range(8)], [290 * (i + 1) + i for i in range(8)], [1] * 8, 0),     # 1106: 12 blocks
}


def _join(c, out, lse, workspace, nbytes, longest):
    """kvfp8_shared_prefix_prefill on these, its return code."""
    k, p, code = c.cache, c.prefix, _native.TORCH_TO_CODE
    scales = [x.data_ptr() if x is not None else None for x in (getattr(k, "k_scales", None), getattr(k, "v_scales", None))]
    return _native.lib().kvfp8_shared_prefix_prefill(
        c.q.data_ptr(), code[c.q.dtype], len(c.q), c.hq, c.hkv, c.d, k.k.data_ptr(), k.v.data_ptr(), code[k.k.dtype], *scales,
        k.k.shape[0], c.page, c.table.data_ptr(), *c.table.shape, p.slots.data_ptr(), code[p.slots.dtype], p.lengths.data_ptr(),
        code[p.lengths.dtype], p.starts.data_ptr(), code[p.starts.dtype], len(p.slots), c.cu.data_ptr(), code[c.cu.dtype],
        len(c.cu) - 1, longest, c.scale, out.data_ptr(), lse.data_ptr(), workspace.data_ptr(), nbytes,
        t.cuda.current_stream().cuda_stream)


def _bytes(states, d):
    """Maxima, sums and weighted values of so many states, each from a multiple of 256 bytes on."""
    return 2 * (-(-4 * states // 256) * 256) + -(-4 * states * d // 256) * 256


def _least(call, most):
    """The least number of bytes with which a call is not refused for its workspace."""
    low, high = 0, most
    while low < high:
        middle = (low + high) // 2
        code = call(middle)
        assert code in (0, -5)
        low, high = (low, middle) if code == 0 else (middle + 1, high)
    return low


@pytest.mark.parametrize("name", PROMPTS)
@pytest.mark.parametrize("form", FORMS, ids=lambda f: "-".join(str(x).replace("torch.", "") for x in f))
def test_prompts_joined_by_the_prefix_kernel(form, name, monkeypatch):
    monkeypatch.setitem(base.PROMPTS, name, PROMPTS[name])
    c = base._prompt(form, name, t.int64 if "uneven" in name else t.int32)
    out, lse = base._run_prompt(c)
    base._check_prompt(c, out, lse)
    again, lse_again = base._run_prompt(c)
    assert t.equal(out, again) and t.equal(lse, lse_again)

    # Which kernels these were: the least workspace that is accepted. Splits leave a state each for every row and q head,
    # a split end for 8 XCDs' blocks of 256 pairs; joined in place there is none.
    longest, pairs = 90, len(c.q) * c.hq
    workspace = t.empty(_bytes(64 * pairs, c.d), dtype=t.uint8, device="cuda")
    needs = _least(lambda nbytes: _join(c, out, lse, workspace, nbytes, longest), workspace.numel())
    if "in place" in name:
        assert needs == 0
    else:
        assert needs in [_bytes(2048 * n, c.d) for n in range(1, 300)] and needs not in [_bytes(n * pairs, c.d) for n in range(1, 65)]

    out, lse = t.full_like(c.q, 7.0), t.full_like(lse, 7.0)
    assert _join(c, out, lse, workspace, needs, longest) == 0

    # Rows past the longest, of no group and of prefixes without tokens are left alone, the others are joined once.
    inside = t.zeros(len(c.q), dtype=t.bool)
    for b, (s0, s1) in enumerate(zip(c.bounds, c.bounds[1:])):
        g = cases.group_of(c, b)
        if g is not None and c.prefixes[g]:
            inside[s0:min(s1, s0 + longest)] = True
    inside = inside.to("cuda")
    assert bool((out[~inside] == 7.0).all()) and bool((lse[~inside] == 7.0).all()) and bool((lse[inside] != 7.0).all())
    out, lse = base._run_prompt(c, longest)
    for b, (s0, s1) in enumerate(zip(c.bounds, c.bounds[1:])):
        inside[s0:min(s1, s0 + longest)] = True
    base._check_prompt(c, out, lse, inside)
