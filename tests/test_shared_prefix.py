"""Shared-prefix attention: refusals, which need no GPU."""

from types import SimpleNamespace

import pytest
import torch as t

from aiproj_amd import _native
from aiproj_amd.kernals.shared_prefix_attention import (SharedPrefix, shared_prefix_decode_attention,
                                                        shared_prefix_prefill_attention)


def _args(**change):
    a = dict(q=t.zeros(3, 4, 64), cache=SimpleNamespace(k=t.zeros(2, 16, 2, 64), v=t.zeros(2, 16, 2, 64), quantized=False, block_size=16),
             table=t.zeros(4, 2, dtype=t.int32), slots=t.zeros(3, dtype=t.int64), lens=t.zeros(3, dtype=t.int32),
             prefix=SharedPrefix.one(3, 5, 3, "cpu"))
    a.update(change)
    return a


def _decode(**change):
    a = _args(**change)
    ctx = SimpleNamespace(cache_slots=a["slots"], context_lengths=a["lens"], block_table=a["table"])
    return shared_prefix_decode_attention(a["q"], a["cache"], ctx, a["prefix"])


def _prefill(k=t.zeros(3, 2, 64), cu=t.tensor([0, 3]), **change):
    a = _args(**change)
    return shared_prefix_prefill_attention(a["q"], k, k, cu, 3, 0.125, a["cache"], a["table"], a["prefix"])


def _cache(**change):
    c = dict(k=t.zeros(2, 16, 2, 64), v=t.zeros(2, 16, 2, 64), quantized=False, block_size=16)
    c.update(change)
    return SimpleNamespace(**c)


def _quantized(scales):
    k = t.zeros(2, 16, 2, 64, dtype=t.uint8).view(t.float8_e4m3fn)
    return _cache(k=k, v=k, quantized=True, k_scales=scales, v_scales=scales)


SHARED = [
    dict(q=t.zeros(3, 256)),
    dict(q=t.zeros(3, 3, 64)),                                                   # 3 q heads over 2 KV heads
    dict(cache=_cache(k=t.zeros(2, 16, 2, 32), v=t.zeros(2, 16, 2, 32))),        # another head size
    dict(cache=_cache(v=t.zeros(3, 16, 2, 64))),
    dict(cache=_cache(v=t.zeros(2, 16, 2, 64, dtype=t.float16))),
    dict(cache=_cache(k=t.zeros(2, 16, 2, 64, dtype=t.float64), v=t.zeros(2, 16, 2, 64, dtype=t.float64))),
    dict(cache=_cache(k=t.zeros(2, 2, 16, 64).transpose(1, 2))),                 # not contiguous
    dict(cache=_cache(block_size=8)),
    dict(cache=_cache(k=t.zeros(2, 12, 2, 64), v=t.zeros(2, 12, 2, 64), block_size=12)),
    dict(cache=_quantized(t.zeros(2, 16, 2, dtype=t.float16))),
    dict(cache=_quantized(t.zeros(2, 16, 1))),
    dict(table=t.zeros(4, 2, dtype=t.int64)),
    dict(table=t.zeros(4, dtype=t.int32)),
    dict(prefix=SharedPrefix(t.zeros(1), t.zeros(1, dtype=t.int64), t.zeros(2, dtype=t.int64))),
    dict(prefix=SharedPrefix(t.zeros(2, dtype=t.int64), t.zeros(1, dtype=t.int64), t.zeros(3, dtype=t.int64))),
    dict(prefix=SharedPrefix(t.zeros(1, dtype=t.int64), t.zeros(1, dtype=t.int64), t.zeros(1, dtype=t.int64))),
    dict(prefix=SharedPrefix(t.zeros(1, 1, dtype=t.int64), t.zeros(1, 1, dtype=t.int64), t.zeros(2, dtype=t.int64))),
]


@pytest.mark.parametrize("change", SHARED)
def test_refused_by_both_forms(change):
    with pytest.raises(ValueError):
        _decode(**change)
    with pytest.raises(ValueError):
        _prefill(**change)


@pytest.mark.parametrize("change", [dict(slots=t.zeros(2, dtype=t.int64)), dict(lens=t.zeros(3, 1, dtype=t.int64)),
                                    dict(lens=t.zeros(3)), dict(q=t.zeros(3, 4, 64, dtype=t.float64))])
def test_refused_decode(change):
    with pytest.raises(ValueError):
        _decode(**change)


def test_refused_prompts():
    with pytest.raises(ValueError):
        _prefill(k=t.zeros(3, 4, 64))       # the cache has 2 heads


def test_host_tensors_are_refused():
    with pytest.raises(RuntimeError):
        _decode()
    with pytest.raises(RuntimeError):
        _prefill()


def test_argument_codes():
    lib = _native.lib()
    some = 4096

    def decode(q_dtype=_native.F32, kv=_native.F32, batch=2, hq=4, hkv=2, d=64, ks=some, bs=16, width=2, slots=_native.I64,
               starts=_native.I64, groups=1, lens=some, q=some):
        return lib.kvfp8_shared_prefix_decode(q, q_dtype, hq * d, d, batch, hq, hkv, d, some, some, kv, ks, ks, 8, bs, some, 4,
                                              width, some, slots, some, _native.I32, 0.1, some, None, 0, None,
                                              some, _native.I64, lens, _native.I64, some, starts, groups)

    assert decode(q_dtype=_native.E4M3FN) == -1 and decode(kv=_native.I32) == -1
    assert decode(slots=_native.F32) == -1 and decode(starts=_native.F16) == -1
    assert decode(hq=3) == -2 and decode(bs=12) == -2 and decode(width=0) == -2 and decode(groups=-1) == -2 and decode(d=0) == -2
    assert decode(d=513) == -6 and decode(batch=2 ** 30) == -6 and decode(width=2 ** 30) == -6
    assert decode(q=None) == -4 and decode(lens=None) == -4 and decode(kv=_native.E4M3FN, ks=None) == -4
    assert decode(width=2 ** 10) == -5          # a long table is split over states in the workspace
    assert decode(batch=0) == 0

    def prefill(cu=_native.I32, rows=2, batch=1, longest=2, cus=some, lse=some, groups=1):
        return lib.kvfp8_shared_prefix_prefill(some, _native.F32, rows, 4, 2, 64, some, some, _native.F32, None, None, 8, 16,
                                               some, 4, 2 ** 10, some, _native.I64, some, _native.I64, some, _native.I64,
                                               groups, cus, cu, batch, longest, 0.1, some, lse, None, 0, None)

    assert prefill(cu=_native.F32) == -1 and prefill(batch=-1) == -2 and prefill(longest=-1) == -2
    assert prefill(cus=None) == -4 and prefill(lse=None) == -4 and prefill() == -5
    assert prefill(rows=0) == 0 and prefill(batch=0) == 0 and prefill(groups=0) == 0 and prefill(longest=0) == 0


def test_workspace_size_depends_on_shapes_only():
    fn = _native.lib().kvfp8_shared_prefix_workspace_bytes
    for prompt in (0, 1):
        assert fn(4, 8, 2, 64, 1, 64, 16, _native.E4M3FN, prompt) == fn(4, 8, 2, 64, 1, 64, 16, _native.E4M3FN, prompt) >= 0
        # A batch without groups, down to fewer pairs than a row block holds.
        assert fn(1, 2, 2, 64, 0, 64, 16, _native.E4M3FN, prompt) >= 0
    assert fn(0, 8, 2, 64, 1, 64, 16, _native.E4M3FN, 0) == 0


def test_rows_past_int32_offsets_take_the_generic_kernel():
    """2^19 KV heads of 128: a row of 16 tokens passes int32 offsets. The generic kernel keeps no states for so many
    rows; the matrix-core kernels would."""
    fn = _native.lib().kvfp8_shared_prefix_workspace_bytes
    assert fn(1, 2 ** 19, 2 ** 19, 128, 1, 4, 16, _native.E4M3FN, 0) == 0
    assert fn(1, 2 ** 18, 2 ** 18, 128, 1, 4, 16, _native.E4M3FN, 0) > 0


def test_tables_up_to_the_end_of_int32_are_refused():
    """The kernels look up to three blocks of tokens past the last one."""
    lib, some = _native.lib(), 4096

    def decode(width):
        return lib.kvfp8_shared_prefix_decode(some, _native.BF16, 256, 64, 1, 4, 2, 64, some, some, _native.BF16, None, None, 8, 16,
                                              some, 4, width, some, _native.I64, some, _native.I32, 0.1, some, None, 0, None,
                                              some, _native.I64, some, _native.I64, some, _native.I64, 1)

    assert decode(2 ** 27 - 512) == -6
    assert decode(2 ** 27 - 513) == -5          # taken, but for its workspace
