"""Attention of a batch whose sequences share long prefixes in the paged cache.

Many answers to one prompt, or many users of one system prompt, hold the same first tokens. They are
kept once: a prefix is a request of its own (its own slot and pages in the `PageAllocator`), a sequence's
slot holds what comes behind it, and `SharedPrefix` says which sequences share which prefix. The
matrix-core kernels then read the prefix once for all rows of its group instead of once per sequence:
float8_e4m3fn caches of head size 64, 80, 96, 112 or 128 with q of any type, and bf16 or f16 caches of
head size 64 or 128 with q of their type, pages of 16 tokens and more, 16-byte aligned, fewer than 2^22
(row, q head) pairs a call. Everything else goes to a vector-ALU kernel in which each row reads its
prefix by itself (32 sequences of 32 heads behind 4096 tokens: 1.2 to 2.0 ms, where the matrix cores
take 24 to 33 µs).

* `shared_prefix_decode_attention(q, paged_kv_cache, cache_batch_context, prefix)` is
  `decode_attention_wrapper` with the prefix in front: q [B, Hq, D], one new token a sequence;
  `context_lengths` count a sequence's own tokens. A sequence without any token gives zeros.
* `append_shared_prefix_decode_attention(q, ks, vs, paged_kv_cache, cache_batch_context, prefix)` is the
  decode step: the new tokens' cache write, then the attention.
* `shared_prefix_prefill_attention(q, k, v, cum_seq, batch_max_seq_len, scale, paged_kv_cache,
  block_table, prefix) -> (output, lse)` is `flash_attention_forward` with the prefix in front: packed
  prompts that continue their group's prefix. Their own keys are the unquantized k and v, as there; the
  prefix comes from the cache as it is stored. Rows of no sequence stay unwritten, as there. The
  two are joined through `output` and `lse` of that call: an output of 16 bits is rounded twice, and
  the weights of prefix and prompt against each other are exact to |lse| 2^-23.

Positions behind a prefix of P tokens start at P: the caller rotates q and k accordingly.

Nothing is synchronized with the host and no device value is read: prefixes and groups may change
between replays of a captured call. No gradients. The reference has no counterpart: its decode reads
every sequence's own pages (`kernals/decode_attention.py:39-191`).
"""

from __future__ import annotations

import functools
import math
from dataclasses import dataclass

import torch as t

from aiproj_amd import _native
from aiproj_amd.kernals.decode_attention import _Q_DTYPES, _index_tensor, _workspace
from aiproj_amd.kernals.flash_attention import flash_attention_forward


@dataclass(frozen=True)
class SharedPrefix:
    """Group g is the sequences `starts[g]` .. `starts[g + 1] - 1` of the batch; its prefix is the first
    `lengths[g]` tokens on block-table row `slots[g]`. Sequences before `starts[0]` and from
    `starts[-1]` on have none. int32 or int64 vectors on the cache's device; `starts` does not
    decrease."""

    slots: t.Tensor      # [G]
    lengths: t.Tensor    # [G]
    starts: t.Tensor     # [G + 1]

    @classmethod
    def one(cls, slot: int, length: int, batch: int, device) -> "SharedPrefix":
        """One prefix in front of a whole batch."""
        return cls(t.tensor([slot], device=device), t.tensor([length], device=device), t.tensor([0, batch], device=device))


def _check_prefix(prefix, what: str):
    slots, lengths, starts = prefix.slots, prefix.lengths, prefix.starts
    if slots.ndim != 1 or lengths.shape != slots.shape or starts.ndim != 1 or starts.shape[0] != slots.shape[0] + 1:
        raise ValueError(f"{what}: prefix slots [G], lengths [G] and starts [G + 1]")
    return _index_tensor(slots), _index_tensor(lengths), _index_tensor(starts)


def _check_cache(cache, block_table, d: int, hq: int, what: str):
    """(k, v, k_scales, v_scales, block table) of a paged cache, contiguous."""
    k, v = cache.k, cache.v
    shape, block_size = k.shape, cache.block_size
    if len(shape) != 4 or shape != v.shape or shape[3] != d or hq % shape[2]:
        raise ValueError(f"{what}: cache rows [num_blocks, block_size, Hkv, D] that match q [.., Hq, D]")
    if shape[1] != block_size or block_size & (block_size - 1):
        raise ValueError(f"{what}: block size must be the cache's and a power of two")
    if block_table.ndim != 2 or block_table.dtype != t.int32:
        raise ValueError(f"{what}: the block table is an int32 matrix")
    if v.dtype != k.dtype:
        raise ValueError(f"{what}: k and v share one dtype")
    contiguous = k.is_contiguous() and v.is_contiguous()
    k_scales = v_scales = None
    if cache.quantized:
        k_scales, v_scales = cache.k_scales, cache.v_scales
        if (k.dtype != t.float8_e4m3fn or k_scales.dtype != t.float32 or v_scales.dtype != t.float32
                or k_scales.shape != shape[:3] or v_scales.shape != shape[:3]):
            raise ValueError(f"{what}: a quantized cache holds float8_e4m3fn and float32 scales per row")
        contiguous = contiguous and k_scales.is_contiguous() and v_scales.is_contiguous()
    elif k.dtype not in _Q_DTYPES:
        raise ValueError(f"{what}: unsupported cache dtype {k.dtype}")
    if not contiguous:
        raise ValueError(f"{what}: cache tensors must be contiguous")
    return k, v, k_scales, v_scales, block_table if block_table.is_contiguous() else block_table.contiguous()


@functools.lru_cache(maxsize=256)
def _workspace_bytes(rows, hq, hkv, d, groups, bt_width, block_size, kv_code, prompt) -> int:
    """kvfp8_shared_prefix_workspace_bytes, which depends on shapes only (cached per shape)."""
    return _native.lib().kvfp8_shared_prefix_workspace_bytes(rows, hq, hkv, d, groups, bt_width, block_size, kv_code, prompt)


def shared_prefix_decode_attention(q: t.Tensor, paged_kv_cache, cache_batch_context, prefix: SharedPrefix) -> t.Tensor:
    what = "shared_prefix_decode_attention"
    if q.ndim != 3:
        raise ValueError(f"{what}: q [B, Hq, D]")
    b, hq, d = q.shape
    ctx = cache_batch_context
    k, v, k_scales, v_scales, table = _check_cache(paged_kv_cache, ctx.block_table, d, hq, what)
    p_slots, p_lens, p_starts = _check_prefix(prefix, what)
    slots, lens = _index_tensor(ctx.cache_slots), _index_tensor(ctx.context_lengths)
    if slots.shape != (b,) or lens.shape != (b,):
        raise ValueError(f"{what}: one cache slot and one context length a sequence")
    if q.dtype not in _Q_DTYPES:
        raise ValueError(f"{what}: unsupported q dtype {q.dtype}")
    device = _native.require_gpu(q, k, v, k_scales, v_scales, table, slots, lens, p_slots, p_lens, p_starts, what=what)
    output = t.empty((b, hq, d), dtype=q.dtype, device=q.device)
    if b == 0:
        return output
    if q.stride(-1) != 1:
        q = q.contiguous()
    num_blocks, block_size, hkv, _ = k.shape
    bt_rows, bt_width = table.shape
    groups, code = p_slots.shape[0], _native.TORCH_TO_CODE
    kv_code, stream = code[k.dtype], _native.stream_handle(device)
    workspace = _workspace(device, stream, _workspace_bytes(b, hq, hkv, d, groups, bt_width, block_size, kv_code, 0))
    rc = _native.fn("kvfp8_shared_prefix_decode")(
        q.data_ptr(), code[q.dtype], q.stride(0), q.stride(1), b, hq, hkv, d, k.data_ptr(), v.data_ptr(),
        kv_code, _native.ptr(k_scales), _native.ptr(v_scales), num_blocks, block_size, table.data_ptr(), bt_rows,
        bt_width, slots.data_ptr(), code[slots.dtype], lens.data_ptr(), code[lens.dtype], 1.0 / math.sqrt(d),
        output.data_ptr(), workspace.data_ptr(), workspace.numel(), stream, p_slots.data_ptr(), code[p_slots.dtype],
        p_lens.data_ptr(), code[p_lens.dtype], p_starts.data_ptr(), code[p_starts.dtype], groups)
    _native.check(rc, "kvfp8_shared_prefix_decode")
    return output


def append_shared_prefix_decode_attention(q: t.Tensor, ks: t.Tensor, vs: t.Tensor, paged_kv_cache, cache_batch_context,
                                          prefix: SharedPrefix) -> t.Tensor:
    """`paged_kv_cache.append_kv(ctx.physical_blocks, ctx.block_offsets, ks, vs)` and the attention over
    the prefix and the own tokens, which hold the new one."""
    ctx = cache_batch_context
    paged_kv_cache.append_kv(ctx.physical_blocks, ctx.block_offsets, ks, vs)
    return shared_prefix_decode_attention(q, paged_kv_cache, ctx, prefix)


def shared_prefix_prefill_attention(q: t.Tensor, k: t.Tensor, v: t.Tensor, cum_seq: t.Tensor, batch_max_seq_len: int,
                                    scale: float, paged_kv_cache, block_table: t.Tensor,
                                    prefix: SharedPrefix) -> tuple[t.Tensor, t.Tensor]:
    what = "shared_prefix_prefill_attention"
    if q.ndim != 3:
        raise ValueError(f"{what}: q [T, Hq, D]")
    total, hq, d = q.shape
    pk, pv, k_scales, v_scales, table = _check_cache(paged_kv_cache, block_table, d, hq, what)
    if k.ndim != 3 or k.shape[1] != pk.shape[2]:
        raise ValueError(f"{what}: k and v have the cache's heads")
    p_slots, p_lens, p_starts = _check_prefix(prefix, what)
    device = _native.require_gpu(q, k, v, cum_seq, pk, pv, k_scales, v_scales, table, p_slots, p_lens, p_starts, what=what)
    if not cum_seq.is_contiguous():
        cum_seq = cum_seq.contiguous()
    output, lse = flash_attention_forward(q, k, v, cum_seq, batch_max_seq_len, scale)
    batch, longest = cum_seq.shape[0] - 1, int(batch_max_seq_len)
    if total == 0 or batch <= 0 or longest <= 0 or p_slots.shape[0] == 0:
        return output, lse
    num_blocks, block_size, hkv, _ = pk.shape
    bt_rows, bt_width = table.shape
    groups, code = p_slots.shape[0], _native.TORCH_TO_CODE
    kv_code, stream = code[pk.dtype], _native.stream_handle(device)
    workspace = _workspace(device, stream, _workspace_bytes(total, hq, hkv, d, groups, bt_width, block_size, kv_code, 1))
    rc = _native.fn("kvfp8_shared_prefix_prefill")(
        q.data_ptr(), code[q.dtype], total, hq, hkv, d, pk.data_ptr(), pv.data_ptr(), kv_code,
        _native.ptr(k_scales), _native.ptr(v_scales), num_blocks, block_size, table.data_ptr(), bt_rows, bt_width,
        p_slots.data_ptr(), code[p_slots.dtype], p_lens.data_ptr(), code[p_lens.dtype], p_starts.data_ptr(),
        code[p_starts.dtype], groups, cum_seq.data_ptr(), code[cum_seq.dtype], batch, longest, float(scale),
        output.data_ptr(), lse.data_ptr(), workspace.data_ptr(), workspace.numel(), stream)
    _native.check(rc, "kvfp8_shared_prefix_prefill")
    return output, lse
