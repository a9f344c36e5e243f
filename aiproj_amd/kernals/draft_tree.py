"""Checking trees of drafted tokens against a model in one pass: their attention over the paged cache, and what is kept.

A drafter proposes several continuations of a sequence as a tree. Its node 0 is the sequence's last chosen token, which is
not in the cache yet, and every other node a guess at what follows its parent. The model runs over all nodes at once: their
keys and values go to the cache behind the sequence's tokens, in node order, and each node attends the tokens before the
draft, the nodes above it and itself. The model's choices then say which path holds, and its cache rows are moved together.

* `DraftTree(starts, parents, max_nodes)`: sequence b has the nodes `starts[b]` .. `starts[b + 1] - 1` of the packed
  rows; `parents[r]` is the number of node r's parent within its sequence, -1 for a root. Parents come before their
  children (anything else counts as a root). `max_nodes` (a host int, at most 256): the most nodes of a sequence; rows
  past it are left out.
* `tree_attention(q, paged_kv_cache, cache_batch_context, tree)`: q [T, Hq, D] -> [T, Hq, D]. `context_lengths` count a
  sequence's tokens with its nodes, as `PageAllocator.create_container` gives them. A slot outside the table, or fewer
  tokens than nodes, gives zeros. Rows of no sequence stay unwritten. Keys and values of nodes that a row does not attend
  do not reach it, NaN and infinities included.
* `append_tree_attention(q, ks, vs, paged_kv_cache, cache_batch_context, tree)`: the nodes' cache write, then the attention.
* `accept_draft(tokens, best, tree, caches, cache_batch_context) -> AcceptedDraft`: `tokens` [T] of the nodes and `best` [T],
  the model's choice behind each (int32 or int64). From node 0 down, the child of lowest number whose token is the
  choice; the kept nodes' rows are moved behind the tokens before the draft in every cache of the list (the layers'
  caches, of one shape and type, without memory in common), codes and scales. The sequence then has its tokens before the
  draft and `counts` more. Sequences of a batch share no pages there.

Matrix cores: float8_e4m3fn caches of head size 64, 80, 96, 112 or 128 with q of any type, and bf16 or f16 caches of head
size 64 or 128 with q of their type, pages of 16 tokens and more, 16-byte aligned. Everything else, up to head size 512, goes
to a vector-ALU kernel. Rows x q heads and sequences x max_nodes x q heads are below 2^22 each (65535 nodes of 64 heads; 255
sequences of up to 256 of them); larger batches are refused, and go in parts.

Nothing is synchronized with the host and no device value is read: trees, lengths and pages may change between replays of a
captured call. No gradients: queries, keys and values that require them are refused while a graph is recorded, and dual
tensors always. The reference has no counterpart: a decode step there has one new token a sequence
(`kernals/decode_attention.py:39-191`).
"""

from __future__ import annotations

import functools
import math
from array import array
from dataclasses import dataclass
from typing import NamedTuple

import torch as t

from aiproj_amd import _native
from aiproj_amd.kernals.decode_attention import _Q_DTYPES, _index_tensor, _workspace
from aiproj_amd.kernals.shared_prefix_attention import _check_cache

MAX_NODES = 256


@dataclass(frozen=True)
class DraftTree:
    starts: t.Tensor      # [B + 1] int32 or int64
    parents: t.Tensor     # [T] int32 or int64
    max_nodes: int

    @classmethod
    def from_parents(cls, parents: list[list[int]], device) -> "DraftTree":
        """The trees with these parents, checked: node 0 a root, every other parent -1 or a smaller node number."""
        for own in parents:
            if not own or len(own) > MAX_NODES or own[0] != -1 or any(not -1 <= p < i for i, p in enumerate(own)):
                raise ValueError(f"DraftTree: 1 to {MAX_NODES} nodes, node 0 a root, parents before their children")
        starts = [0]
        for own in parents:
            starts.append(starts[-1] + len(own))
        flat = [p for own in parents for p in own]
        return cls(t.tensor(starts, dtype=t.int32, device=device), t.tensor(flat, dtype=t.int32, device=device),
                   max(map(len, parents), default=0))

    @staticmethod
    def depths(parents: list[list[int]]) -> list[list[int]]:
        """How far each node is behind its root: its position behind that of node 0."""
        found = []
        for own in parents:
            deep = []
            for p in own:
                deep.append(0 if p < 0 else deep[p] + 1)
            found.append(deep)
        return found


class AcceptedDraft(NamedTuple):
    counts: t.Tensor        # [B] int32: kept nodes, node 0 among them
    path: t.Tensor          # [B, max_nodes] int32: their numbers, -1 behind them
    next_tokens: t.Tensor   # [B] int64: the model's choice behind the last of them, -1 without nodes


def _check_tree(tree: DraftTree, ctx, what: str):
    """(starts, parents, slots, lengths), contiguous index vectors."""
    starts, parents, slots, lens = (_index_tensor(x) for x in (tree.starts, tree.parents, ctx.cache_slots, ctx.context_lengths))
    if starts.ndim != 1 or parents.ndim != 1 or starts.shape[0] < 1:
        raise ValueError(f"{what}: tree starts [B + 1] and parents [T]")
    if isinstance(tree.max_nodes, bool) or not isinstance(tree.max_nodes, int) or not 0 <= tree.max_nodes <= MAX_NODES:
        raise ValueError(f"{what}: max_nodes is an int from 0 to {MAX_NODES}")
    b = starts.shape[0] - 1
    if slots.shape != (b,) or lens.shape != (b,):
        raise ValueError(f"{what}: one cache slot and one context length a sequence")
    return starts, parents, slots, lens


@functools.lru_cache(maxsize=256)
def _workspace_bytes(seqs, max_nodes, hq, hkv, d, block_size, kv_code) -> int:
    """kvfp8_tree_attention_workspace_bytes, which depends on shapes only (cached per shape)."""
    return _native.lib().kvfp8_tree_attention_workspace_bytes(seqs, max_nodes, hq, hkv, d, block_size, kv_code)


def tree_attention(q: t.Tensor, paged_kv_cache, cache_batch_context, tree: DraftTree) -> t.Tensor:
    what = "tree_attention"
    if q.ndim != 3:
        raise ValueError(f"{what}: q [T, Hq, D]")
    rows, hq, d = q.shape
    ctx = cache_batch_context
    k, v, k_scales, v_scales, table = _check_cache(paged_kv_cache, ctx.block_table, d, hq, what)
    starts, parents, slots, lens = _check_tree(tree, ctx, what)
    if parents.shape != (rows,):
        raise ValueError(f"{what}: one parent a row of q")
    if q.dtype not in _Q_DTYPES:
        raise ValueError(f"{what}: unsupported q dtype {q.dtype}")
    _native.refuse_gradients(q, what=what)
    device = _native.require_gpu(q, k, v, k_scales, v_scales, table, starts, parents, slots, lens, what=what)
    output = t.empty((rows, hq, d), dtype=q.dtype, device=device)
    seqs = starts.shape[0] - 1
    if rows == 0 or seqs == 0 or tree.max_nodes == 0:
        return output
    if q.stride(-1) != 1:
        q = q.contiguous()
    num_blocks, block_size, hkv, _ = k.shape
    code = _native.TORCH_TO_CODE
    kv_code = code[k.dtype]
    workspace = _workspace(device, _native.stream_handle(device), _workspace_bytes(seqs, tree.max_nodes, hq, hkv, d, block_size, kv_code))
    _native.launch(
        "kvfp8_tree_attention", device, q.data_ptr(), code[q.dtype], q.stride(0), q.stride(1), rows, hq, hkv, d, k.data_ptr(),
        v.data_ptr(), kv_code, _native.ptr(k_scales), _native.ptr(v_scales), num_blocks, block_size, table.data_ptr(),
        table.shape[0], table.shape[1], slots.data_ptr(), code[slots.dtype], lens.data_ptr(), code[lens.dtype], starts.data_ptr(),
        code[starts.dtype], parents.data_ptr(), code[parents.dtype], seqs, tree.max_nodes, 1.0 / math.sqrt(d), output.data_ptr(),
        workspace.data_ptr(), workspace.numel())
    return output


def append_tree_attention(q: t.Tensor, ks: t.Tensor, vs: t.Tensor, paged_kv_cache, cache_batch_context, tree: DraftTree) -> t.Tensor:
    """`paged_kv_cache.append_kv(ctx.physical_blocks, ctx.block_offsets, ks, vs)` and the attention over the cache with the nodes."""
    ctx = cache_batch_context
    _native.refuse_gradients(q, ks, vs, what="append_tree_attention")
    paged_kv_cache.append_kv(ctx.physical_blocks, ctx.block_offsets, ks, vs)
    return tree_attention(q, paged_kv_cache, ctx, tree)


def accept_draft(tokens: t.Tensor, best: t.Tensor, tree: DraftTree, caches, cache_batch_context) -> AcceptedDraft:
    what = "accept_draft"
    ctx = cache_batch_context
    starts, parents, slots, lens = _check_tree(tree, ctx, what)
    tokens, best, rows = _index_tensor(tokens), _index_tensor(best), parents.shape[0]
    if tokens.shape != (rows,) or best.shape != (rows,):
        raise ValueError(f"{what}: one token and one choice a node")
    table = ctx.block_table
    if table.ndim != 2 or table.dtype != t.int32:
        raise ValueError(f"{what}: the block table is an int32 matrix")
    table = table if table.is_contiguous() else table.contiguous()
    device = _native.require_gpu(tokens, best, starts, parents, slots, lens, table, what=what)
    seqs, most = starts.shape[0] - 1, tree.max_nodes
    if most == 0:
        raise ValueError(f"{what}: max_nodes is at least 1")
    shape, row_bytes, scale_bytes, addresses, index, same = (1, 1, 1, 1), 1, 0, array("Q"), device.index, True
    for i, cache in enumerate(caches):
        k, v, quantized = cache.k, cache.v, cache.quantized
        if i == 0:
            shape, dtype, scaled = k.shape, k.dtype, quantized
            if len(shape) != 4 or shape[1] & (shape[1] - 1) or dtype not in _native.TORCH_TO_CODE:
                raise ValueError(f"{what}: cache rows [num_blocks, block_size, Hkv, D], the block size a power of two")
            row_bytes, scale_bytes, scale_shape = shape[2] * shape[3] * k.element_size(), 4 * shape[2] if scaled else 0, shape[:3]
        if k.shape != shape or v.shape != shape or k.dtype != dtype or v.dtype != dtype or quantized != scaled:
            raise ValueError(f"{what}: caches of one shape and type")
        same = same and k.get_device() == v.get_device() == index and k.is_contiguous() and v.is_contiguous()
        if scaled:
            ks, vs = cache.k_scales, cache.v_scales
            if ks.dtype != t.float32 or vs.dtype != t.float32 or ks.shape != scale_shape or vs.shape != scale_shape:
                raise ValueError(f"{what}: a quantized cache holds float32 scales per row")
            same = same and ks.get_device() == vs.get_device() == index and ks.is_contiguous() and vs.is_contiguous()
            addresses.extend((k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr()))
        else:
            addresses.extend((k.data_ptr(), v.data_ptr(), 0, 0))
    if not same:
        raise ValueError(f"{what}: cache tensors are contiguous and on the tokens' device")
    counts = t.empty(seqs, dtype=t.int32, device=device)
    path = t.empty((seqs, most), dtype=t.int32, device=device)
    next_tokens = t.empty(seqs, dtype=t.int64, device=device)
    if seqs:
        code = _native.TORCH_TO_CODE
        _native.launch(
            "kvfp8_accept_draft", device, tokens.data_ptr(), code[tokens.dtype], best.data_ptr(), code[best.dtype], starts.data_ptr(),
            code[starts.dtype], parents.data_ptr(), code[parents.dtype], rows, seqs, most, slots.data_ptr(), code[slots.dtype],
            lens.data_ptr(), code[lens.dtype], table.data_ptr(), table.shape[0], table.shape[1], shape[0], shape[1],
            addresses.buffer_info()[0], len(addresses) // 4, row_bytes, scale_bytes, counts.data_ptr(), path.data_ptr(),
            next_tokens.data_ptr())
    return AcceptedDraft(counts, path, next_tokens)
