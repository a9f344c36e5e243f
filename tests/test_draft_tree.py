"""Drafted trees without a GPU: what the calls and the C entries refuse."""

from types import SimpleNamespace

import pytest
import torch as t

from aiproj_amd import _native
from aiproj_amd.kernals.draft_tree import DraftTree, accept_draft, tree_attention

FP8, BF16, F32, I32, I64 = _native.E4M3FN, _native.BF16, _native.F32, _native.I32, _native.I64
SOME = 4096          # an address that a refused call does not look at


def _case(**more):
    c = SimpleNamespace(q=t.zeros(3, 4, 64, dtype=t.bfloat16), tokens=t.zeros(3, dtype=t.int64), best=t.zeros(3, dtype=t.int64),
                        cache=SimpleNamespace(k=t.zeros(5, 16, 2, 64, dtype=t.bfloat16), v=t.zeros(5, 16, 2, 64, dtype=t.bfloat16),
                                              k_scales=None, v_scales=None, quantized=False, block_size=16),
                        slots=t.zeros(2, dtype=t.int64), lens=t.ones(2, dtype=t.int32), table=t.zeros(4, 3, dtype=t.int32),
                        starts=t.tensor([0, 1, 3]), parents=t.tensor([-1, -1, 0]), max_nodes=2)
    for name, x in more.items():
        setattr(c, name, x)
    c.ctx = SimpleNamespace(cache_slots=c.slots, context_lengths=c.lens, block_table=c.table)
    c.tree = DraftTree(c.starts, c.parents, c.max_nodes)
    return c


BAD = [dict(slots=t.zeros(3, dtype=t.int64)), dict(lens=t.ones(1, dtype=t.int32)), dict(lens=t.ones(2)), dict(table=t.zeros(4, 3)),
       dict(table=t.zeros(3, dtype=t.int32)), dict(starts=t.tensor([0, 1, 3, 3])), dict(starts=t.tensor([], dtype=t.int64)),
       dict(starts=t.tensor([[0, 1, 3]])), dict(parents=t.tensor([-1, 0])), dict(parents=t.tensor([-1.0, -1.0, 0.0])), dict(max_nodes=-1),
       dict(max_nodes=257), dict(max_nodes=True), dict(max_nodes=2.0)]


@pytest.mark.parametrize("bad", BAD + [dict(q=t.zeros(3, 4, 64, dtype=t.float64)), dict(q=t.zeros(3, 256)), dict(q=t.zeros(3, 5, 64)),
                                       dict(q=t.zeros(3, 4, 32)), dict(q=t.zeros(2, 4, 64))])
def test_attention_refuses(bad):
    c = _case(**bad)
    with pytest.raises(ValueError):
        tree_attention(c.q, c.cache, c.ctx, c.tree)


@pytest.mark.parametrize("bad", BAD + [dict(tokens=t.zeros(2, dtype=t.int64)), dict(best=t.zeros(3)), dict(best=t.zeros(3, 1, dtype=t.int64)),
                                       dict(max_nodes=0)])
def test_accept_refuses(bad):
    c = _case(**bad)
    with pytest.raises((ValueError, RuntimeError)):
        accept_draft(c.tokens, c.best, c.tree, [c.cache], c.ctx)


def test_cpu_tensors_are_refused():
    c = _case()
    with pytest.raises(RuntimeError, match="GPU"):
        tree_attention(c.q, c.cache, c.ctx, c.tree)
    with pytest.raises(RuntimeError, match="GPU"):
        accept_draft(c.tokens, c.best, c.tree, [c.cache], c.ctx)


def test_trees_from_lists():
    lists = [[-1, 0, 0, 1], [-1], [-1, 0, -1, 2]]
    tree = DraftTree.from_parents(lists, "cpu")
    assert tree.starts.tolist() == [0, 4, 5, 9] and tree.parents.tolist() == sum(lists, []) and tree.max_nodes == 4
    assert DraftTree.depths(lists) == [[0, 1, 1, 2], [0], [0, 1, 0, 1]]
    for bad in ([[]], [[0]], [[-1, 1]], [[-1, -2]], [[-1] * 257], [[-1, 0], [2]]):
        with pytest.raises(ValueError):
            DraftTree.from_parents(bad, "cpu")


def _attend(rows=3, hq=4, hkv=2, d=64, q_dtype=BF16, kv=BF16, scales=None, blocks=5, page=16, bt_rows=4, width=3, slots=I64, ctx=I32,
            starts=I64, parents=I64, seqs=2, nodes=2, q=SOME, tree=SOME, out=SOME, ws=None, size=0):
    return (q, q_dtype, hq * d, d, rows, hq, hkv, d, SOME, SOME, kv, scales, scales, blocks, page, SOME, bt_rows, width, SOME, slots, SOME,
            ctx, tree, starts, tree, parents, seqs, nodes, 0.125, out, ws, size, None)


@pytest.mark.parametrize("more,code", [
    (dict(q_dtype=FP8), -1), (dict(kv=I32), -1), (dict(slots=F32), -1), (dict(ctx=BF16), -1), (dict(starts=FP8), -1), (dict(parents=F32), -1),
    (dict(rows=-1), -2), (dict(hq=5), -2), (dict(hkv=0), -2), (dict(d=0), -2), (dict(blocks=0), -2), (dict(page=12), -2), (dict(width=0), -2),
    (dict(bt_rows=0), -2), (dict(seqs=-1), -2), (dict(nodes=-1), -2), (dict(d=513), -6), (dict(nodes=257), -6), (dict(rows=2 ** 20), -6),
    (dict(rows=2 ** 62), -6), (dict(seqs=2 ** 31 - 1, nodes=256), -6), (dict(seqs=2 ** 19), -6), (dict(width=2 ** 60), -6),
    (dict(width=2 ** 27), -6), (dict(bt_rows=2 ** 31), -6), (dict(hq=2 ** 30, hkv=2 ** 30, d=64, page=16), -6), (dict(q=None), -4),
    (dict(tree=None), -4), (dict(out=None), -4), (dict(kv=FP8), -4), (dict(), -5), (dict(kv=FP8, scales=SOME), -5),
    (dict(ws=SOME, size=64), -5), (dict(rows=0), 0), (dict(seqs=0), 0), (dict(nodes=0), 0)])
def test_attention_entry_refuses(more, code):
    for entry in (_native.lib().kvfp8_tree_attention, _native.fn("kvfp8_tree_attention")):
        assert entry(*_attend(**more)) == code


@pytest.mark.parametrize("sizes", [(0, 2, 4, 2, 64, 16), (2, 0, 4, 2, 64, 16), (2, 2, 5, 2, 64, 16), (2, 257, 4, 2, 64, 16), (2, 2, 4, 2, 513, 16),
                                   (2 ** 31 - 1, 256, 4, 2, 64, 16), (2, 2, 2 ** 31 - 1, 1, 64, 16), (2, 2, 4, 2, 64, 0)])
def test_workspace_of_sizes_that_are_refused(sizes):
    assert [_native.lib().kvfp8_tree_attention_workspace_bytes(*sizes, kv) for kv in range(4)] == [0] * 4


def test_workspace_of_sizes_that_are_taken():
    assert _native.lib().kvfp8_tree_attention_workspace_bytes(2, 2, 4, 2, 64, 16, FP8) > 0
    assert _native.lib().kvfp8_tree_attention_workspace_bytes(2, 2, 4, 2, 40, 16, FP8) == 0        # the vector ALU needs none


def _accept(tok=I64, best=I64, starts=I64, parents=I64, rows=3, seqs=2, nodes=2, slots=I64, ctx=I32, bt_rows=4, width=3, blocks=5, page=16,
            caches=None, layers=0, row=256, scale=8, tree=SOME, out=SOME):
    return (SOME, tok, SOME, best, tree, starts, SOME, parents, rows, seqs, nodes, SOME, slots, SOME, ctx, SOME, bt_rows, width, blocks, page,
            caches, layers, row, scale, out, SOME, SOME, None)


@pytest.mark.parametrize("more,code", [
    (dict(tok=F32), -1), (dict(best=FP8), -1), (dict(starts=F32), -1), (dict(parents=BF16), -1), (dict(slots=F32), -1), (dict(ctx=F32), -1),
    (dict(rows=-1), -2), (dict(seqs=-1), -2), (dict(nodes=0), -2), (dict(layers=-1), -2), (dict(page=24), -2), (dict(row=0), -2),
    (dict(scale=-4), -2), (dict(scale=6), -2), (dict(width=0), -2), (dict(nodes=257), -6), (dict(rows=2 ** 31), -6), (dict(seqs=2 ** 17), -6),
    (dict(width=2 ** 60), -6), (dict(blocks=2 ** 52), -6), (dict(tree=None), -4), (dict(out=None), -4), (dict(layers=1), -4), (dict(seqs=0), 0)])
def test_accept_entry_refuses(more, code):
    for entry in (_native.lib().kvfp8_accept_draft, _native.fn("kvfp8_accept_draft")):
        assert entry(*_accept(**more)) == code


def test_accept_entry_refuses_addresses():
    import array

    entry = _native.lib().kvfp8_accept_draft
    for four, code in (((SOME, SOME, SOME, 0), -4), ((0, SOME, SOME, SOME), -4), ((SOME, SOME, SOME + 2, SOME), -3)):
        held = array.array("Q", four)
        assert entry(*_accept(caches=held.buffer_info()[0], layers=1)) == code
