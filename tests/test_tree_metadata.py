"""The metadata of steps of drafted trees and the refusals of the tree operators, on the CPU:
masks, depths and slots against a walk over the parents; lists that do not fit raise before
anything is launched; the C entries reject bad arguments without a HIP call."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import tree as oracle
from tinybatch_amd import _lib, build_tree_metadata, commit_tree, tree_attention, verify_tree, verify_tree_greedy
from tinybatch_amd.tree import MAX_NODES


def random_trees(seed, sizes):
    g = np.random.default_rng(seed)
    return [[-1] + [int(g.integers(0, i)) for i in range(1, n)] if n else [] for n in sizes]


def meta_of(parents, cached, tables, bs=16, nb=64, **kw):
    kw = dict(num_heads=14, num_kv_heads=2, head_dim=64, dtype=torch.bfloat16) | kw
    return build_tree_metadata(parents, cached, tables, block_size=bs, num_blocks=nb, **kw)


@pytest.mark.parametrize("sizes", [[1], [5, 1, 0, 33], [64, 65, 3], [130]])
def test_masks_depths_and_slots(sizes):
    parents = random_trees(sum(sizes), sizes)
    g = np.random.default_rng(3)
    cached = [int(g.integers(0, 70)) for _ in sizes]
    ids = g.permutation(64)
    tables, at = [], 0
    for c, n in zip(cached, sizes):
        k = -(-(c + n) // 16)
        tables.append([int(x) for x in ids[at:at + k]])
        at += k
    m = meta_of(parents, cached, tables)
    row = 0
    for b, t in enumerate(parents):
        seen = oracle.visible(t)
        for i in range(len(t)):
            bits = [(int(m.mask_np[row, j // 32]) >> (j % 32)) & 1 for j in range(32 * m.mask_words)]
            assert bits == seen[i].astype(int).tolist() + [0] * (32 * m.mask_words - len(t))
            assert m.depths_np[row] == seen[i].sum() - 1 and m.row_seq_np[row] == b
            pos = cached[b] + i
            assert m.slot_mapping_np[row] == tables[b][pos // 16] * 16 + pos % 16
            row += 1
    assert row == m.num_rows and m.row_starts_np.tolist() == np.concatenate([[0], np.cumsum(sizes)]).tolist()
    m.to(torch.device("cpu"))
    assert m.positions.tolist() == [c + int(d) for c, n, s in zip(cached, sizes, m.row_starts_np) for d in m.depths_np[s:s + n]]


def test_visible_replaces_the_ancestors():
    v = np.zeros((3, 3), dtype=bool)
    v[0, 2] = v[2, 0] = True
    m = meta_of([[-1, 0, 0], [-1, 0]], [4, 0], [[1], [2]], visible=[v, None])
    assert m.mask_np[:, 0].tolist() == [4, 0, 1, 1, 3]


def test_lists_that_do_not_fit_are_refused():
    for bad in ([0], [-1, -1], [-1, 1], [-1, 0, 5], [-1, -2]):
        with pytest.raises(ValueError, match="parent"):
            build_tree_metadata([[-1], bad])
    with pytest.raises(ValueError, match=f"at most {MAX_NODES}"):
        build_tree_metadata([list(range(-1, MAX_NODES))])
    assert build_tree_metadata([list(range(-1, MAX_NODES - 1))]).max_nodes == MAX_NODES
    with pytest.raises(IndexError, match="needs 2 blocks"):
        meta_of([[-1, 0]], [15], [[3]])
    with pytest.raises(IndexError, match="outside the pool"):
        meta_of([[-1]], [0], [[64]])
    with pytest.raises(IndexError, match="outside the pool"):
        meta_of([[-1]], [16], [[-1, 2]])
    with pytest.raises(ValueError, match="share a pool slot"):
        meta_of([[-1], [-1]], [3, 3], [[7], [7]])
    meta_of([[-1], [-1]], [16, 16], [[7, 8], [7, 9]])            # a shared prefix is fine
    with pytest.raises(ValueError, match=">= 0"):
        meta_of([[-1]], [-1], [[0]])
    with pytest.raises(ValueError, match="multiple"):
        meta_of([[-1]], [0], [[0]], num_heads=13)
    with pytest.raises(ValueError, match="power of two"):
        meta_of([[-1]], [0], [[0]], bs=12)
    with pytest.raises(ValueError, match="describe"):
        meta_of([[-1]], [0], [[0]], dtype=torch.float64)
    with pytest.raises(ValueError, match="one entry per sequence"):
        meta_of([[-1], [-1]], [0], [[0]])
    with pytest.raises(ValueError, match="without cached_lens"):
        build_tree_metadata([[-1]], None, [[0]])
    with pytest.raises(ValueError, match=r"visible\[0\]"):
        build_tree_metadata([[-1, 0]], visible=[np.ones((2, 3), dtype=bool)])


def test_no_cpu_fallback():
    m = meta_of([[-1, 0]], [0], [[0]]).to(torch.device("cpu"))
    with pytest.raises(RuntimeError, match="GPU"):
        tree_attention(torch.zeros(2, 14, 64, dtype=torch.bfloat16), torch.zeros(64, 2, 2, 16, 64, dtype=torch.bfloat16), m)
    ids = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="GPU"):
        verify_tree(m, ids, torch.zeros(2), torch.zeros(2, 8))
    with pytest.raises(RuntimeError, match="GPU"):
        verify_tree_greedy(m, ids, ids)
    with pytest.raises(RuntimeError, match="GPU"):
        commit_tree(torch.zeros(1, 64, 2, 2, 16, 64), m, torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


def test_entries_reject_bad_arguments_without_launching():
    L, f = _lib.lib(), ctypes.c_void_p(4096)
    bad, unsupported = _lib.TB_ERR_INVALID_ARG, _lib.TB_ERR_UNSUPPORTED

    def verify(probs=f, stride=100, draft=None, dstride=0, vocab=100, dt=0, tokens=f, seqs=2, width=4, acc=f):
        return L.tb_tree_verify(probs, stride, draft, dstride, vocab, dt, tokens, f, f, f, seqs, acc, f, f, width, None)

    assert verify(stride=99) == bad                    # rows overlap
    assert verify(draft=f, dstride=99) == bad
    assert verify(vocab=0) == bad and verify(dt=3) == bad and verify(width=0) == bad
    assert verify(probs=None) == bad and verify(tokens=None) == bad and verify(acc=None) == bad
    assert verify(width=MAX_NODES + 1) == unsupported
    assert verify(seqs=0, probs=None) == _lib.TB_OK
    assert L.tb_tree_verify_greedy(f, f, f, f, 2, f, f, f, 0, None) == bad
    assert L.tb_tree_verify_greedy(None, f, f, f, 2, f, f, f, 4, None) == bad
    assert L.tb_tree_verify_greedy(None, f, f, f, 0, f, f, f, 4, None) == _lib.TB_OK

    def commit(storage=f, layers=2, stride=1 << 20, nb=8, hkv=2, d=64, bs=16, dt=1, width=4, seqs=2):
        return L.tb_tree_commit(storage, layers, stride, nb, f, 4, f, seqs, f, width, f, hkv, d, bs, dt, None)

    assert commit(storage=ctypes.c_void_p(4104)) == bad          # not 16-byte aligned
    assert commit(stride=8 * 2 * 2 * 16 * 64 * 2 - 16) == bad    # layers overlap
    assert commit(bs=12) == bad and commit(width=0) == bad and commit(hkv=0) == bad
    assert commit(d=4) == unsupported                            # rows of 8 bytes
    assert commit(layers=0) == _lib.TB_OK and commit(seqs=0) == _lib.TB_OK
