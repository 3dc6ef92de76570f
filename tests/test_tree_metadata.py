"""The metadata of steps of drafted trees and the refusals of the tree operators, on the CPU:
masks, depths and slots against a walk over the parents; lists that do not fit raise before
anything is launched; the C entries reject bad arguments without a HIP call."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import tree as oracle
from tinybatch_amd import _lib, build_tree_metadata, commit_tree, tree_attention, verify_tree, verify_tree_greedy
from tinybatch_amd.tree import MAX_NODES, MAX_VOCAB


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
    with pytest.raises(ValueError, match="another sequence's cached"):
        meta_of([[-1], [-1]], [4, 9], [[7], [7]])                # the first's node would overwrite the second's position 4
    with pytest.raises(ValueError, match="another sequence's cached"):
        meta_of([[-1], []], [20, 32], [[6, 7], [5, 7]])
    meta_of([[-1], []], [20, 20], [[6, 7], [5, 7]])              # behind what the other one has there
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


def test_tables_end_with_no_block():
    m = meta_of([[-1], [-1, 0], []], [40, 3, 0], [[7, 8, 9, 10], [5, 6], [4]])
    assert m.block_tables_np.tolist() == [[7, 8, 9], [5, -1, -1], [-1, -1, -1]]


@pytest.mark.parametrize("as_", [np.asarray, torch.tensor, tuple])
def test_lists_of_any_kind(as_):
    m = meta_of([as_([-1, 0, 0]), as_([-1])], as_([20, 5]), [as_([3, 9, 1, 1, 1]), as_([2])])
    n = meta_of([[-1, 0, 0], [-1]], [20, 5], [[3, 9], [2]])
    for name in ("parents_np", "positions_np", "mask_np", "block_tables_np", "slot_mapping_np", "work_np"):
        assert np.array_equal(getattr(m, name), getattr(n, name)), name
    long = meta_of([[-1]], [5], [list(range(63, -1, -1)) * 4])      # far longer than its context
    assert long.block_tables_np.tolist() == [[63]] and long.slot_mapping_np.tolist() == [63 * 16 + 5]


def test_refusals_of_a_walk():
    def most(tree, node):
        below = [i for i in range(node + 1, len(tree)) if tree[i] == node]
        return max([len(below) - 1, 0] + [k + most(tree, i) for k, i in enumerate(below)])

    for seed in range(20):
        trees = random_trees(seed, [1 + seed % 7, 0, 30])
        assert build_tree_metadata(trees).max_refusals == max(most(t, 0) for t in trees if t)
    assert build_tree_metadata([list(range(-1, 9)), [-1]]).max_refusals == 0
    assert build_tree_metadata([[-1] + [0] * 9]).max_refusals == 8


def test_rows_entry_names_what_is_wrong():
    L = _lib.lib()

    def rows(parents=(-1, 0, -1), starts=(0, 2, 3), cached=(14, 3), tables=((5, 6), (7, 7)), bs=16, nb=8, words=1, nul=None):
        a = [np.array(x, dtype=np.int32) for x in (parents, starts, cached, tables)]
        t = len(parents)
        out = [np.zeros((t, max(words, 1)), np.uint32), np.zeros(t, np.int64), np.zeros(t, np.int32), np.zeros(t, np.int32)]
        info = np.zeros(4, np.int32)
        ptr = {i: x.ctypes.data for i, x in enumerate(a + out)}
        if nul is not None:
            ptr[nul] = None
        st = L.tb_build_tree_rows(ptr[0], ptr[1], len(starts) - 1, ptr[2], ptr[3], a[3].shape[1], bs, nb, ptr[4], words,
                                  ptr[5], ptr[6], ptr[7], info.ctypes.data)
        return st, info.tolist(), out

    bad, index = _lib.TB_ERR_INVALID_ARG, _lib.TB_ERR_INDEX
    st, info, (mask, positions, seq, slots) = rows()
    assert st == _lib.TB_OK and info == [0, 16, 0, 0]
    assert mask[:, 0].tolist() == [1, 3, 1] and positions.tolist() == [14, 15, 3] and seq.tolist() == [0, 0, 1]
    assert slots.tolist() == [5 * 16 + 14, 5 * 16 + 15, 7 * 16 + 3]
    assert rows(nul=2)[1:][0] == [0, 2, 0, 0]                        # the trees alone: depths
    for parents, at in (((-1, 1, -1), 1), ((-1, -1, -1), 1), ((0, 0, -1), 0), ((-1, 0, 0), 2), ((-1, -2, -1), 1)):
        st, info, _ = rows(parents=parents)
        assert st == bad and info[2:] == [1, at]
    assert rows(cached=(14, 31), tables=((5,), (7,)))[0] == index
    assert rows(cached=(14, 31), tables=((5,), (7,)))[1][2:] == [2, 1]
    assert rows(tables=((5, 6), (8, 7)))[0] == index and rows(tables=((5, 6), (8, 7)))[1][2:] == [3, 1]
    assert rows(tables=((-1, 6), (7, 7)))[1][2:] == [3, 0]
    assert rows(nb=1 << 28, tables=((5, 6), ((1 << 28) - 1, 7)))[1][2:] == [4, 1]
    assert rows(cached=(14, 15), tables=((5, 6), (5, 7)))[1][2:] == [5, 5]
    assert rows(cached=(14, 16), tables=((5, 6), (5, 7)))[1][2:] == [6, 5]
    assert rows(cached=(16, 0), tables=((5, 5), (7, 7)))[1][2:] == [6, 5]   # a block twice in one table
    for kw in (dict(nul=0), dict(nul=1), dict(nul=3), dict(nul=4), dict(nul=5), dict(nul=6), dict(nul=7), dict(bs=12),
               dict(nb=0), dict(words=0), dict(cached=(-1, 3)), dict(starts=(0, 3, 2)), dict(starts=(1, 2, 3))):
        assert rows(**kw)[0] == bad, kw
    assert rows(parents=range(-1, 32), starts=(0, 33), cached=(0,), tables=((0, 1, 2),), words=1)[0] == bad


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

    def verify(probs=f, stride=100, draft=None, dstride=0, vocab=100, dt=0, tokens=f, seqs=2, width=4, acc=f,
               children=1, ws=f, wsb=1 << 20, arrivals=None, units=0):
        return L.tb_tree_verify(probs, stride, draft, dstride, vocab, dt, tokens, f, f, f, seqs, children, acc, f, f,
                                width, ws, wsb, arrivals, units, None)

    assert verify(stride=99) == bad                    # rows overlap
    assert verify(draft=f, dstride=99) == bad
    assert verify(vocab=0) == bad and verify(dt=3) == bad and verify(width=0) == bad
    assert verify(probs=None) == bad and verify(tokens=None) == bad and verify(acc=None) == bad
    assert verify(children=-1) == bad and verify(ws=None) == bad and verify(ws=ctypes.c_void_p(4100)) == bad
    assert verify(wsb=L.tb_tree_verify_workspace_bytes(2, 100, 4) - 1) == bad
    assert verify(arrivals=f, units=1) == bad                    # fewer counters than sequences
    assert verify(width=MAX_NODES + 1) == unsupported
    assert verify(vocab=1 << 25, stride=1 << 25, wsb=1 << 30) == unsupported
    assert verify(vocab=MAX_VOCAB + 1, stride=1 << 25, wsb=1 << 30) == unsupported
    assert verify(vocab=MAX_VOCAB, stride=1 << 25, ws=None) == bad
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

    def attention(q=f, d=64, bs=16, hq=14, hkv=2, dt=1, qs=896, words=1, work=f, nw=8, blocks=1, split=None, ns=0, slots=0,
                  ws=None, wsb=0, rows=4, rc=None, rs=None, rmax=0, arrivals=None, units=0):
        return L.tb_tree_attention(q, qs, f, 64, f, 896, f, 4, f, f, 2, f, rows, f, words, work, nw, blocks, split, ns,
                                   slots, ws, wsb, arrivals, units, hq, hkv, d, bs, 0.125, dt, f, rc, rs, rmax, None)

    assert attention(d=96) == unsupported
    assert attention(hq=13) == bad and attention(bs=12) == bad and attention(dt=3) == bad and attention(words=0) == bad
    assert attention(q=None) == bad and attention(q=ctypes.c_void_p(4104)) == bad
    assert attention(qs=895) == bad and attention(qs=900) == bad          # rows overlap; rows not 16-byte aligned
    assert attention(blocks=3) == bad and attention(work=None) == bad and attention(work=ctypes.c_void_p(4104)) == bad
    assert attention(ns=1, split=f) == bad                                # split rows without partial slots
    assert attention(ns=1, slots=2) == bad                                # ... without their records
    assert attention(ns=1, slots=2, split=f) == bad                       # ... without a workspace
    assert attention(ns=1, slots=2, split=f, ws=f, wsb=2 * 14 * 66 * 4 - 1) == bad
    assert attention(ns=5, slots=9, split=f, ws=f, wsb=1 << 20) == bad    # more split rows than rows
    assert attention(ns=1, slots=2, split=f, ws=f, wsb=1 << 20, arrivals=f, units=0) == bad
    assert attention(rc=f, rmax=64) == bad and attention(rc=f, rs=f, rmax=0) == bad
    assert attention(rows=0, q=None) == _lib.TB_OK and attention(nw=0) == _lib.TB_OK
    assert L.tb_tree_attention_workspace_bytes(10, 14, 64) == 10 * 14 * 66 * 4


@pytest.mark.parametrize("hq,hkv,d,dtype", [(14, 2, 64, torch.bfloat16), (32, 8, 128, torch.float16), (5, 5, 128, torch.float32),
                                            (33, 1, 64, torch.float32)])
@pytest.mark.parametrize("sizes,cached", [([5], [600]), ([60, 0, 3, 33], [0, 50, 7000, 31]), ([1] * 70, list(range(0, 7000, 100))),
                                          ([1024], [0]), ([0, 0], [4, 0]), ([], [])])
def test_work_covers_every_context_once(hq, hkv, d, dtype, sizes, cached):
    """Every (sequence, kv head, column group) has each chunk of its context in one entry, parts of one length;
    its partial slots are its own; entry g's piece stays on XCD g % 8."""
    parents = [list(range(-1, n - 1)) for n in sizes]
    at, tables = 0, []
    for c, n in zip(cached, sizes):
        k = -(-(c + n) // 16)
        tables.append(list(range(at, at + k)))
        at += k
    m = build_tree_metadata(parents, cached, tables, block_size=16, num_blocks=max(at, 1), num_heads=hq, num_kv_heads=hkv,
                            head_dim=d, dtype=dtype)
    cols, rep = 32 * m.column_blocks, hq // hkv
    assert m.work_np.shape[0] % 8 == 0
    seen, slots, where, units, orders = {}, {}, {}, {}, {}
    for g, (row0, seq, c, n, col0, kvh, chunk0, chunks, slot, once, unit, order) in enumerate(m.work_np.tolist()):
        if n == 0:
            continue
        assert once == (n * rep <= cols)
        assert (row0, c, n) == (m.row_starts_np[seq], cached[seq], sizes[seq]) and chunks > 0
        seen.setdefault((seq, kvh, col0), []).extend(range(chunk0, chunk0 + chunks))
        slots.setdefault(seq, {})[chunk0] = slot
        if slot >= 0:
            assert units.setdefault((seq, kvh, col0), unit) == unit
            orders.setdefault(unit, {})[order & 0xFFFF] = (chunk0, order >> 16)
        assert where.setdefault((seq, kvh, chunk0), g % 8) == g % 8
    want = {(b, h, x): list(range(-(-(cached[b] + n) // 32))) for b, n in enumerate(sizes) for h in range(hkv)
            for x in range(0, n * rep, cols)}
    assert {k: sorted(v) for k, v in seen.items()} == want
    used, records = [], []
    for seq, by in slots.items():
        n, parts = sizes[seq], [by[k] for k in sorted(by)]
        if len(parts) == 1:
            assert parts == [-1]
            continue
        assert parts == [parts[0] + i * n for i in range(len(parts))]
        used += range(parts[0], parts[0] + len(parts) * n)
        records += [[int(m.row_starts_np[seq]) + i, parts[0] + i, len(parts), n] for i in range(n)]
    if m.units:                                  # parts in the order of their chunks, a counter for each unit
        assert sorted(units.values()) == list(range(m.units))
        for by in orders.values():
            assert sorted(by) == list(range(len(by))) and all(n == len(by) for _, n in by.values())
            assert [by[i][0] for i in range(len(by))] == sorted(x for x, _ in by.values())
    assert sorted(used) == list(range(m.partial_slots)) and sorted(m.split_np.tolist()) == sorted(records)


@pytest.mark.parametrize("hq,hkv,d,dt,sizes,cached", [
    (64, 8, 128, 2, [512] * 2, [500000, 499000]), (32, 8, 128, 2, [1024] * 4, [100000, 100001, 99000, 1]),
    (64, 8, 128, 2, [1024] * 8, list(range(30000, 30008))), (40, 40, 128, 2, [773], [98924]),
    (14, 2, 64, 1, [1024] * 64, [1 << 20] * 64), (4, 4, 128, 0, [60], [1 << 24])])
def test_partials_stay_within_their_bound(hq, hkv, d, dt, sizes, cached):
    """Large trees behind long contexts: what a call needs beside the cache does not grow with them."""
    L, counts = _lib.lib(), np.zeros(5, dtype=np.int32)
    c, n = np.array(cached, dtype=np.int32), np.array(sizes, dtype=np.int32)
    assert L.tb_build_tree_work(c.ctypes.data, n.ctypes.data, len(sizes), hq, hkv, d, dt, 256, 8, None, 0, None, 0,
                                counts.ctypes.data) == _lib.TB_OK
    assert L.tb_tree_attention_workspace_bytes(int(counts[2]), hq, d) <= 128 << 20
    assert counts[0] >= 256 or counts[2] > 0               # nor is the chip left empty for it


def test_rows_of_one_head_or_none():
    """A dimension of one entry, and a tensor without any, may hold any stride: torch's own results do."""
    from tinybatch_amd.ops import _rows_view
    empty = torch.empty(0, 1, 128) * 0.5
    assert empty.stride(1) == 0 and _rows_view("q", empty, 1, 128) == 128
    one = torch.zeros(5 * 200).as_strided((5, 1, 128), (200, 0, 1))
    assert _rows_view("q", one, 1, 128) == 200
    for bad in (torch.zeros(5, 128, 2)[..., 0].view(5, 1, 128), torch.zeros(5, 3, 128)[:, ::2]):
        with pytest.raises(ValueError, match="contiguous"):
            _rows_view("q", bad, bad.shape[1], 128)
