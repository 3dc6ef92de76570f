"""Steps built from lengths and the beams' states (tinybatch_amd/device_tables.py, beams.py) without a GPU:
the plain forms against the host's own builders, what from_lists refuses, and the C entries' refusals
before any launch."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import beams as oracle
from tinybatch_amd import _lib, build_step_metadata, device_tables
from tinybatch_amd.block_manager import BlockManager


def random_state(seed, groups, beams, bs, longest, spare=8, held=0):
    """A plain state as a search leaves it: prompts' whole blocks shared, the rest a row's own."""
    g = np.random.default_rng(seed)
    prompts = [int(g.integers(0, longest + 1)) for _ in range(groups)]
    made = [[int(g.integers(0, 3 * bs)) if p else 0 for _ in range(beams)] for p in prompts]
    need = [p // bs + sum(-(-(p + m) // bs) - p // bs for m in ms) for p, ms in zip(prompts, made)]
    nb = sum(need) + spare + 1
    ids = g.permutation(nb).tolist()
    tables, lens, at = [], [], 0
    for p, ms in zip(prompts, made):
        whole = ids[at:at + p // bs]
        at += p // bs
        for m in ms:
            mine = -(-(p + m) // bs) - p // bs
            tables.append(whole + ids[at:at + mine])
            lens.append(p + m)
            at += mine
    return oracle.State(tables, lens, ids[at:at + spare], nb, bs, beams, held=tables[0][:held] if tables else ())


@pytest.mark.parametrize("seed", range(6))
def test_plain_step_is_the_hosts_step(seed):
    """The oracle's positions and slots against build_step_metadata, its blocks against BlockManager."""
    s = random_state(seed, 5, 1, 16, 100, spare=60)
    g = np.random.default_rng(seed)
    new = [int(x) for x in g.integers(0, 40, 5)]
    after, starts, positions, slots, ctx = oracle.step(s, new)
    rows = [b for b in range(5) if new[b]]
    meta = build_step_metadata(positions, [(starts[b], starts[b + 1]) for b in rows], [after.tables[b] for b in rows],
                               [after.lens[b] for b in rows], block_size=16, num_blocks=s.nb, partition_tokens=64)
    assert meta.slot_mapping_np.tolist() == slots and meta.row_ctx_np.tolist() == ctx
    bm = BlockManager(s.nb, 16, enable_prefix_caching=False)
    bm.free_ids = list(s.free)
    for b in range(5):
        table = list(s.tables[b])
        for i in range(new[b]):
            bm.append_slot(table, [0] * (s.lens[b] + i))
        assert table == after.tables[b]
    assert bm.free_ids == after.free


@pytest.mark.parametrize("seed", range(20))
def test_plain_reorder_keeps_count(seed):
    """Every block is held as often as it is counted, free or held, and never both; nothing is shared that is written."""
    s = random_state(seed, 3, 4, 4, 20, spare=12, held=2 * (seed % 2))
    g = np.random.default_rng(seed)
    for _ in range(4):
        s, _ = oracle.reorder(s, [int(x) for x in g.integers(-1, 4, 12)])
        held = [0] * s.nb
        for t, n in zip(s.tables, s.lens):
            assert len(t) == -(-n // s.bs)
            for b in t:
                held[b] += 1
            assert n % s.bs == 0 or s.refs[t[-1]] == 1
        extra = [r - h for r, h in zip(s.refs, held)]
        assert min(extra) >= 0 and sum(extra) <= 2 and len(set(s.free)) == len(s.free)
        assert all(s.refs[b] == 0 for b in s.free)
        s, *_ = oracle.step(s, [int(x) for x in g.integers(0, 2, 12)]) if len(s.free) > 12 else (s,)


def arrays(tables, lens, free, max_blocks=4, bs=16, nb=32, group=1, held=()):
    return device_tables._state_arrays(tables, lens, free, max_blocks, bs, nb, group, held)


def test_lists_become_arrays():
    counted, tables, refs, stack, shared = arrays([[3, 4], [3, 5, 9], [], [3]], [20, 33, 0, 16], [7, 8], group=2, held=[3])
    assert counted.tolist() == [20, 33, 0, 16, 2] and stack[:2].tolist() == [7, 8]
    assert tables.tolist() == [[3, 4, -1, -1], [3, 5, 9, -1], [-1] * 4, [3, -1, -1, -1]]
    assert refs[[3, 4, 5, 9, 7]].tolist() == [4, 1, 1, 1, 0] and shared.tolist() == [1, 1]
    # a table that reaches further than its positions keeps the blocks that hold them
    assert arrays([[3, 4, 5]], [16], [])[1].tolist() == [[3, -1, -1, -1]]


@pytest.mark.parametrize("bad,error", [
    (dict(tables=[[1]], lens=[17], free=[]), IndexError),              # a table too short
    (dict(tables=[[1, 2, 3, 4, 5]], lens=[65], free=[]), IndexError),  # more blocks than a row holds
    (dict(tables=[[32]], lens=[1], free=[]), IndexError),              # outside the pool
    (dict(tables=[[-1]], lens=[1], free=[]), IndexError),
    (dict(tables=[[1]], lens=[1], free=[1]), ValueError),              # held and free
    (dict(tables=[[1]], lens=[1], free=[2, 2]), ValueError),
    (dict(tables=[[1]], lens=[1], free=[40]), IndexError),
    (dict(tables=[[1]], lens=[1], free=[2], held=[2]), ValueError),
    (dict(tables=[[1]], lens=[-1], free=[]), ValueError),
    (dict(tables=[[1]], lens=[1, 2], free=[]), ValueError),
    (dict(tables=[[1], [2], [3]], lens=[1, 1, 1], free=[], group=2), ValueError),
    (dict(tables=[[1]], lens=[1], free=[], group=65), ValueError),
    (dict(tables=[[1]], lens=[1], free=[], bs=12), ValueError),
    (dict(tables=[[1]], lens=[1], free=[], nb=1 << 28), ValueError),   # slots past 32 bits
])
def test_lists_that_are_refused(bad, error):
    with pytest.raises(error):
        arrays(**bad)


def test_device_tables_need_a_gpu():
    with pytest.raises(RuntimeError, match="GPU"):
        device_tables.DeviceTables(2, max_blocks=2, block_size=16, num_blocks=4, device="cpu")


F = ctypes.c_void_p(4096)
OTHER = ctypes.c_void_p(8192)


def call(fn, defaults, **kw):
    a = dict(defaults)
    assert set(kw) <= set(a)
    a.update(kw)
    return fn(*a.values())


STEP = dict(tables=F, max_nb=8, cached=F, new=F, rows=4, refs=F, free=F, num_free=F, nb=64, bs=16, pad=0, tokens=32,
            lens=OTHER, num_free_out=OTHER, starts=F, positions=F, slots=F, ctx=F, P=64, group=2, offsets=F, items=F,
            max_items=8, parts=8, split=F, max_split=8, counts=F, status=F, ws=None, ws_bytes=0, stream=None)


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(max_nb=0), dict(nb=0), dict(bs=12), dict(bs=0), dict(nb=1 << 27), dict(max_nb=1 << 27, bs=16),
    dict(tokens=1 << 24), dict(tokens=-1), dict(pad=3), dict(pad=-1), dict(num_free=None), dict(num_free_out=F),
    dict(lens=F), dict(status=None), dict(cached=None), dict(new=None), dict(slots=None), dict(positions=None),
    dict(ctx=None), dict(P=-1), dict(group=0), dict(group=17), dict(offsets=None), dict(counts=None), dict(items=None),
    dict(split=None), dict(items=ctypes.c_void_p(4100)), dict(max_items=1 << 24), dict(parts=-1), dict(starts=None),
    dict(rows=2000, tokens=32), dict(rows=2000, ws=F, ws_bytes=100), dict(free=None), dict(refs=None), dict(tables=None)])
def test_step_refusals(bad):
    assert call(_lib.lib().tb_device_step, STEP, **bad) == _lib.TB_ERR_INVALID_ARG


SELECT = dict(logits=F, stride=1000, vocab=1000, dtype=2, scores=F, finished=None, end=0, rows=8, beams=4, picks=8, out=F,
              parents=F, tokens=F, ws=F, ws_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("bad", [
    dict(logits=None), dict(stride=999), dict(vocab=0), dict(vocab=(1 << 30) + 1), dict(dtype=3), dict(scores=None),
    dict(finished=F, end=-1), dict(finished=F, end=1000), dict(rows=7), dict(rows=65536), dict(beams=0),
    dict(beams=65, rows=65), dict(picks=0), dict(picks=129), dict(out=None), dict(parents=None), dict(tokens=None),
    dict(ws=None), dict(ws_bytes=16), dict(ws=ctypes.c_void_p(4104)), dict(logits=ctypes.c_void_p(4097))])
def test_select_refusals(bad):
    assert call(_lib.lib().tb_beam_select, SELECT, **bad) == _lib.TB_ERR_INVALID_ARG


REORDER = dict(storage=F, layers=2, stride=1 << 20, nb=64, hkv=2, d=64, bs=16, dtype=2, tables=F, max_nb=8, rows=8, beams=4,
               lens_in=F, lens_out=F, refs=F, free=F, num_in=F, num_out=F, shared=F, parents=F, status=F, ws=F,
               ws_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("bad", [
    dict(storage=None), dict(layers=-1), dict(layers=65536), dict(stride=1000), dict(stride=1024), dict(nb=0), dict(hkv=0),
    dict(d=0), dict(bs=12), dict(dtype=5), dict(tables=None), dict(max_nb=0), dict(rows=6), dict(beams=0),
    dict(beams=65, rows=65), dict(lens_in=None), dict(lens_out=None), dict(refs=None), dict(free=None), dict(num_in=None),
    dict(num_out=None), dict(shared=None), dict(parents=None), dict(status=None), dict(ws=None), dict(ws_bytes=64),
    dict(ws=ctypes.c_void_p(4104)), dict(storage=ctypes.c_void_p(4104)), dict(max_nb=1 << 27, rows=4, layers=0)])
def test_reorder_refusals(bad):
    assert call(_lib.lib().tb_beam_reorder, REORDER, **bad) == _lib.TB_ERR_INVALID_ARG


def test_rows_of_no_whole_pieces_are_unsupported_and_no_rows_are_nothing():
    L = _lib.lib()
    assert call(L.tb_beam_reorder, REORDER, d=12) == _lib.TB_ERR_UNSUPPORTED
    assert call(L.tb_beam_reorder, REORDER, rows=0) == _lib.TB_OK
    assert call(L.tb_beam_select, SELECT, rows=0, logits=None) == _lib.TB_OK


PLAN = dict(ctx=F, shared=F, rows=8, beams=4, max_nb=8, hq=4, hkv=2, d=64, bs=16, dtype=2, plan=F, bytes=1 << 20, stream=None)
ATTEND = dict(q=F, qs=256, pool=F, nb=64, out=F, os=256, tables=F, max_nb=8, rows=8, beams=4, hq=4, hkv=2, d=64, bs=16,
              scale=0.125, dtype=2, plan=F, bytes=1 << 20, ws=F, ws_bytes=1 << 28, stream=None)


@pytest.mark.parametrize("bad", [
    dict(rows=7), dict(rows=-4), dict(beams=0), dict(beams=65, rows=65), dict(hq=5), dict(hq=0), dict(hkv=0), dict(dtype=3),
    dict(bs=24), dict(bs=0), dict(max_nb=0), dict(max_nb=1 << 27), dict(plan=None), dict(plan=ctypes.c_void_p(4104)),
    dict(bytes=64)])
def test_plan_and_attention_refusals(bad):
    L = _lib.lib()
    assert call(L.tb_beam_plan, PLAN, **bad) == _lib.TB_ERR_INVALID_ARG
    assert call(L.tb_beam_attention, ATTEND, **bad) == _lib.TB_ERR_INVALID_ARG


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(pool=None), dict(out=None), dict(tables=None), dict(ws=None), dict(qs=255), dict(os=255), dict(qs=260),
    dict(os=260), dict(nb=0), dict(q=ctypes.c_void_p(4104)), dict(out=ctypes.c_void_p(4104)), dict(ws_bytes=1000)])
def test_attention_refusals(bad):
    assert call(_lib.lib().tb_beam_attention, ATTEND, **bad) == _lib.TB_ERR_INVALID_ARG


def test_attention_unsupported_and_empty():
    L = _lib.lib()
    for bad in (dict(d=96), dict(bs=8)):
        assert call(L.tb_beam_plan, PLAN, **bad) == _lib.TB_ERR_UNSUPPORTED
        assert call(L.tb_beam_attention, ATTEND, **bad) == _lib.TB_ERR_UNSUPPORTED
    assert call(L.tb_beam_plan, PLAN, rows=0, ctx=None) == _lib.TB_OK
    assert call(L.tb_beam_attention, ATTEND, rows=0, q=None) == _lib.TB_OK
    assert call(L.tb_beam_plan, PLAN, ctx=None) == _lib.TB_ERR_INVALID_ARG
    assert call(L.tb_beam_plan, PLAN, shared=None) == _lib.TB_ERR_INVALID_ARG


BEAM_STEP = {k: v for name in STEP for k, v in ([(name, STEP[name])] if name != "refs" else
                                               [("shared", F), ("beams", 2), ("refs", F)])}


@pytest.mark.parametrize("bad", [
    dict(beams=0), dict(beams=-1), dict(beams=3), dict(beams=65, rows=65), dict(shared=None), dict(rows=-2), dict(bs=12),
    dict(tokens=1 << 24), dict(num_free_out=F), dict(lens=F), dict(status=None), dict(group=17), dict(rows=2000, tokens=32)])
def test_beam_step_refusals(bad):
    assert call(_lib.lib().tb_beam_step, BEAM_STEP, **bad) == _lib.TB_ERR_INVALID_ARG
