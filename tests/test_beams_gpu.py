"""Beam search's operators (tinybatch_amd/device_tables.py, beams.py) on the GPU against their plain forms
(oracle/beams.py). Steps and reorderings are whole numbers and moved rows: equal, bit for bit.

Selection's scores: the result is rounded to fp32 (2^-24 |c|). A term of the sum e^(x - r) has its argument rounded and log2(e) in
it, 2^-24 |x - r| each at most, and its value by 2 of an exponential's steps, as has the reference's; 16 terms are added in fp32.
|x - r| is at most (m - x) + 4, and the mean of m - x under the terms is at most log V <= 21 (the terms' entropy): the sum, and
with it its logarithm, is off by (2 (21 + 4) + 4 + 16) 2^-24 < 106 2^-24 at most; everything else is in 64 bits.

Attention's tolerance counts roundings, with h half a step of the element type: the output is off by h |out|; the weights that
multiply V are rounded to the type (h each) and so is their sum (h): 2 h sum p|v|; a score, an fp32 sum of d products,
by (d + 4) 2^-24 sum|q k| (its weight by that relatively, and the sum of weights again), and the sums over
the context by 2^-24 a term."""
import threading

import numpy as np
import pytest
import torch

from oracle import beams as oracle
from test_device_tables import random_state
from tinybatch_amd import BeamPlan, DeviceTables, beam_attention, build_device_step, ops, reorder_beams, select_beams
from tinybatch_amd.block_manager import OutOfBlocks
from tinybatch_amd.metadata import build_step_metadata

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
TYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def check_attention(got, q, pool, tables, lens, heads, scale=None):
    d = pool.shape[-1]
    out, weight, spread = oracle.attention(q.cpu().double().numpy(), pool.cpu().double().numpy(), tables, lens, heads, scale)
    h = HALF[pool.dtype]
    exact = 2 * ((d + 4) * 2.0 ** -24 * spread[:, :, None] + (max(lens, default=0) + 64) * 2.0 ** -24)
    tol = h * np.abs(out) + (2 * h + exact) * weight + 1e-30
    off = np.abs(got.cpu().double().numpy().reshape(out.shape) - out)
    assert np.isfinite(off).all() and (off <= tol).all(), (off / tol).max()


def upload(s: oracle.State, max_blocks=None, held=()):
    width = max([len(t) for t in s.tables] + [1]) if max_blocks is None else max_blocks
    return DeviceTables.from_lists(s.tables, s.lens, s.free, max_blocks=width, block_size=s.bs, num_blocks=s.nb,
                                   group_size=s.beams, device=DEV, held=held)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def check_state(t: DeviceTables, s: oracle.State, lens=None, num_free=None):
    assert (t.context_lens if lens is None else lens).tolist() == s.lens
    n = int((t.num_free if num_free is None else num_free).item())
    assert t.free_blocks[:n].tolist() == s.free
    assert t.ref_counts.tolist() == s.refs
    got = t.block_tables.tolist()
    for row, want in zip(got, s.tables):
        assert row[:len(want)] == want


# ---- steps ------------------------------------------------------------------------
@pytest.mark.parametrize("rows", [1, 2, 63, 256, 257, 1024, 1025, 2600])
@pytest.mark.parametrize("bs,P,group", [(16, 64, 1), (1, 64, 3), (32, 256, 2)])
def test_step_of_many_rows(rows, bs, P, group):
    s = random_state(rows + bs, rows, 1, bs, 300 if rows < 300 else 40, spare=12 * rows + 60)
    g = np.random.default_rng(rows)
    new = [int(x) for x in g.choice([0, 1, 1, 1, 2, 7], rows)]
    new[rows // 2] += 50
    after, starts, positions, slots, ctx = oracle.step(s, new)
    t = upload(s, max_blocks=max(len(x) for x in after.tables) + 1)
    step = t.new_step(max_tokens=sum(new) + 5, partition_tokens=P, rows_per_item=group)
    for _ in range(2):                             # a step may be built again
        build_device_step(t, i32(new), step)
        check_state(t, after, step.context_lens, step.num_free)
        assert t.context_lens.tolist() == s.lens
        n = sum(new)
        assert step.query_start_loc.tolist() == starts
        assert step.positions.tolist() == positions + [0] * 5
        assert step.slot_mapping.tolist() == slots + [-1] * 5
        assert step.row_ctx.tolist() == ctx + [0] * 5
    live = [b for b in range(rows) if new[b]]
    meta = build_step_metadata(positions, [(starts[b], starts[b + 1]) for b in live], [after.tables[b] for b in live],
                               [after.lens[b] for b in live], block_size=bs, num_blocks=s.nb, partition_tokens=P,
                               rows_per_item=group)
    items, split, _, parts = step.counts.tolist()
    assert (items, split, parts) == (meta.num_work_items, meta.num_split_rows, meta.total_partitions)
    want = meta.work_np.copy()
    want[:, 1] = np.asarray(live)[want[:, 1]]      # the host's step leaves rows without tokens out
    assert sorted(step.work_items[:items].tolist()) == sorted(want.tolist())
    assert step.row_part_offsets.tolist() == meta.row_part_off_np.tolist() + [parts] * 5
    assert step.split_rows[:split].tolist() == meta.split_rows_np[:split].tolist()
    assert not step.work_items[items:].any() and not step.split_rows[split:].any()
    t.take(step)
    check_state(t, after)
    t.check()


@pytest.mark.parametrize("padded", [1, 3])
@pytest.mark.parametrize("rows", [5, 1200])
def test_step_of_padded_rows(rows, padded):
    s = random_state(rows, rows, 1, 8, 60, spare=rows + 40)
    g = np.random.default_rng(rows)
    new = [int(x) for x in g.integers(0, padded + 1, rows)]
    after, starts, positions, slots, ctx = oracle.step(s, new, padded)
    t = upload(s, max_blocks=max(len(x) for x in after.tables) + 3)
    step = t.new_step(padded=padded, partition_tokens=16)
    build_device_step(t, i32(new), step)
    check_state(t, after, step.context_lens, step.num_free)
    assert step.query_start_loc.tolist() == starts and step.positions.tolist() == positions
    assert step.slot_mapping.tolist() == slots and step.row_ctx.tolist() == ctx
    parts = [-(-c // 16) for c in ctx]
    assert step.row_part_offsets.tolist() == [0] + np.cumsum(parts).tolist()
    assert step.work_items[:sum(parts)].tolist() == [[r, r // padded, p, c] for r, c in enumerate(ctx)
                                                     for p in range(-(-c // 16))]


@pytest.mark.parametrize("rows", [4, 1500])
@pytest.mark.parametrize("why", ["blocks", "row", "tokens", "length", "cached", "work", "padded"])
def test_steps_that_do_not_fit_are_empty(rows, why):
    s = random_state(3, rows, 1, 16, 50, spare=6 if why == "blocks" else 4 * rows + 30)
    new = [1] * rows
    if why == "blocks":
        new[0] = 16 * 7
    if why == "length":
        new[-1] = -1
    after_blocks = max(len(t) for t in s.tables)
    t = upload(s, max_blocks=after_blocks if why == "row" else after_blocks + 20)
    if why == "row":
        new[1] = 16 * after_blocks + 1
    if why == "cached":
        t.context_lens[1] = -3
        s.lens[1] = -3
    step = (t.new_step(padded=1) if why == "padded" else
            t.new_step(max_tokens=rows - 1 if why == "tokens" else sum(max(n, 0) for n in new), partition_tokens=16,
                       max_items=2 if why == "work" else None))
    if why == "padded":
        new[2] = 2
    build_device_step(t, i32(new), step)
    assert step.context_lens.tolist() == s.lens and step.num_free.tolist() == [len(s.free)]
    if why != "cached":
        check_state(t, s)
    assert not step.row_ctx.any() and not step.positions.any() and (step.slot_mapping == -1).all()
    assert step.query_start_loc.tolist() == (list(range(rows + 1)) if why == "padded" else [0] * (rows + 1))
    if why != "padded":
        assert not step.counts.any() and not step.row_part_offsets.any()
    with pytest.raises({"blocks": OutOfBlocks, "row": IndexError}.get(why, ValueError)):
        t.check()
    t.check()                                      # told once


def test_step_without_rows_or_tokens():
    t = DeviceTables(0, max_blocks=1, block_size=16, num_blocks=4, device=DEV)
    step = t.new_step(max_tokens=3, partition_tokens=64)
    build_device_step(t, i32([]), step)
    assert step.slot_mapping.tolist() == [-1] * 3 and step.counts.tolist() == [0] * 4
    s = random_state(1, 3, 1, 16, 40)
    t = upload(s)
    step = t.new_step(max_tokens=0)
    build_device_step(t, i32([0, 0, 0]), step)
    check_state(t, s, step.context_lens, step.num_free)
    t.check()


@pytest.mark.parametrize("dtype,hq,hkv,d", [(torch.float32, 6, 2, 64), (torch.bfloat16, 14, 2, 64), (torch.float16, 8, 2, 128)])
def test_step_serves_paged_attention(dtype, hq, hkv, d):
    """Append and attention over a step built on the GPU against those of the host's step."""
    s = random_state(7, 9, 1, 16, 700, spare=80)
    new = [1, 0, 5, 1, 20, 1, 1, 3, 1]
    after, starts, positions, slots, ctx = oracle.step(s, new)
    g = torch.Generator().manual_seed(1)
    pool = torch.randn(s.nb, 2, hkv, 16, d, generator=g).to(dtype).to(DEV)
    T = len(slots)
    q, k, v = (torch.randn(T, h, d, generator=g).to(dtype).to(DEV) for h in (hq, hkv, hkv))
    t = upload(s, max_blocks=60)
    step = t.new_step(max_tokens=T + 2, partition_tokens=ops.partition_tokens(dtype, d),
                      rows_per_item=ops.rows_per_item(dtype, hq, hkv))
    build_device_step(t, i32(new), step)
    other = pool.clone()
    pad = lambda x: torch.cat([x, x[:2]])
    ops.kv_append(pool, pad(k), pad(v), step.slot_mapping)
    got = ops.paged_attention(pad(q), pool, step.metadata(t), num_heads=hq)
    live = [b for b in range(9) if new[b]]
    meta = build_step_metadata(positions, [(starts[b], starts[b + 1]) for b in live], [after.tables[b] for b in live],
                               [after.lens[b] for b in live], block_size=16, num_blocks=s.nb,
                               partition_tokens=ops.partition_tokens(dtype, d),
                               rows_per_item=ops.rows_per_item(dtype, hq, hkv)).to(DEV)
    ops.kv_append(other, k, v, meta.slot_mapping)
    want = ops.paged_attention(q, other, meta, num_heads=hq)
    assert torch.equal(pool, other)
    # (fp32 launches take the kernel that suits their number of work items, here the capacity)
    assert dtype == torch.float32 or torch.equal(got[:T], want)
    rows = [b for b in range(9) for _ in range(new[b])]
    check_attention(got[:T], q, pool, [after.tables[b] for b in rows], ctx, hq)


# ---- selection ----------------------------------------------------------------------
def check_select(logits, scores, picks, finished=None, end=-1):
    got = select_beams(logits.to(DEV), scores.to(DEV), num_candidates=picks,
                       finished=None if finished is None else finished.to(DEV), end_token=end)
    c, parents, tokens = oracle.select(logits.double().numpy(), scores.numpy(), picks,
                                       None if finished is None else finished.numpy(), end)
    assert got.parents.tolist() == parents.tolist() and got.tokens.tolist() == tokens.tolist()
    value = got.scores.cpu().double().numpy()
    assert (np.isinf(value) == np.isinf(c)).all() or np.abs(c[np.isinf(value) != np.isinf(c)]).min() > 3.4e38
    both = np.isfinite(value) & np.isfinite(c)
    assert (np.abs(value[both] - c[both]) <= 2.0 ** -24 * np.abs(c[both]) + 106 * 2.0 ** -24).all()
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("G,K,V,M", [(1, 1, 1, 1), (1, 1, 1, 5), (2, 3, 7, 6), (1, 4, 511, 8), (3, 2, 512, 4), (2, 5, 513, 10),
                                     (1, 1, 50257, 128), (5, 4, 32001, 8), (1, 8, 151936, 16), (2, 64, 1000, 128),
                                     (70, 6, 257, 12)])
def test_select(G, K, V, M, dtype):
    g = torch.Generator().manual_seed(G * 1000 + V)
    logits = (torch.randn(G * K, V, generator=g) * 4).to(dtype)
    check_select(logits, torch.randn(G, K, generator=g) * 2 - 10, M)


@pytest.mark.parametrize("dtype", TYPES)
def test_select_ended_and_lost_beams(dtype):
    g = torch.Generator().manual_seed(5)
    logits = (torch.randn(6 * 5, 3001, generator=g) * 4).to(dtype)
    scores = torch.randn(6, 5, generator=g) * 3
    finished = torch.rand(6, 5, generator=g) < 0.4
    finished[0], finished[1] = True, False
    scores[2, 1:], scores[3], scores[4, 0] = -float("inf"), -float("inf"), float("nan")
    finished[2, 2], finished[3, 1], finished[4, 0] = True, True, True
    got = check_select(logits, scores, 9, finished, 17)
    assert (got.parents[3] == -1).all() and (got.scores[3] == -float("inf")).all()
    assert got.tokens[0, :5].tolist() == [17] * 5 and got.parents[0, 5:].tolist() == [-1] * 4
    check_select(logits, torch.full((6, 5), -float("inf")), 5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [300, 5000, 151936])
def test_select_ties(V, dtype):
    """Equal logits and equal beams: the smaller beam, then the smaller token; -0 is 0."""
    logits = torch.zeros(4, V, dtype=dtype)
    scores = torch.zeros(1, 4)
    got = check_select(logits, scores, 20)
    assert got.parents.tolist() == [[0] * 20] and got.tokens.tolist() == [list(range(20))]
    logits[:, ::2] = -0.0
    check_select(logits, scores, 20)
    g = torch.Generator().manual_seed(V)
    logits[:] = torch.randint(0, 3, (1, V), generator=g).to(dtype)    # beams alike: candidates tie across them
    check_select(logits, scores, 30)
    logits[:, :] = torch.arange(V).to(dtype) / 256                    # rising: many of a 16-bit type's steps tie
    check_select(logits, scores, 50)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [1, 3])
def test_select_rows_of_any_alignment(offset, dtype):
    """Rows inside a wider tensor, from any element on; rows alike give values alike, to the bit."""
    g = torch.Generator().manual_seed(offset)
    wide = torch.full((6, 2000), 1000.0, dtype=dtype, device=DEV)
    logits = (torch.randn(1, 1403, generator=g) * 3).to(dtype).expand(6, 1403)
    wide[:, offset:offset + 1403] = logits.to(DEV)
    scores = torch.zeros(1, 6)
    got = select_beams(wide[:, offset:offset + 1403], scores.to(DEV), num_candidates=24)
    _, parents, tokens = oracle.select(logits.double().numpy(), scores.numpy(), 24)
    assert got.parents.tolist() == parents.tolist() and got.tokens.tolist() == tokens.tolist()


@pytest.mark.parametrize("dtype", TYPES)
def test_select_masked_and_special_logits(dtype):
    inf, nan = float("inf"), float("nan")
    g = torch.Generator().manual_seed(2)
    V = 2100
    x = (torch.randn(9, V, generator=g) * 3).to(dtype)
    x[0] = -inf                                                       # nothing left
    x[1, :V - 1] = -inf                                               # one token left
    x[2] = torch.finfo(dtype).min                                     # masked by the lowest value
    x[3, 5:] = torch.finfo(dtype).min
    x[4, 7] = nan
    x[5] = nan
    x[6, 9], x[6, 700] = inf, inf
    x[7, 0] = torch.finfo(dtype).max
    x[8] = torch.arange(V, dtype=torch.float32).flip(0).mul(-0.01).to(dtype)
    for rows in ([0], [1], [2], [3], [4], [5], [6], [7], [8], list(range(9))):
        check_select(x[rows].clone(), torch.zeros(1, len(rows)), 12)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("few", [-1000.0, "lowest", 60000.0, 3e38])
def test_select_of_few_far_logits(few, dtype):
    """Runs of -inf alone in rows of few logits, which lie far from 0, or on both sides of where the terms change form."""
    few = torch.finfo(dtype).min if few == "lowest" else min(few, torch.finfo(dtype).max)
    x = torch.full((4, 40_000), -float("inf"), dtype=dtype)
    x[:, 39_000], x[:, 39_990] = few, few
    x[1, 7::1000] = 3.0
    x[2, 20_000:20_600] = 65_500.0 + torch.arange(600).to(dtype)
    x[3] = few
    for rows in ([0], [1], [2], [3], [0, 1, 2, 3]):
        check_select(x[rows].clone(), torch.zeros(1, len(rows)), 12)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [5000, 151936])
def test_select_rising_rows(V, dtype):
    """Every tile's largest logit above the last one's: the reference moves again and again, at every size of logits."""
    g = torch.Generator().manual_seed(V)
    x = torch.stack([torch.arange(V) * by for by in (1e-4, 0.01, 0.4, 100.0)]) + torch.randn(4, V, generator=g)
    x = torch.cat([x, -x.flip(1)]).clamp(-60000, 60000).to(dtype)
    for rows in range(8):
        check_select(x[rows:rows + 1], torch.zeros(1, 1), 9)


@pytest.mark.parametrize("K,M", [(64, 128), (48, 96), (64, 9), (9, 64)])
def test_select_of_many_beams(K, M):
    """More candidates than are ranked at once: alike to the bit, alike in fp32 alone, few left, none left."""
    g = torch.Generator().manual_seed(K)
    inf = float("inf")
    check_select(torch.zeros(K, 300), torch.zeros(1, K), M)
    check_select(torch.zeros(K, 300), torch.randint(0, 2, (1, K), generator=g) * -1.0, M)
    x = torch.randn(K, 700, generator=g)
    check_select(x, torch.full((1, K), -3e9), M)                      # fp32 scores of steps of 256
    check_select(x, -3e9 - 256.0 * torch.randint(0, 3, (1, K), generator=g), M)
    check_select(x, torch.randn(1, K, generator=g) * 1e-3 - 4.0, M)
    masked = torch.full((K, 300), -inf)
    masked[3, 5], masked[7, 200:203] = 1.0, 0.5
    check_select(masked, torch.zeros(1, K), M)
    check_select(x, torch.full((1, K), -inf), M)
    lowest = torch.full((K, 300), torch.finfo(torch.float32).min)     # values below fp32's range count
    lowest[:, 0] = torch.finfo(torch.float32).max
    check_select(lowest, torch.zeros(1, K), M)
    ended = torch.rand(1, K, generator=g) < 0.7
    check_select(x, torch.randn(1, K, generator=g) - 5.0, M, ended, 3)


@pytest.mark.parametrize("dtype", TYPES)
def test_select_long_rows_of_small_terms(dtype):
    """A flat row of many tokens: the sum's terms are as good as equal, nothing of it is lost."""
    x = torch.full((2, 1_000_003), -5.0, dtype=dtype)
    x[0, 999_999] = 3.0
    check_select(x, torch.zeros(1, 2), 3)


def replayed(run, outputs, between=lambda: None, inputs=()):
    """The outputs of `run` captured into a graph and replayed three times, other work between the replays; before each one
    the inputs' copies are what they were."""
    keep = [x.clone() for x in inputs]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run()                                      # what is allocated once is allocated
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        held = run()
    got = []
    for _ in range(3):
        for x, y in zip(inputs, keep):
            x.copy_(y)
        between()
        graph.replay()
        torch.cuda.synchronize()
        got.append([x.clone() for x in outputs(held)])
        torch.randn(1 << 16, device=DEV).sum().item()
    for x, y in zip(inputs, keep):
        x.copy_(y)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("G,K,V,M", [(3, 4, 32001, 8), (1, 48, 5000, 96), (5, 2, 300, 4)])
def test_select_captured(G, K, V, M, dtype):
    """Captured and replayed beside eager calls: the same values, to the bit."""
    g = torch.Generator().manual_seed(V)
    logits = (torch.randn(G * K, V, generator=g) * 3).to(dtype).to(DEV)
    scores = (torch.randn(G, K, generator=g) - 5).to(DEV)
    finished = (torch.rand(G, K, generator=g) < 0.3).to(DEV)
    call = lambda: select_beams(logits, scores, num_candidates=M, finished=finished, end_token=3)
    want = call()
    for got in replayed(call, list, between=call):
        assert all(torch.equal(x, y) for x, y in zip(got, want))


# ---- reordering ---------------------------------------------------------------------
def random_parents(g, groups, K):
    return [int(min(K - 1, K * g.random() ** 1.5)) if g.random() < 0.95 else -1 for _ in range(groups * K)]


def check_reorder(s, parents, storage, t, step=None):
    after, copies = oracle.reorder(s, parents)
    want = storage.clone()
    for src, dst, n in copies:
        want[:, dst, :, :, :n] = storage[:, src, :, :, :n]
    reorder_beams(storage, t, i32(parents).view(-1, s.beams), step)
    check_state(t, after)
    assert t.shared_blocks.tolist() == after.shared()
    assert torch.equal(storage.view(torch.uint8), want.view(torch.uint8))
    for r, row in enumerate(t.block_tables.tolist()):
        g0 = r // s.beams * s.beams
        width = max(len(x) for x in s.tables[g0:g0 + s.beams])
        assert row[len(after.tables[r]):width] == [-1] * (width - len(after.tables[r]))
    return after


@pytest.mark.parametrize("dtype,hkv,d", [(torch.bfloat16, 2, 64), (torch.float32, 1, 128), (torch.float16, 3, 8)])
@pytest.mark.parametrize("groups,K,bs,longest", [(1, 1, 16, 40), (3, 4, 16, 200), (2, 8, 1, 30), (40, 5, 4, 60), (2, 64, 8, 100),
                                                 (5, 3, 2, 900)])
def test_reorder(groups, K, bs, longest, dtype, hkv, d):
    """Steps and selections in turn: every state, count and row as the plain form's."""
    s = random_state(groups + K, groups, K, bs, longest, spare=8 * groups * K + 8, held=2)
    g = np.random.default_rng(K)
    held = s.tables[0][:2]
    t = upload(s, max_blocks=max(len(x) for x in s.tables) + 6, held=held)
    storage = torch.randn(3, s.nb, 2, hkv, bs, d, device=DEV).to(dtype)
    step = t.new_step(padded=1)
    for turn in range(4):
        s = check_reorder(s, random_parents(g, groups, K), storage, t)
        new = [int(n > 0 and g.random() < 0.9) for n in s.lens]
        after, *_ = oracle.step(s, new)
        build_device_step(t, i32(new), step)
        s = after
        s = check_reorder(s, random_parents(g, groups, K), storage, t, step)
    t.check()


def test_reorder_from_one_prompt():
    """The first selection: one row has the prompt, the others nothing."""
    s = oracle.State([[4, 2, 7]] + [[]] * 4, [37, 0, 0, 0, 0], [0, 1, 3, 5, 6, 8], 9, 16, 5)
    t = upload(s, max_blocks=4)
    storage = torch.randn(2, 9, 2, 2, 16, 64, device=DEV)
    after = check_reorder(s, [0, 0, 0, 0, 0], storage, t)
    assert after.shared() == [2] and len(after.free) == 2
    after = check_reorder(after, [-1] * 5, storage, t)               # the request has ended: all its blocks are free
    assert len(after.free) == 9 and after.lens == [0] * 5


def test_reorder_open_block_that_someone_else_holds():
    """Two requests on one prompt's blocks, its last one not full: every child copies it."""
    s = oracle.State([[3, 1], [], [3, 1], []], [20, 0, 20, 0], [0, 2, 4, 5, 6], 8, 16, 2)
    t = upload(s)
    storage = torch.randn(1, 8, 2, 1, 16, 64, device=DEV)
    after = check_reorder(s, [0, 0, 0, -1], storage, t)
    assert after.free[-1] == 1 and after.refs[3] == 3


@pytest.mark.parametrize("groups,K,shared", [(3, 2, 5), (40, 8, 3), (70, 8, 40), (300, 2, 2)])
def test_reorder_many_requests_on_one_prompt(groups, K, shared):
    """Blocks that all requests hold are let go of by all at once: in few and in many lists."""
    tables = [list(range(shared)) + [shared + 3 * r + j for j in range(3)] for r in range(groups * K)]
    nb = shared + 3 * groups * K + 5
    s = oracle.State(tables, [16 * (shared + 2) + 1 + r % 16 for r in range(groups * K)], [nb - 1, nb - 2], nb, 16, K)
    t = upload(s)
    storage = torch.randn(1, nb, 2, 1, 16, 8, device=DEV)
    s = check_reorder(s, [0 if r % K else -1 for r in range(groups * K)][::-1] if groups < 5 else [-1] * (groups * K), storage, t)
    check_reorder(s, [-1] * (groups * K), storage, t)


def test_reorder_blocks_that_several_requests_let_go_of():
    tables = [[5, 6, 7], [5, 6, 8], [5, 6, 9], [5, 10, 11]]
    s = oracle.State(tables, [48, 48, 48, 48], [0, 1], 12, 16, 2)
    t = upload(s)
    storage = torch.randn(1, 12, 2, 1, 16, 64, device=DEV)
    after = check_reorder(s, [-1, -1, -1, -1], storage, t)
    assert after.free == [0, 1, 5, 6, 7, 8, 10, 9, 11]               # (request, column, row)


@pytest.mark.parametrize("why", ["blocks", "parent", "low"])
def test_reorderings_that_do_not_fit_change_nothing(why):
    s = random_state(4, 2, 4, 16, 60, spare=1)
    s.lens = [n + (n % 16 == 0) if n else n for n in s.lens]
    s = oracle.State([t + [s.free[0]] * (len(t) < -(-n // 16)) for t, n in zip(s.tables, s.lens)], s.lens, [], s.nb, 16, 4)
    t = upload(s)
    storage = torch.randn(2, s.nb, 2, 2, 16, 64, device=DEV)
    keep = [x.clone() for x in (storage, t.block_tables, t.context_lens, t.ref_counts, t.free_blocks, t.num_free)]
    bad = {"blocks": [0, 0, 0, 0], "parent": [0, 1, 2, 4], "low": [-2, 1, 2, 3]}[why]
    reorder_beams(storage, t, i32([bad, bad]))
    for x, y in zip((storage, t.block_tables, t.context_lens, t.ref_counts, t.free_blocks, t.num_free), keep):
        assert torch.equal(x, y)
    with pytest.raises(OutOfBlocks if why == "blocks" else IndexError):
        t.check()


@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 31 - 16, 16 * 9 + 1, -1, -2 ** 31])
def test_reorder_lengths_that_no_table_holds(length):
    s = random_state(2, 2, 3, 16, 90, spare=9)
    t = upload(s, max_blocks=9)
    storage = torch.randn(1, s.nb, 2, 1, 16, 64, device=DEV)
    step = t.new_step(padded=1)
    t.take(build_device_step(t, i32([0] * 6), step))
    step.context_lens[4] = length
    keep = [x.clone() for x in (storage, t._buffer[:-64])]
    reorder_beams(storage, t, i32([[0, 1, 2], [1, 1, 1]]), step)
    assert torch.equal(storage, keep[0]) and torch.equal(t._buffer[:-64], keep[1])
    with pytest.raises(ValueError):
        t.check()


@pytest.mark.parametrize("groups,K", [(130, 8), (17, 64), (1100, 1)])
def test_reorder_and_attention_of_many_rows(groups, K):
    """More rows than a workgroup has threads."""
    s = random_state(groups, groups, K, 16, 40, spare=2 * groups * K)
    g = np.random.default_rng(K)
    t = upload(s, max_blocks=max(len(x) for x in s.tables) + 1)
    storage = torch.randn(1, s.nb, 2, 1, 16, 64, device=DEV, dtype=torch.bfloat16)
    s = check_reorder(s, random_parents(g, groups, K), storage, t)
    q = torch.randn(groups * K, 2, 64).bfloat16()
    plan = BeamPlan(t, num_heads=2, num_kv_heads=1, head_dim=64, dtype=torch.bfloat16).build()
    check_attention(beam_attention(q.to(DEV), storage[0], plan), q, storage[0].cpu(), s.tables, s.lens, 2)


def test_reorder_the_tables_alone():
    s = random_state(9, 3, 4, 16, 100, spare=12)
    t = upload(s)
    g = np.random.default_rng(1)
    parents = random_parents(g, 3, 4)
    after, _ = oracle.reorder(s, parents)
    reorder_beams(None, t, i32(parents).view(3, 4))
    check_state(t, after)


# ---- attention ------------------------------------------------------------------------
def attend(s, hq, hkv, d, dtype, seed=1, magnitude=1.0, ctx=None, scale=None, spare_value=float("nan"), q=None):
    """Attention over a plain state's rows; every slot that no row sees holds NaN."""
    g = torch.Generator().manual_seed(seed)
    ctx = s.lens if ctx is None else ctx
    pool = torch.full((s.nb, 2, hkv, s.bs, d), spare_value, dtype=dtype)
    for t, n in zip(s.tables, ctx):
        for j in range(-(-n // s.bs)):
            rows = min(s.bs, n - s.bs * j)
            pool[t[j], :, :, :rows] = torch.randn(2, hkv, rows, d, generator=g).to(dtype)
    if q is None:
        q = (torch.randn(len(ctx), hq, d, generator=g) * magnitude).to(dtype)
    t = upload(s)
    plan = BeamPlan(t, num_heads=hq, num_kv_heads=hkv, head_dim=d, dtype=dtype).build(i32(ctx))
    dev = pool.to(DEV)
    got = beam_attention(q.to(DEV), dev, plan, scale=scale)
    check_attention(got, q, pool, s.tables, ctx, hq, scale)
    return got, q, dev, plan


GEOMETRIES = [(14, 2, 64), (32, 8, 128), (4, 4, 64), (12, 1, 128), (5, 5, 128), (33, 1, 64), (70, 1, 128)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hkv,d", GEOMETRIES)
@pytest.mark.parametrize("groups,K", [(5, 1), (4, 3), (3, 8), (1, 24)])
def test_attention(groups, K, hq, hkv, d, dtype):
    attend(random_state(groups * K, groups, K, 16, 400), hq, hkv, d, dtype)


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 64)])
@pytest.mark.parametrize("bs", [16, 32, 128])
def test_attention_block_sizes(bs, dtype, d):
    attend(random_state(bs, 4, 4, bs, 500), 6, 2, d, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (8, 2, 128)])
def test_attention_around_its_chunks(hq, hkv, d, dtype):
    """Contexts that end one position before, on and behind multiples of 16, 64 and 128."""
    lens = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 191, 255, 256, 257, 320]
    at, tables = 0, []
    for n in lens:
        tables.append(list(range(at, at + -(-n // 16))))
        at += len(tables[-1])
    attend(oracle.State(tables, lens, [], at + 1, 16, 1), hq, hkv, d, dtype)
    for K in (2, 5):                               # the same with shared blocks in front
        shared = list(range(at, at + 9))
        rows = [shared + t for t in tables[:10]]
        attend(oracle.State(rows, [144 + n for n in lens[:10]], [], at + 9, 16, K), hq, hkv, d, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_of_long_contexts(dtype):
    """Few rows: the contexts are cut over workgroups and joined."""
    s = random_state(3, 1, 4, 16, 1)
    for K, hq, hkv, d, n in ((4, 14, 2, 64, 9001), (1, 4, 2, 128, 7003), (16, 8, 1, 64, 5000)):
        shared = list(range(n // 16))
        own = [[n // 16 + 20 * k + j for j in range(20)] for k in range(K)]
        lens = [n // 16 * 16 + 37 * (k % 8) + 1 for k in range(K)]
        attend(oracle.State([shared + o for o in own], lens, [], n // 16 + 20 * K, 16, K), hq, hkv, d, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_rows_that_see_nothing(dtype):
    """Ended beams (nothing seen) among live ones, a request without any, a row's own table never read then; their
    q may hold anything."""
    s = random_state(6, 5, 4, 16, 200)
    ctx = list(s.lens)
    for r in (0, 3, 5, 6, 8, 9, 10, 11, 18):
        ctx[r] = 0
    q = torch.randn(20, 14, 64).to(dtype)
    got, *_ = attend(s, 14, 2, 64, dtype, ctx=ctx, q=q)
    assert not got[[r for r in range(20) if ctx[r] == 0]].any()
    q = torch.where(torch.tensor(ctx)[:, None, None] > 0, q, float("nan"))
    t = upload(s)
    plan = BeamPlan(t, num_heads=14, num_kv_heads=2, head_dim=64, dtype=dtype).build(i32(ctx))
    pool = torch.randn(s.nb, 2, 2, 16, 64).to(dtype).to(DEV)
    got = beam_attention(q.to(DEV), pool, plan)
    assert torch.isfinite(got).all() and not got[[r for r in range(20) if ctx[r] == 0]].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [0.0, -0.5, 3.0])
def test_attention_scales_and_large_scores(dtype, scale):
    attend(random_state(8, 3, 4, 16, 300), 8, 2, 64, dtype, scale=scale)
    attend(random_state(9, 3, 4, 16, 300), 8, 2, 128, dtype, magnitude=6.0)


def test_attention_into_strided_rows():
    s = random_state(12, 3, 4, 16, 300)
    got, q, pool, plan = attend(s, 14, 2, 64, torch.bfloat16)
    wide = torch.full((12, 2 * 14 * 64), 7.0, dtype=torch.bfloat16, device=DEV)
    wide[:, :896] = q.to(DEV).view(12, -1)
    out = torch.full((12, 1000), 7.0, dtype=torch.bfloat16, device=DEV)
    beam_attention(wide[:, :896], pool, plan, out=out[:, 8:904])
    assert torch.equal(out[:, 8:904], got) and (out[:, :8] == 7).all() and (out[:, 904:] == 7).all()


@pytest.mark.parametrize("seed", range(40))
def test_attention_of_random_states(seed):
    g = np.random.default_rng(500 + seed)
    dtype, d = TYPES[seed % 3], (64, 128)[seed // 3 % 2]
    hkv, rep, K = int(g.integers(1, 4)), int(g.choice([1, 2, 3, 5, 7, 8, 12, 33])), int(g.choice([1, 2, 3, 4, 8, 13]))
    s = random_state(seed, int(g.integers(1, 7)), K, int(g.choice([16, 32, 64])), int(g.choice([20, 200, 3000])))
    attend(s, hkv * rep, hkv, d, dtype, seed=seed)


# ---- large offsets, graphs, streams, threads -------------------------------------------
def test_blocks_behind_the_first_4_gb():
    """The same rows in the last blocks of a pool of 4.8 GB a layer as in a small one: copies, appended rows, attention."""
    s = random_state(31, 2, 4, 16, 300, spare=16)
    nb, far = s.nb, 300_000
    move = lambda ids: [far - 1 - b for b in ids]
    small = torch.randn(1, nb, 2, 2, 16, 64, device=DEV)
    big = torch.zeros(1, far, 2, 2, 16, 64, device=DEV)
    big[0, far - nb:] = small[0].flip(0)
    q, k, v = (torch.randn(8, h, 64, device=DEV) for h in (4, 2, 2))
    outs = []
    for storage, tables, free, blocks in ((small, s.tables, s.free, nb), (big, map(move, s.tables), move(s.free), far)):
        t = DeviceTables.from_lists(list(tables), s.lens, free, max_blocks=24, block_size=16, num_blocks=blocks, group_size=4, device=DEV)
        reorder_beams(storage, t, i32([[1, 1, 0, 3], [2, 2, 2, 2]]))
        step = build_device_step(t, i32([1] * 8), t.new_step(padded=1))
        ops.kv_append(storage[0], k, v, step.slot_mapping)
        plan = BeamPlan(t, num_heads=4, num_kv_heads=2, head_dim=64, dtype=torch.float32).build(step.row_ctx)
        outs.append(beam_attention(q, storage[0], plan))
        t.check()
    assert torch.equal(*outs) and torch.equal(big[0, far - nb:].flip(0), small[0]) and not big[0, :far - nb].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_select_rows_far_apart(dtype):
    logits = (torch.randn(6, 5000, device=DEV) * 3).to(dtype)
    stride = (5 << 30) // logits.element_size() // 5
    wide = torch.empty(5 * stride + 5000, dtype=dtype, device=DEV).as_strided((6, 5000), (stride, 1))
    wide.copy_(logits)
    scores = torch.randn(2, 3, device=DEV)
    for x, y in zip(select_beams(wide, scores, num_candidates=7), select_beams(logits, scores, num_candidates=7)):
        assert torch.equal(x, y)


class Loop:
    """A search's step on its own state: run() it, or reset() and run() again."""

    def __init__(self, seed, groups=3, K=4, dtype=torch.bfloat16):
        g = torch.Generator().manual_seed(seed)
        self.s = s = random_state(seed, groups, K, 16, 500, spare=3 * groups * K)
        R, d = groups * K, 64
        self.t = upload(s, max_blocks=max(len(x) for x in s.tables) + 2)
        self.storage = torch.randn(2, s.nb, 2, 2, 16, d, generator=g).to(dtype).to(DEV)
        self.q, self.k, self.v = (torch.randn(R, h, d, generator=g).to(dtype).to(DEV) for h in (6, 2, 2))
        self.logits = torch.randn(R, 20011, generator=g).to(dtype).to(DEV)
        self.scores, self.new = (torch.randn(groups, K, generator=g) - 9).to(DEV), i32([1] * R)
        self.step = self.t.new_step(padded=1)
        self.plan = BeamPlan(self.t, num_heads=6, num_kv_heads=2, head_dim=d, dtype=dtype)
        self.state = [self.t._buffer, self.storage]
        self.start = [x.clone() for x in self.state]

    def reset(self):
        for x, y in zip(self.state, self.start):
            x.copy_(y)

    def run(self):
        build_device_step(self.t, self.new, self.step)
        self.plan.build(self.step.row_ctx)
        outs = []
        for pool in self.storage:
            ops.kv_append(pool, self.k, self.v, self.step.slot_mapping)
            outs.append(beam_attention(self.q, pool, self.plan))
        choice = select_beams(self.logits, self.scores)
        reorder_beams(self.storage, self.t, choice.parents, self.step)
        return [*outs, *choice]

    def results(self, outs):
        return [x.clone() for x in [*outs, *self.state]]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b, strict=True))


def test_a_whole_step_captured():
    """Two captured steps, replayed in turn beside eager steps of a third state: each as it runs by itself."""
    loops = [Loop(1), Loop(2, 5, 2), Loop(3, 1, 9)]
    want = []
    for x in loops:
        outs = x.run()
        want.append(x.results(outs))
        x.reset()
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graphs = []
    for x in loops[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs = x.run()
        graphs.append((graph, outs))
    for _ in range(3):
        for x in loops:
            x.reset()
        for graph, _ in graphs:
            graph.replay()
        third = loops[2].run()
        torch.cuda.synchronize()
        for x, outs, w in zip(loops, [graphs[0][1], graphs[1][1], third], want):
            assert same(x.results(outs), w)
        torch.randn(1 << 16, device=DEV).sum().item()
    for x in loops:
        x.t.check()


def test_steps_on_several_streams_and_threads():
    """Three threads, two of them on one stream: every state goes its own way."""
    loops = [Loop(4), Loop(5, 5, 2), Loop(6, 1, 9)]
    want = []
    for x in loops:
        want.append([x.results(x.run()) for _ in range(3)])
        x.reset()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    failed = []

    def work(x, stream, w):
        try:
            with torch.cuda.stream(stream):
                for _ in range(10):
                    got = [x.results(x.run()) for _ in range(3)]
                    x.reset()
                    stream.synchronize()
                    assert all(same(a, b) for a, b in zip(got, w))
        except BaseException as e:
            failed.append(e)

    threads = [threading.Thread(target=work, args=(x, streams[i % 2], w)) for i, (x, w) in enumerate(zip(loops, want))]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    assert not failed, failed[0]


# ---- refusals -------------------------------------------------------------------------
def test_refusals():
    logits, scores = torch.zeros(4, 10, device=DEV), torch.zeros(2, 2, device=DEV)
    for bad in (lambda: select_beams(logits.cpu(), scores), ):
        with pytest.raises(RuntimeError, match="GPU"):
            bad()
    for bad in (lambda: select_beams(logits.long(), scores), lambda: select_beams(logits, scores.double()),
                lambda: select_beams(logits, scores.cpu()),
                lambda: select_beams(logits, scores, finished=torch.zeros(2, 2, device=DEV), end_token=0)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: select_beams(logits[:3], scores), lambda: select_beams(logits.t(), scores),
                lambda: select_beams(logits[:1].expand(4, 10), scores), lambda: select_beams(logits, scores[0]),
                lambda: select_beams(logits, scores, num_candidates=0), lambda: select_beams(logits, scores, num_candidates=129),
                lambda: select_beams(logits, torch.zeros(4, 65, device=DEV)),
                lambda: select_beams(logits, scores, finished=torch.zeros(2, 2, dtype=torch.bool, device=DEV), end_token=10),
                lambda: select_beams(logits, scores, finished=torch.zeros(2, 2, dtype=torch.bool, device=DEV))):
        with pytest.raises(ValueError):
            bad()
    s = random_state(1, 2, 2, 16, 40)
    t = upload(s)
    storage = torch.zeros(2, s.nb, 2, 1, 16, 64, device=DEV)
    parents = i32([[0, 1], [0, 1]])
    for bad in (lambda: reorder_beams(storage, t, parents.long()), lambda: reorder_beams(storage, t, parents[:1]),
                lambda: reorder_beams(storage, t, parents.cpu()), lambda: reorder_beams(storage.long(), t, parents)):
        with pytest.raises(TypeError):
            bad()
    other = upload(random_state(1, 3, 2, 16, 40))
    for bad in (lambda: reorder_beams(storage[0], t, parents), lambda: reorder_beams(storage[:, 1:], t, parents),
                lambda: reorder_beams(storage[:, 1:].contiguous(), t, parents),
                lambda: reorder_beams(torch.zeros(1, s.nb, 2, 1, 16, 6, device=DEV), t, parents),
                lambda: reorder_beams(storage, t, parents, other.new_step(padded=1))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        build_device_step(t, torch.zeros(4, dtype=torch.int64, device=DEV), t.new_step(padded=1))
    for bad in (lambda: build_device_step(t, i32([1] * 4), other.new_step(padded=1)), lambda: t.new_step(),
                lambda: t.new_step(max_tokens=-1), lambda: t.new_step(max_tokens=5, padded=1), lambda: t.new_step(padded=-1),
                lambda: t.new_step(max_tokens=4, partition_tokens=64, rows_per_item=17),
                lambda: t.new_step(max_tokens=4, partition_tokens=64, max_items=1 << 24),
                lambda: t.new_step(max_tokens=4).metadata(t)):
        with pytest.raises(ValueError):
            bad()


def test_attention_refusals():
    s = random_state(1, 2, 2, 16, 40)
    t = upload(s)
    kw = dict(num_heads=4, num_kv_heads=2, head_dim=64, dtype=torch.float16)
    plan = BeamPlan(t, **kw)
    q, pool = torch.zeros(4, 4, 64, dtype=torch.float16, device=DEV), torch.zeros(s.nb, 2, 2, 16, 64, dtype=torch.float16, device=DEV)
    with pytest.raises(ValueError, match="built"):
        beam_attention(q, pool, plan)
    plan.build()
    for bad in (dict(num_heads=5), dict(head_dim=96), dict(num_kv_heads=0)):
        with pytest.raises(ValueError):
            BeamPlan(t, **{**kw, **bad})
    with pytest.raises(ValueError):
        BeamPlan(upload(random_state(1, 2, 2, 8, 40)), **kw)
    with pytest.raises(TypeError):
        BeamPlan(t, **{**kw, "dtype": torch.int8})
    for bad in (lambda: plan.build(i32([1] * 3)), lambda: plan.build(torch.ones(4, dtype=torch.int32)),
                lambda: beam_attention(q.float(), pool, plan), lambda: beam_attention(q.float(), pool.float(), plan)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: beam_attention(q[:3], pool, plan), lambda: beam_attention(q, pool[:-1], plan),
                lambda: beam_attention(q, pool[:, :, :1].contiguous(), plan), lambda: beam_attention(q[:, :3], pool, plan),
                lambda: beam_attention(q, pool, plan, out=q.float()), lambda: beam_attention(q, pool, plan, out=q[:3]),
                lambda: beam_attention(q.transpose(1, 2), pool, plan)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        beam_attention(q.cpu(), pool, plan)


# ---- rows that were empty --------------------------------------------------------------
def refill(s, t, new, chunk, pool):
    """Steps of up to ``chunk`` new tokens a row until every row has its new[r], each taken; their K/V rows are random."""
    new, d, hkv = list(new), pool.shape[-1], pool.shape[2]
    step = t.new_step(padded=chunk)
    g = torch.Generator().manual_seed(sum(new))
    while any(new):
        part = [min(n, chunk) for n in new]
        s = oracle.step(s, part, chunk)[0]
        build_device_step(t, i32(part), step)
        k, v = (torch.randn(len(new) * chunk, hkv, d, generator=g).to(pool.dtype).to(DEV) for _ in range(2))
        ops.kv_append(pool, k, v, step.slot_mapping)
        yield s, step
        t.take(step)
        new = [n - p for n, p in zip(new, part)]
    t.check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("chunk", [1, 7, 32])
@pytest.mark.parametrize("lens,new", [([37, 0], [0, 32]), ([37, 0], [3, 40]), ([33, 40, 0, 36, 32, 0, 0, 50], [1, 0, 33, 0, 0, 0, 48, 17]),
                                      ([0, 0, 40, 37], [20, 35, 1, 1])])
def test_attention_of_rows_that_were_empty(lens, new, chunk, dtype):
    """A row without positions gets tokens, in blocks of its own: it shares none with its request's other rows, whatever they
    shared before; the request beside it still does."""
    K = 2 if len(lens) < 8 else 4
    tables, at = [], 40
    for r, n in enumerate(lens):                   # two whole blocks in common, the rest a row's own
        whole = [2 * (r // K), 2 * (r // K) + 1][:n // 16]
        own = -(-n // 16) - len(whole)
        tables.append(whole + list(range(at, at + own)))
        at += own
    s = oracle.State(tables, lens, list(range(10, 34)), 64, 16, K)
    t = upload(s, max_blocks=6)
    assert t.shared_blocks.tolist() == s.shared()
    pool = torch.randn(64, 2, 2, 16, 64, device=DEV).to(dtype)
    plan = BeamPlan(t, num_heads=6, num_kv_heads=2, head_dim=64, dtype=dtype)
    q = torch.randn(len(lens), 6, 64).to(dtype)
    for after, step in refill(s, t, new, chunk, pool):
        # before it is taken: over the step's lengths, and over the lengths that are still the state's
        for n, rows in ((after.lens, step.context_lens), (s.lens, None)):
            check_attention(beam_attention(q.to(DEV), pool, plan.build(rows)), q, pool.cpu(), after.tables, n, 6)
        s = after
    check_state(t, s)
    check_attention(beam_attention(q.to(DEV), pool, plan.build()), q, pool.cpu(), s.tables, s.lens, 6)
    assert all(x <= y for x, y in zip(t.shared_blocks.tolist(), s.shared()))
    assert all(t.shared_blocks[g // K] == 2 for g in range(0, len(lens), K) if all(lens[g:g + K]))


def test_steps_keep_what_rows_share():
    """Steps whose new tokens go to rows with positions, steps that do not fit, steps of one row a request: as shared as before."""
    s = oracle.State([[0, 1, 4], [0, 1, 5], [2, 3], []], [37, 40, 32, 0], [10, 11], 16, 16, 2)
    t = upload(s, max_blocks=4)
    assert t.shared_blocks.tolist() == [2, 2]
    step = t.new_step(padded=40)
    build_device_step(t, i32([1, 8, 1, 0]), step)
    assert t.shared_blocks.tolist() == [2, 2]
    build_device_step(t, i32([0, 0, 0, 40]), step)                     # three blocks of two
    assert t.shared_blocks.tolist() == [2, 2] and not step.row_ctx.any()
    with pytest.raises(OutOfBlocks):
        t.check()
    build_device_step(t, i32([0, 0, 0, 20]), step)
    assert t.shared_blocks.tolist() == [2, 0]
    one = DeviceTables.from_lists([[0], []], [16, 0], [3], max_blocks=2, block_size=16, num_blocks=4, device=DEV)
    build_device_step(one, i32([0, 1]), one.new_step(padded=1))
    one.check()
