"""The operators of speculative decoding (tinybatch_amd/tree.py) on the GPU against their plain
64-bit forms (oracle/tree.py).

Attention's tolerance counts roundings: with h half a step of the element type, the output is off by
h |out|; the weights that multiply V are rounded to the type (h each) and their sum with them (h),
so 2 h sum p|v|; a score's fp32 sum of d products by (d + 4) 2^-24 sum|q k| (its weight by that
relatively, and the sum of weights again), and the sums over the context by 2^-24 a term. Verification
and commit are exact."""
import threading

import numpy as np
import pytest
import torch

from oracle import tree as oracle
from test_tree_metadata import random_trees
from tinybatch_amd import (PagedKVCache, build_tree_metadata, commit_tree, tree_attention, verify_tree,
                           verify_tree_greedy)
from tinybatch_amd.model import rope_tables
from tinybatch_amd.ops import Rope

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


class Case:
    """A step of trees over a shuffled pool; every slot that no sequence owns holds NaN."""

    def __init__(self, seed, hq, hkv, d, dtype, sizes, cached, bs=16, visible=None, parents=None, magnitude=1.0):
        g = torch.Generator().manual_seed(seed)
        self.hq, self.hkv, self.d, self.dtype, self.bs = hq, hkv, d, dtype, bs
        self.parents = parents or random_trees(seed, sizes)
        self.cached, self.sizes = list(cached), [len(t) for t in self.parents]
        need = [-(-(c + n) // bs) for c, n in zip(self.cached, self.sizes)]
        self.nb = sum(need) + 3
        ids = torch.randperm(self.nb, generator=g).tolist()
        self.tables, at = [], 0
        self.pool = torch.full((self.nb, 2, hkv, bs, d), float("nan"), dtype=dtype)
        for c, n, k in zip(self.cached, self.sizes, need):
            table = ids[at:at + k]
            at += k
            self.tables.append(table)
            pos = torch.arange(c + n)
            t = torch.tensor(table + [0], dtype=torch.int64)
            self.pool[t[pos // bs], :, :, pos % bs] = torch.randn(c + n, 2, hkv, d, generator=g).to(dtype)
        self.q = (torch.randn(sum(self.sizes), hq, d, generator=g) * magnitude).to(dtype)
        self.visible = visible
        self.seen = [oracle.visible(t) if visible is None or visible[b] is None else np.asarray(visible[b])
                     for b, t in enumerate(self.parents)]

    def meta(self):
        return build_tree_metadata(self.parents, self.cached, self.tables, block_size=self.bs, num_blocks=self.nb,
                                   num_heads=self.hq, num_kv_heads=self.hkv, head_dim=self.d, dtype=self.dtype,
                                   visible=self.visible).to(DEV)

    def want(self, q=None, scale=None):
        return oracle.attention(self.q if q is None else q, self.pool, self.seen, self.cached, self.tables, self.hq, scale)

    def check(self, got, q=None, scale=None):
        out, weight, spread = self.want(q, scale)
        h, ctx = HALF[self.dtype], max([c + n for c, n in zip(self.cached, self.sizes)], default=0)
        exact = 2 * ((self.d + 4) * 2.0 ** -24 * spread[:, :, None] + (ctx + 64) * 2.0 ** -24)
        tol = h * out.abs() + (2 * h + exact) * weight + 1e-30
        got = got.cpu().double().view_as(out)
        assert torch.isfinite(got).all()
        bad = (got - out).abs() > tol
        assert not bad.any(), ((got - out).abs() / tol).max()


GEOMETRIES = [(14, 2, 64), (32, 8, 128), (4, 4, 64), (12, 1, 128), (5, 5, 128), (33, 1, 64)]
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hkv,d", GEOMETRIES)
def test_attention_of_ragged_trees(hq, hkv, d, dtype):
    c = Case(1, hq, hkv, d, dtype, [1, 5, 0, 17, 33, 2, 40], [0, 1, 7, 15, 46, 127, 300])
    c.check(tree_attention(c.q.to(DEV), c.pool.to(DEV), c.meta()))


@pytest.mark.parametrize("bs", [1, 4, 16, 32, 128])
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 64)])
def test_attention_block_sizes(bs, dtype, d):
    c = Case(2, 6, 2, d, dtype, [9, 1, 20], [31, 64, 100], bs=bs)
    c.check(tree_attention(c.q.to(DEV), c.pool.to(DEV), c.meta()))


@pytest.mark.parametrize("bs", [1, 2, 8])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hkv,d,sizes,cached", [(8, 2, 64, [8, 3], [2000, 37]), (14, 2, 64, [9, 2, 0], [900, 0, 5]),
                                                   (14, 2, 64, [70, 1], [1500, 300]), (8, 2, 128, [5, 33], [600, 1]),
                                                   (8, 2, 128, [130, 17], [95, 1100])])
def test_attention_in_small_blocks(hq, hkv, d, sizes, cached, dtype, bs):
    """Every number of column blocks and contexts in parts, the rows of a tile in blocks of their own; an eager call
    and one that joins its parts by a launch."""
    c = Case(bs + d, hq, hkv, d, dtype, sizes, cached, bs=bs)
    m, q, pool = c.meta(), c.q.to(DEV), c.pool.to(DEV)
    c.check(tree_attention(q, pool, m))
    m.units = 0
    c.check(tree_attention(q, pool, m))


@pytest.mark.parametrize("seed", range(48))
def test_attention_of_random_steps(seed):
    """Steps of any geometry, type, block size and raggedness, every third one with masks of its own."""
    g = np.random.default_rng(1000 + seed)
    dtype, d = TYPES[seed % 3], (64, 128)[seed // 3 % 2]
    hkv, rep = int(g.integers(1, 4)), int(g.choice([1, 2, 3, 5, 7, 8, 12, 33]))
    seqs, most = int(g.integers(1, 6)), int(g.choice([1, 6, 40, 150]))
    sizes = [int(g.integers(0 if seqs > 1 else 1, most + 1)) for _ in range(seqs)]
    cached = [int(g.choice([0, 1, 17, 63, 64, 300, 1500])) for _ in range(seqs)]
    visible = [g.random((n, n)) < g.choice([0.0, 0.1, 0.9]) for n in sizes] if seed % 3 == 2 else None
    c = Case(2000 + seed, hkv * rep, hkv, d, dtype, sizes, cached, bs=int(g.choice([1, 2, 8, 16, 32, 64])), visible=visible)
    c.check(tree_attention(c.q.to(DEV), c.pool.to(DEV), c.meta()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (8, 2, 128)])
def test_attention_around_its_chunks(hq, hkv, d, dtype):
    # contexts that end one position before, on and behind multiples of 16, 32 and 128, from an empty cache on
    cached = [0, 14, 15, 16, 30, 31, 32, 62, 63, 64, 126, 127, 128, 129, 255, 256]
    c = Case(3, hq, hkv, d, dtype, [2] * len(cached), cached)
    c.check(tree_attention(c.q.to(DEV), c.pool.to(DEV), c.meta()))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_long_context(dtype):
    # one request: its context is split over workgroups and joined
    c = Case(4, 14, 2, 64, dtype, [6, 3], [7001, 4096])
    c.check(tree_attention(c.q.to(DEV), c.pool.to(DEV), c.meta()))
    c = Case(5, 4, 2, 128, dtype, [37], [5003])
    c.check(tree_attention(c.q.to(DEV), c.pool.to(DEV), c.meta()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_large_trees(dtype):
    c = Case(6, 4, 1, 64, dtype, [257, 100], [65, 0])
    c.check(tree_attention(c.q.to(DEV), c.pool.to(DEV), c.meta()))
    chain = [list(range(-1, 1023))]
    c = Case(7, 2, 1, 64, dtype, None, [5], parents=chain)
    c.check(tree_attention(c.q.to(DEV), c.pool.to(DEV), c.meta()))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_masks_of_any_kind(dtype):
    # rows that see nothing (empty cache, no node), everything, others only; from the metadata and from the device
    g = np.random.default_rng(8)
    vis = [g.random((n, n)) < 0.3 for n in (33, 70, 5)]
    vis[0][4] = False
    vis[1][69] = False
    vis[2][:] = False
    c = Case(8, 14, 2, 64, dtype, [33, 70, 5], [0, 40, 0], visible=vis)
    meta = c.meta()
    got = tree_attention(c.q.to(DEV), c.pool.to(DEV), meta)
    c.check(got)
    assert not got[4].any() and not got[103:108].any()
    assert got[33 + 69].any()                          # its cached positions
    plain = build_tree_metadata(c.parents, c.cached, c.tables, block_size=16, num_blocks=c.nb, num_heads=14,
                                num_kv_heads=2, head_dim=64, dtype=dtype).to(DEV)
    again = tree_attention(c.q.to(DEV), c.pool.to(DEV), plain, mask=meta.mask.clone())
    assert torch.equal(again, got)
    beyond = meta.mask.clone()                         # bits past the tree say nothing
    beyond[:33, 1] |= -2                               # nodes 33 .. 63 of a tree of 33 nodes
    beyond[:33, 2] = -1
    beyond[103:, 0] |= -32
    beyond[103:, 1:] = -1
    assert torch.equal(tree_attention(c.q.to(DEV), c.pool.to(DEV), plain, mask=beyond), got)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_attention_unseen_infinities(dtype, d):
    # what a node does not see has no effect on it, also where it is infinite or NaN
    parents = [[-1] + [0] * 39, [-1, 0, 0, 1, 1, 2]]
    c = Case(9, 6, 2, d, dtype, None, [21, 0], parents=parents)
    clean = tree_attention(c.q.to(DEV), c.pool.to(DEV), c.meta())
    c.check(clean)
    dirty = c.pool.clone()
    for b, node, kv, value in [(0, 3, 1, float("inf")), (0, 17, 1, float("nan")), (0, 18, 0, float("nan")),
                               (0, 39, 1, float("-inf")), (0, 38, 0, float("inf")), (1, 5, 1, float("inf")),
                               (1, 4, 0, float("-inf"))]:
        pos = c.cached[b] + node
        dirty[c.tables[b][pos // 16], kv, :, pos % 16, 5:9] = value
    got = tree_attention(c.q.to(DEV), dirty.to(DEV), c.meta())
    hurt = {3, 17, 18, 39, 38, 40 + 5, 40 + 4}
    fine = [i for i in range(46) if i not in hurt]
    # one value may take another way through the sums, so equal within the tolerance, not in bits
    out, weight, spread = c.want()
    h = HALF[dtype]
    tol = (h * out.abs() + (2 * h + 2 * ((d + 4) * spread[:, :, None] + 130) * 2.0 ** -24) * weight)[fine]
    assert ((got.cpu().double().view_as(out)[fine] - out[fine]).abs() <= tol).all()
    for row in (3, 39, 45):
        assert torch.isinf(got[row].float()).any()     # a visible infinity arrives
    assert torch.isnan(got[17].float()).any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0, 3.0])
def test_attention_scales(dtype, scale):
    c = Case(10, 14, 2, 64, dtype, [5, 20], [50, 3], magnitude=0.5)
    c.check(tree_attention(c.q.to(DEV), c.pool.to(DEV), c.meta(), scale=scale), scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_scores_far_apart(dtype):
    # one dominant position late in the context: the running maximum jumps
    c = Case(11, 4, 2, 64, dtype, [3], [400])
    pos = 390
    c.pool[c.tables[0][pos // 16], 0, :, pos % 16] = (c.q[0, ::2] * 4).to(dtype)
    c.check(tree_attention(c.q.to(DEV), c.pool.to(DEV), c.meta()))


@pytest.mark.parametrize("hq", [1, 33])
def test_attention_of_a_flat_tail_behind_a_dominant_key(hq):
    """fp16: 2^18 keys of a weight of 2^-25.4 beside one of 1 hold 0.6% of the sum. 512 sequences share them as a
    prefix, so that contexts stay whole and a wave's weights all refer to the dominant one. A weight is rounded to a
    multiple of 2^-24 and the reference maximum lies 7 below the first one: half a step is 2^-32 of the dominant weight, 1.1%
    of a tail weight; 2^-10 bounds the roundings of the output, of the scores and of the sums."""
    n, B, d, bs = 1 << 18, 512, 64, 128
    pool = torch.zeros(n // bs + B, 2, 1, bs, d, dtype=torch.float16)
    pool[:n // bs, 1] = 1.0
    pool[0, 0, 0, 5, 0], pool[0, 1, 0, 5] = 17.6, 0.0              # the dominant key: its value is 0
    pool[n // bs:, 0, :, :, 0], pool[n // bs:, 1] = -100.0, 0.0    # the nodes hold nothing
    score = float(pool[0, 0, 0, 5, 0])
    q = torch.zeros(B, hq, d, dtype=torch.float16)
    q[:, :, 0] = 1.0
    prefix = list(range(n // bs))
    meta = build_tree_metadata([[-1]] * B, [n] * B, [prefix + [n // bs + b] for b in range(B)], block_size=bs,
                               num_blocks=pool.shape[0], num_heads=hq, num_kv_heads=1, head_dim=d, dtype=torch.float16)
    assert meta.split_np.shape[0] == 0                             # the case that the test is about
    got = tree_attention(q.to(DEV), pool.to(DEV), meta.to(DEV), scale=1.0).cpu().double()
    tail = (n - 1) * np.exp(-score)
    want = tail / (1 + tail)
    assert 0.005 < want < 0.007
    assert ((got - want).abs() <= want * (2.0 ** -32 / np.exp(-score) + 2.0 ** -10)).all(), got.unique() / want


@pytest.mark.parametrize("step", [0.0, 0.004, 0.016, 0.03])
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_of_scores_past_24_bits(dtype, step):
    # scores of about 2^25.6 (in powers of two) that rise by up to some tens: in 32 bits they are off by 1 and more
    # themselves, and the weights with them, but a mean of the values it stays
    c = Case(16, 2, 1, 64, dtype, [2], [700])
    for pos in range(702):
        block = c.pool[c.tables[0][pos // 16], 0, :, pos % 16]
        block.fill_(2080.0)
        block[:, 0] = step * (pos // 64)
    c.q.fill_(2080.0)
    got = tree_attention(c.q.to(DEV), c.pool.to(DEV), c.meta()).cpu().double().view(2, 2, 64)
    v = torch.cat([c.pool[b, 1, 0] for b in c.tables[0]])[:702].double()
    assert torch.isfinite(got).all()
    slack = (HALF[dtype] + 702 * 2.0 ** -24) * v.abs().max(0).values
    assert (got <= v.max(0).values + slack).all() and (got >= v.min(0).values - slack).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_rope_positions_are_depths(dtype, d):
    c = Case(12, 6, 2, d, dtype, [12, 1, 25], [37, 0, 90])
    cos, sin = rope_tables(d, 1e6, 256, torch.device("cpu"))
    depth = [sum(s[i]) - 1 for s in c.seen for i in range(s.shape[0])]
    pos = torch.tensor([cc + int(x) for cc, n, s in zip(c.cached, c.sizes, np.cumsum([0] + c.sizes)) for x in depth[s:s + n]])
    rope = Rope(cos.to(DEV), sin.to(DEV))
    meta = c.meta()
    assert meta.positions.cpu().tolist() == pos.tolist()
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(38, 2, d, generator=g).to(dtype) for _ in range(2))
    from tinybatch_amd import tree_append
    pool = c.pool.to(DEV)
    tree_append(pool, k.to(DEV), v.to(DEV), meta, rope=rope)
    kr = oracle.rotate(k, cos[pos], sin[pos])
    row = 0
    for cc, n, t in zip(c.cached, c.sizes, c.tables):
        for i in range(n):
            at = cc + i
            c.pool[t[at // 16], 0, :, at % 16], c.pool[t[at // 16], 1, :, at % 16] = kr[row], v[row]
            row += 1
    used = torch.isfinite(c.pool.float()).view(torch.int8).bool()
    assert torch.equal(pool.cpu()[used], c.pool[used])
    c.check(tree_attention(c.q.to(DEV), pool, meta, rope=rope), q=oracle.rotate(c.q, cos[pos], sin[pos]))


def test_strided_rows_and_given_outputs():
    c = Case(13, 14, 2, 64, torch.bfloat16, [5, 9], [60, 20])
    want = tree_attention(c.q.to(DEV), c.pool.to(DEV), c.meta())
    wide = torch.zeros(14, 18 * 64, dtype=torch.bfloat16, device=DEV)      # q inside a row of q|k|v
    wide[:, :896] = c.q.view(14, 896).to(DEV)
    out = torch.full((20, 1024), 7.0, dtype=torch.bfloat16, device=DEV)
    got = tree_attention(wide[:, :896], c.pool.to(DEV), c.meta(), out=out[3:17, :896])
    assert got.data_ptr() == out[3:].data_ptr() and torch.equal(got, want)
    assert (out[:3] == 7).all() and (out[17:] == 7).all() and (out[:, 896:] == 7).all()


def test_a_larger_pool_than_the_metadata_s_and_an_empty_step():
    c = Case(14, 6, 2, 64, torch.float16, [4], [30])
    big = torch.full((c.nb + 9, 2, 2, 16, 64), float("nan"), dtype=torch.float16)
    big[:c.nb] = c.pool
    c.check(tree_attention(c.q.to(DEV), big.to(DEV), c.meta()))
    e = Case(14, 6, 2, 64, torch.float16, [0, 0], [30, 0])
    assert tree_attention(e.q.to(DEV), e.pool.to(DEV), e.meta()).shape == (0, 384)
    v = verify_tree(e.meta(), torch.zeros(0, dtype=torch.int64, device=DEV), torch.zeros(0, device=DEV), torch.zeros(0, 9, device=DEV))
    assert v.num_accepted.tolist() == [0, 0] and (v.tokens == -1).all() and (v.accepted == -1).all()


def test_offsets_past_32_bits():
    # a pool of more than 4 GiB, the sequence's blocks at its end
    nb = (5 << 30) // (2 * 2 * 64 * 128 * 2)
    c = Case(15, 4, 2, 128, torch.bfloat16, [6], [150], bs=64)
    pool = torch.empty(nb, 2, 2, 64, 128, dtype=torch.bfloat16, device=DEV)
    tables = [[nb - 1 - x for x in c.tables[0]]]
    for a, b in zip(c.tables[0], tables[0]):
        pool[b] = c.pool[a].to(DEV)
    meta = build_tree_metadata(c.parents, c.cached, tables, block_size=64, num_blocks=nb, num_heads=4, num_kv_heads=2,
                               head_dim=128, dtype=torch.bfloat16).to(DEV)
    c.check(tree_attention(c.q.to(DEV), pool, meta))


# ---- verification -------------------------------------------------------------------
def verify_case(seed, sizes, vocab, dtype, drafts, sharp=3.0, noise=1.0):
    g = torch.Generator().manual_seed(seed)
    parents = random_trees(seed, sizes)
    rows = sum(sizes)
    logits = torch.randn(rows, vocab, generator=g) * sharp
    probs = torch.softmax(logits, -1).to(dtype)
    logits = logits + torch.randn(rows, vocab, generator=g) * noise
    draft = torch.softmax(logits, -1).to(dtype) if drafts else None
    tokens = torch.zeros(rows, dtype=torch.int64)
    start = 0
    for t in parents:
        for i, p in enumerate(t):
            if p < 0:
                continue
            if drafts:
                tokens[start + i] = torch.multinomial(draft[start + p].float(), 1, generator=g)[0]
            else:
                tokens[start + i] = logits[start + p].topk(1 + t[:i].count(p)).indices[-1]
        start += len(t)
    return parents, tokens, torch.rand(rows, generator=g), probs, draft


def check_verify(parents, tokens, uniforms, probs, draft, got):
    acc, num, out = (x.cpu() for x in got)
    start, total = 0, 0
    for b, t in enumerate(parents):
        n = len(t)
        if n == 0:
            assert num[b] == 0 and (acc[b] == -1).all() and (out[b] == -1).all()
            continue
        s = slice(start, start + n)
        path, told = oracle.verify(t, tokens[s], uniforms[s], probs[s].double().numpy(),
                                   None if draft is None else draft[s].double().numpy())
        assert num[b] == len(path)
        assert acc[b].tolist() == path + [-1] * (acc.shape[1] - len(path))
        assert out[b].tolist() == told + [-1] * (out.shape[1] - len(told))
        start, total = start + n, total + len(path)
    return total


def on_gpu(parents, tokens, uniforms, probs, draft=None):
    meta = build_tree_metadata(parents).to(DEV)
    return verify_tree(meta, tokens.to(DEV), uniforms.to(DEV), probs.to(DEV), None if draft is None else draft.to(DEV))


@pytest.mark.parametrize("drafts", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 7, 1000, 1024, 32001, 151936])
def test_verify_against_the_walk(vocab, dtype, drafts):
    if vocab < 64:
        sizes = [3, 1, 2, 0, 1]
        case = verify_case(vocab, sizes, vocab, dtype, True)
        case = case if drafts else case[:4] + (None,)
    else:
        case = verify_case(vocab, [6, 1, 0, 24, 2, 13], vocab, dtype, drafts)
    check_verify(*case, on_gpu(*case))


@pytest.mark.parametrize("drafts", [False, True])
def test_verify_many_seeds(drafts):
    # small vocabularies, so that drafts are kept, refused and drawn twice
    kept = 0
    for seed in range(12):
        case = verify_case(seed, [30, 8, 64, 65, 3, 1, 70], 50, torch.float32, drafts, sharp=1.5, noise=0.5)
        kept += check_verify(*case, on_gpu(*case)) - 7
    assert kept > 20


def test_verify_trees_of_many_nodes_and_rounds():
    case = verify_case(5, [1024, 300], 2000, torch.float32, True, sharp=4.0, noise=4.0)
    check_verify(*case, on_gpu(*case))
    parents = [[-1] + [0] * 99, [-1] + [0] * 40]                 # many refusals at one node
    g = torch.Generator().manual_seed(6)
    probs = torch.softmax(torch.randn(141, 5000, generator=g) * 2, -1)
    draft = torch.softmax(torch.randn(141, 5000, generator=g) * 2, -1)
    tokens = torch.zeros(141, dtype=torch.int64)
    tokens[:100] = torch.multinomial(draft[0], 100, replacement=True, generator=g)
    tokens[100:] = torch.multinomial(draft[100], 41, replacement=True, generator=g)
    u = 0.9 + 0.1 * torch.rand(141, generator=g)
    u[0] = 0.3
    check_verify(parents, tokens, u, probs, draft, on_gpu(parents, tokens, u, probs, draft))
    check_verify(parents, tokens, u, probs, None, on_gpu(parents, tokens, u, probs))


def test_verify_edges():
    V = 40
    one = torch.zeros(2, V)
    one[:, 5] = 1.0
    z = torch.zeros(2)
    t = lambda *x: torch.tensor(x, dtype=torch.int64)  # noqa: E731
    parents = [[-1, 0]]
    for draft in (None, one):
        # a draft of all the mass is kept for every random number, a draft of none for no number
        for u in (0.0, 0.5, 1 - 2.0 ** -24):
            got = on_gpu(parents, t(0, 5), torch.full((2,), u), one, draft)
            assert got.num_accepted.tolist() == [2] and got.tokens.tolist() == [[5, 5]]
    got = on_gpu(parents, t(0, 6), z, one)
    assert got.num_accepted.tolist() == [1] and got.tokens.tolist() == [[5, -1]]
    # the target and the draft agree: always kept
    g = torch.Generator().manual_seed(1)
    p = torch.softmax(torch.randn(2, V, generator=g), -1)
    for x in range(V):
        assert on_gpu(parents, t(0, x), torch.full((2,), 1 - 2.0 ** -24), p, p).num_accepted.tolist() == [2]
    # a refused token that held all: nothing is left, the row's own distribution is taken
    both = [[-1, 0, 0]]
    p3 = torch.zeros(3, V)
    p3[:, 7], p3[:, 8] = 0.5, 0.5
    u = torch.tensor([0.75, 0.9, 0.99])
    got = on_gpu(both, t(0, 7, 7), u, p3)              # the same token twice: refused the second time too
    assert got.tokens.tolist() == [[8, -1, -1]]
    d3 = torch.zeros(3, V)
    d3[:, 3] = 1.0
    got = on_gpu(both, t(0, 3, 3), u, p3, d3)
    check_verify(both, t(0, 3, 3), u, p3, d3, got)
    # no mass at all, NaN, tokens outside the vocabulary
    got = on_gpu(parents, t(0, 5), z + 0.5, torch.zeros(2, V))
    assert got.tokens.tolist() == [[-1, -1]] and got.num_accepted.tolist() == [1]
    got = on_gpu(parents, t(0, 5), z + 0.5, torch.full((2, V), float("nan")))
    assert got.tokens.tolist() == [[-1, -1]] and got.num_accepted.tolist() == [1]
    for x in (-1, V, 1 << 40):
        got = on_gpu(parents, t(0, x), z, one)
        assert got.tokens.tolist() == [[5, -1]]
        got = on_gpu(parents, t(0, x), z, one, p)
        assert got.num_accepted.tolist() == [1]
    # a random number of 1 (outside the range) still gives a token that has weight
    assert on_gpu([[-1]], t(0), torch.ones(1), p3[:1]).tokens.tolist() == [[8]]
    assert on_gpu([[-1]], t(0), torch.zeros(1), p3[:1]).tokens.tolist() == [[7]]


def test_verify_rows_with_strides():
    parents, tokens, u, probs, draft = verify_case(9, [12, 5], 1001, torch.float32, True)
    wide = torch.full((17, 1203), float("nan"), device=DEV)
    wide[:, 1:1002] = probs.to(DEV)
    dwide = torch.full((17, 1500), float("nan"), device=DEV)
    dwide[:, 3:1004] = draft.to(DEV)
    meta = build_tree_metadata(parents).to(DEV)
    got = verify_tree(meta, tokens.to(DEV), u.to(DEV), wide[:, 1:1002], dwide[:, 3:1004])
    check_verify(parents, tokens, u, probs, draft, got)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [50, 5003])
def test_verify_of_entries_that_are_no_probabilities(vocab, dtype):
    """NaN and entries below 0 count as 0 in the draft's rows as in the target's: in the tests, in the sums
    after refusals and in the token drawn at the end."""
    differ = 0
    for seed in range(8):
        parents, tokens, u, probs, draft = verify_case(70 + seed, [30, 8, 66, 3, 1], vocab, dtype, True, sharp=1.5, noise=1.5)
        g = torch.Generator().manual_seed(seed)
        dirty = []
        for t in (probs, draft):
            r = torch.rand(t.shape, generator=g)
            t = torch.where(r < 0.15, torch.full_like(t, float("nan")), torch.where(r < 0.3, -t, t))
            dirty.append(t)
        probs, draft = dirty
        zeros = [torch.where(t > 0, t, torch.zeros_like(t)) for t in (probs, draft)]
        got = on_gpu(parents, tokens, u, probs, draft)
        check_verify(parents, tokens, u, *zeros, got)
        check_verify(parents, tokens, u, zeros[0], None, on_gpu(parents, tokens, u, probs))
        at = 0
        for t in parents:                              # children that only a draft entry of 0 lets through
            differ += sum(bool(zeros[0][at + p, tokens[at + i]] > 0) and not bool(draft[at + p, tokens[at + i]] > 0)
                          for i, p in enumerate(t) if i)
            at += len(t)
    assert differ > 20


def test_verify_keeps_the_target_s_distribution():
    # 20000 pairs of drafts of one distribution, drawn or taken as they are: the first emitted token's counts against the target's
    # probabilities, chi-square with 11 degrees of freedom (its 1 - 1e-9 quantile is 66)
    g = torch.Generator().manual_seed(3)
    B, V = 20000, 12
    p = torch.softmax(torch.randn(V, generator=g), -1)
    q = torch.softmax(torch.randn(V, generator=g), -1)
    probs, draft = p.expand(3 * B, V).contiguous(), q.expand(3 * B, V).contiguous()
    tokens = torch.multinomial(q, 3 * B, replacement=True, generator=g)
    u = torch.rand(3 * B, generator=g)
    for d in (draft, None):
        got = on_gpu([[-1, 0, 0]] * B, tokens, u, probs, d)
        count = torch.bincount(got.tokens[:, 0].cpu(), minlength=V).double()
        want = p.double() * B
        assert ((count - want) ** 2 / want).sum() < 66
        assert (got.num_accepted > 1).any() and (got.num_accepted == 1).any()


@pytest.mark.parametrize("sizes", [[1], [6, 0, 130, 64, 65, 1], [1024]])
def test_verify_greedy(sizes):
    g = torch.Generator().manual_seed(len(sizes))
    parents = random_trees(4, sizes)
    rows = sum(sizes)
    tokens, ids = torch.randint(0, 4, (rows,), generator=g), torch.randint(0, 4, (rows,), generator=g)
    meta = build_tree_metadata(parents).to(DEV)
    acc, num, out = (x.cpu() for x in verify_tree_greedy(meta, tokens.to(DEV), ids.to(DEV)))
    s = 0
    for b, t in enumerate(parents):
        path, told = [], []
        if t:
            path = [0]
            while True:
                nxt = [i for i in range(1, len(t)) if t[i] == path[-1] and tokens[s + i] == ids[s + path[-1]]]
                told.append(int(ids[s + path[-1]]))
                if not nxt:
                    break
                path.append(nxt[0])
        assert num[b] == len(path) and acc[b].tolist() == path + [-1] * (acc.shape[1] - len(path))
        assert out[b].tolist() == told + [-1] * (out.shape[1] - len(told))
        s += len(t)


# ---- commit ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,hkv,d,bs", [(torch.bfloat16, 2, 64, 16), (torch.float32, 8, 128, 32), (torch.float16, 1, 64, 4)])
def test_commit_moves_rows_and_nothing_else(dtype, hkv, d, bs):
    g = torch.Generator().manual_seed(bs)
    parents = random_trees(2, [1, 40, 0, 9, 200, 17])
    cached = [3, 30, 5, 0, 61, 16]
    need = [-(-(c + len(t)) // bs) for c, t in zip(cached, parents)]
    ids = torch.randperm(sum(need) + 2, generator=g).tolist()
    tables, at = [], 0
    for k in need:
        tables.append(ids[at:at + k])
        at += k
    storage = torch.randn(3, len(ids), 2, hkv, bs, d, generator=g).to(dtype)
    paths = []
    for t in parents:
        node, path = len(t) - 1, []
        while node >= 0:
            path.append(node)
            node = t[node]
        paths.append(path[::-1])
    paths[4] = list(range(0, 200, 3))                  # long paths, as any rising list of nodes
    paths[1] = [0] + list(range(5, 40))
    acc = torch.tensor([p + [-1] * (200 - len(p)) for p in paths], dtype=torch.int32)
    num = torch.tensor([len(p) for p in paths], dtype=torch.int32)
    want = storage.clone()
    for p, c, t in zip(paths, cached, tables):
        for j, i in enumerate(p):
            a, b = c + i, c + j
            want[:, t[b // bs], :, :, b % bs] = storage[:, t[a // bs], :, :, a % bs]
    meta = build_tree_metadata(parents, cached, tables, block_size=bs, num_blocks=len(ids), num_heads=hkv, num_kv_heads=hkv,
                               head_dim=d, dtype=dtype).to(DEV)
    dev = storage.to(DEV)
    commit_tree(dev, meta, acc.to(DEV), num.to(DEV))
    assert torch.equal(dev.cpu(), want)


def test_commit_of_paths_that_are_none():
    """Nodes outside the sequence's table, negative counts and counts past the row: what lies outside the
    table is left out, no other block changes."""
    parents, cached = [[-1, 0, 1], [-1, 0], [-1, 0, 0, 0]], [14, 32, 5]
    tables = [[9, 4], [2, 7, 5], [11]]
    storage = torch.randn(2, 13, 2, 2, 16, 64, generator=torch.Generator().manual_seed(3))
    acc = torch.tensor([[0, 2, 2 ** 31 - 1, 2 ** 30], [0, 1, -2 ** 31, 10 ** 6], [0, 3, 40, -7]], dtype=torch.int32)
    num = torch.tensor([4, -3, 2 ** 31 - 1], dtype=torch.int32)
    want = storage.clone()
    want[:, 9, :, :, 15] = storage[:, 4, :, :, 0]      # positions 16 and 8 to 15 and 6
    want[:, 11, :, :, 6] = storage[:, 11, :, :, 8]
    meta = build_tree_metadata(parents, cached, tables, block_size=16, num_blocks=13, num_heads=2, num_kv_heads=2,
                               head_dim=64, dtype=torch.float32).to(DEV)
    dev = storage.to(DEV)
    commit_tree(dev, meta, acc.to(DEV), num.to(DEV))
    assert torch.equal(dev.cpu(), want)


# ---- together ----------------------------------------------------------------------------
def step_case(cache, parents, cached, tables, hq, seed, rope):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rows = sum(len(t) for t in parents)
    q, k, v = (torch.randn(rows, h, cache.head_dim, generator=g, device=DEV).to(cache.dtype)
               for h in (hq, cache.n_kv_heads, cache.n_kv_heads))
    meta = cache.tree_metadata(parents, cached, tables, num_heads=hq)
    return meta, q, k, v


@pytest.mark.parametrize("largest", [0.5, 0.02])       # of the random numbers: some or most drafts kept
def test_a_step_from_append_to_commit(largest):
    """Append, attention, verification and commit of a step, then the next step's decode attention
    over the committed cache: the same as appending the kept tokens one after the other."""
    hq, hkv, d, bs, layers = 14, 2, 64, 16, 3
    dt = torch.bfloat16
    cos, sin = rope_tables(d, 1e6, 512, DEV)
    rope = Rope(cos, sin)
    cached = [33, 0, 120]
    parents = random_trees(21, [12, 7, 30])
    tables = [[2, 9, 5, 30], [7], [1, 3, 4, 6, 8, 10, 11, 12, 13, 14]]
    a, b = (PagedKVCache(layers, 40, bs, hkv, d, DEV, dt) for _ in range(2))
    g = torch.Generator(device=DEV).manual_seed(2)
    a.storage.normal_(generator=g)
    b.storage.copy_(a.storage)
    meta, q, k, v = step_case(a, parents, cached, tables, hq, 3, rope)
    for layer in range(layers):
        a.tree_append(layer, k, v, meta, rope=rope)
        out = a.tree_attention(layer, q, meta, rope=rope)
    assert torch.isfinite(out.float()).all()
    vocab = 60
    probs = torch.softmax(torch.randn(49, vocab, generator=g, device=DEV) * 2, -1)
    draft = torch.softmax(torch.randn(49, vocab, generator=g, device=DEV) * 2, -1)
    starts = np.cumsum([0] + [len(t) for t in parents])
    prow = torch.tensor([int(starts[i]) + max(p, 0) for i, t in enumerate(parents) for p in t], device=DEV)
    tokens = torch.multinomial(draft[prow], 1, generator=g)[:, 0]
    u = torch.rand(49, generator=g, device=DEV) * largest
    verdict = verify_tree(meta, tokens, u, probs, draft)
    a.commit_tree(meta, verdict.accepted, verdict.num_accepted)
    check_verify(parents, tokens.cpu(), u.cpu(), probs.cpu(), draft.cpu(), verdict)
    num = verdict.num_accepted.tolist()
    assert max(num) >= (2 if largest == 0.5 else 4)
    # the kept path as an ordinary prompt tail in the other cache
    rows = [int(s) + i for s, acc, n in zip(starts, verdict.accepted.tolist(), num) for i in acc[:n]]
    ends = np.cumsum([0] + num)
    slices = [(int(x), int(y)) for x, y in zip(ends, ends[1:])]
    positions = torch.tensor([c + j for c, n in zip(cached, num) for j in range(n)], device=DEV)
    ctx = [c + n for c, n in zip(cached, num)]
    for layer in range(layers):
        b.write(layer, k[rows], v[rows], positions, slices, tables, rope=rope)
        want = b.attention(layer, q[rows], positions, slices, tables, ctx, rope=rope)
    for t, c in zip(tables, ctx):
        pos = torch.arange(c)
        ids = torch.tensor(t)[pos // bs]
        assert torch.equal(a.storage[:, ids, :, :, pos % bs], b.storage[:, ids, :, :, pos % bs])
    torch.testing.assert_close(out[rows].float(), want.float(), atol=2e-2, rtol=2e-2)


def test_streams_and_graphs():
    """Two calls of one metadata on two streams, and each operator captured and replayed with other work
    between, give the eager results every time."""
    c = Case(31, 14, 2, 64, torch.bfloat16, [6, 20, 3], [3000, 700, 15])
    d = Case(32, 14, 2, 64, torch.bfloat16, [30, 2], [2500, 90])
    cases = [(c, c.meta(), c.q.to(DEV), c.pool.to(DEV)), (d, d.meta(), d.q.to(DEV), d.pool.to(DEV))]
    want = [tree_attention(q, pool, m) for _, m, q, pool in cases]
    vc = verify_case(33, [20, 6, 1], 30011, torch.float32, True)
    vm = build_tree_metadata(vc[0]).to(DEV)
    args = [x.to(DEV) for x in vc[1:]]
    ids = args[2].argmax(-1)
    verdict, greedy = verify_tree(vm, *args), verify_tree_greedy(vm, args[0], ids)
    check_verify(*vc, verdict)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        outs = []
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for s in streams:
            with torch.cuda.stream(s):
                outs.append([tree_attention(cases[0][2], cases[0][3], cases[0][1]), verify_tree(vm, *args)])
        torch.cuda.synchronize()
        for o, v in outs:
            assert torch.equal(o, want[0])
            assert all(torch.equal(x, y) for x, y in zip(v, verdict))
    graphs = []
    for _, m, q, pool in cases:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            got = tree_attention(q, pool, m), verify_tree(vm, *args), verify_tree_greedy(vm, args[0], ids)
        graphs.append((g, got))
    for i in range(4):
        for g, got in graphs:
            for t in (got[0], *got[1], *got[2]):
                t.zero_()
        eager = tree_attention(cases[i % 2][2], cases[i % 2][3], cases[i % 2][1])
        torch.cuda.synchronize()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager, want[i % 2])
        for (_, got), w in zip(graphs, want):
            assert torch.equal(got[0], w), f"replay {i}"
            assert all(torch.equal(x, y) for x, y in zip(got[1] + got[2], verdict + greedy)), f"replay {i}"


def test_threads_on_one_stream():
    """Calls of several threads on the same stream share its workspace, and none disturbs another."""
    c = Case(41, 14, 2, 64, torch.float32, [6, 20], [9000, 700])
    m, q, pool = c.meta(), c.q.to(DEV), c.pool.to(DEV)
    cases = [verify_case(s, [20, 6, 1], 30011, torch.float32, True) for s in (42, 43, 44)]
    metas = [build_tree_metadata(v[0]).to(DEV) for v in cases]
    args = [[x.to(DEV) for x in v[1:]] for v in cases]
    want, verdicts = tree_attention(q, pool, m), [verify_tree(vm, *a) for vm, a in zip(metas, args)]
    wrong = []

    def work(i):
        torch.cuda.set_device(DEV)
        for _ in range(100):
            got = [tree_attention(q, pool, m)] if i == 3 else list(verify_tree(metas[i], *args[i]))
            if not all(torch.equal(x, y) for x, y in zip(got, [want] if i == 3 else verdicts[i])):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("dtype,hq,hkv,d", [(torch.bfloat16, 14, 2, 64), (torch.float16, 16, 4, 64), (torch.bfloat16, 8, 4, 128),
                                            (torch.float32, 4, 2, 64), (torch.float32, 6, 6, 128)])
def test_parts_joined_here_and_by_a_launch(dtype, hq, hkv, d):
    """Few parts of few columns are joined by the last workgroup to arrive in an eager call, by a launch in a
    captured one: the same bits, the counters back at zero, calls one behind the other and of two streams."""
    from tinybatch_amd.tree import _SCRATCH
    vis = np.tril(np.ones((3, 3), dtype=bool))
    vis[1] = False
    cases = [Case(51, hq, hkv, d, dtype, [4], [600]), Case(52, hq, hkv, d, dtype, [3, 4, 1], [0, 700, 333], visible=[vis, None, None])]
    made = [(c, c.meta(), c.q.to(DEV), c.pool.to(DEV)) for c in cases]
    assert all(m.units for _, m, _, _ in made)         # these sizes take that way
    want = []
    for c, m, q, pool in made:
        want.append(tree_attention(q, pool, m))
        c.check(want[-1])
    assert not want[1][1].any()                        # a row that sees nothing, whole or in parts
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for i in range(6):
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got += [tree_attention(q, pool, m) for _, m, q, pool in (made if i % 2 else made[::-1])]
        torch.cuda.synchronize()
        for k, o in enumerate(got):
            assert torch.equal(o, want[k % 2 if i % 2 else 1 - k % 2])
    assert all(not s.arrivals.any() for s in _SCRATCH.values())
    for (c, m, q, pool), w in zip(made, want):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = tree_attention(q, pool, m)
        for _ in range(3):
            out.zero_()
            assert torch.equal(tree_attention(q, pool, m), w)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, w)


@pytest.mark.parametrize("drafts", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_verify_ends_here_and_by_a_launch(dtype, drafts):
    # the same of verification, whose captured calls end in a launch of their own
    from tinybatch_amd.tree import _SCRATCH
    for seed, sizes in ((61, [30, 1, 0, 12]), (62, [100, 70])):
        case = verify_case(seed, sizes, 5003, dtype, drafts, sharp=2.0, noise=2.0)
        meta = build_tree_metadata(case[0]).to(DEV)
        args = [None if x is None else x.to(DEV) for x in case[1:]]
        want = verify_tree(meta, *args)
        check_verify(*case, want)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            got = verify_tree(meta, *args)
        for _ in range(3):
            for t in got:
                t.zero_()
            again = verify_tree(meta, *args)
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(want, got, again))
    assert all(not s.arrivals.any() for s in _SCRATCH.values())


def test_verify_with_a_hint_too_small():
    # max_refusals only says how many launches sums get: a caller's mistake costs time, not the result
    case = verify_case(63, [40, 9], 3001, torch.float32, True, sharp=3.0, noise=3.0)
    meta = build_tree_metadata(case[0]).to(DEV)
    for refusals in (0, 1, 2, 50):
        meta.max_refusals = refusals
        check_verify(*case, verify_tree(meta, *[x.to(DEV) for x in case[1:]]))


def test_commit_replays_from_a_graph():
    hkv, d, bs = 2, 64, 16
    g = torch.Generator(device=DEV).manual_seed(5)
    first = torch.randn(2, 12, 2, hkv, bs, d, generator=g, device=DEV).to(torch.float16)
    parents, cached, tables = random_trees(3, [20, 9]), [10, 40], [[0, 1], [2, 3, 4, 5]]
    meta = build_tree_metadata(parents, cached, tables, block_size=bs, num_blocks=12, num_heads=hkv, num_kv_heads=hkv,
                               head_dim=d, dtype=torch.float16).to(DEV)
    acc = torch.tensor([[0, 4, 9, 19], [0, 3, 8, -1]], dtype=torch.int32, device=DEV)
    num = torch.tensor([4, 3], dtype=torch.int32, device=DEV)
    want = first.clone()
    commit_tree(want, meta, acc, num)
    storage = first.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        commit_tree(storage, meta, acc, num)
    for _ in range(3):
        storage.copy_(first)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(storage, want)


# ---- refusals on the GPU -------------------------------------------------------------------
def test_calls_that_do_not_fit_are_refused():
    c = Case(41, 6, 2, 64, torch.float16, [4], [30])
    q, pool, meta = c.q.to(DEV), c.pool.to(DEV), c.meta()
    with pytest.raises(ValueError, match="rows"):
        tree_attention(q[:3], pool, meta)
    with pytest.raises(TypeError, match="dtype"):
        tree_attention(q.float(), pool, meta)
    with pytest.raises(ValueError, match="metadata is for"):
        tree_attention(q, pool[:, :, :1].contiguous(), meta)
    with pytest.raises(ValueError, match="metadata is for"):
        tree_attention(q, pool[:4].contiguous(), meta)
    with pytest.raises(ValueError, match="uploaded"):
        tree_attention(q, pool, build_tree_metadata(c.parents))
    with pytest.raises(ValueError, match="without cached_lens"):
        tree_attention(q, pool, build_tree_metadata(c.parents).to(DEV))
    with pytest.raises(TypeError, match="mask"):
        tree_attention(q, pool, meta, mask=meta.mask[:3])
    with pytest.raises(ValueError, match="out"):
        tree_attention(q, pool, meta, out=torch.empty(4, 384, device=DEV))
    short = Rope(torch.zeros(31, 32, device=DEV), torch.zeros(31, 32, device=DEV))
    with pytest.raises(IndexError, match="rope"):
        tree_attention(q, pool, meta, rope=short)
    from tinybatch_amd import tree_append
    with pytest.raises(IndexError, match="rope"):
        tree_append(pool, q[:, :2], q[:, 2:4], meta, rope=short)
    with pytest.raises(RuntimeError, match="invalid"):           # rows that are not 16-byte aligned
        tree_attention(torch.zeros(4, 385, dtype=torch.float16, device=DEV)[:, 1:], pool, meta)
    t, u, p = torch.zeros(4, dtype=torch.int64, device=DEV), torch.zeros(4, device=DEV), torch.zeros(4, 9, device=DEV)
    with pytest.raises(ValueError, match="probs"):
        verify_tree(meta, t, u, p[:3])
    with pytest.raises(ValueError, match="draft_probs"):
        verify_tree(meta, t, u, p, p[:, :8])
    with pytest.raises(TypeError, match="draft_probs"):
        verify_tree(meta, t, u, p, p.half())
    with pytest.raises(TypeError, match="tokens"):
        verify_tree(meta, t.int(), u, p)
    with pytest.raises(TypeError, match="uniforms"):
        verify_tree(meta, t, u.double(), p)
    with pytest.raises(TypeError, match="unsupported"):
        verify_tree(meta, t, u, p.double())
    with pytest.raises(TypeError, match="target_ids"):
        verify_tree_greedy(meta, t, t[:3])
    acc, num = torch.zeros(1, 4, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    with pytest.raises(TypeError, match="accepted"):
        commit_tree(pool[None], meta, acc.long(), num)
    with pytest.raises(TypeError, match="num_accepted"):
        commit_tree(pool[None], meta, acc, num.long())
    with pytest.raises(ValueError, match="storage"):
        commit_tree(pool, meta, acc, num)


@pytest.mark.parametrize("dtype,hq,hkv,d,cached", [(torch.float32, 2, 1, 64, 560), (torch.float32, 8, 2, 64, 600), (torch.bfloat16, 32, 8, 128, 1000),
                                                   (torch.float16, 8, 4, 128, 900)])
def test_more_than_eight_parts_joined_both_ways(dtype, hq, hkv, d, cached):
    # a second turn of loads in either join: the same bits there and by a launch, for any values
    seen = 0
    for seed in range(40):
        c = Case(100 + seed, hq, hkv, d, dtype, [1 + seed % 9], [cached - seed])
        m, q, pool = c.meta(), c.q.to(DEV), c.pool.to(DEV)
        if not m.units or int(m.split_np[:, 2].max()) <= 8:
            continue
        seen += 1
        here = tree_attention(q, pool, m)
        m.units = 0
        assert torch.equal(here, tree_attention(q, pool, m)), seed
    assert seen > 5
