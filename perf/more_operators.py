"""What is measured of beam search over the paged cache: a request decodes several
continuations (its beams) side by side, and everything between two forward passes stays on the
GPU. Four operators serve a step:

* ``step``: which blocks the rows' new tokens need, taken from the free blocks, with the block
  tables, positions, slots and attention work items of the step, from lengths that only the GPU
  knows (``build_device_step``); rows are beams or any other requests;
* ``attend``: one new token per beam over the paged cache, the blocks that a request's beams
  share and those of each beam (``beam_attention``);
* ``select``: the best continuations of a request over its beams and the vocabulary
  (``select_beams``);
* ``reorder``: the beams' tables, reference counts and K/V follow the parents that were selected
  (``reorder_beams``).

Lengths, parents and who has ended are drawn from the case alone (``lengths`` seeds them), so
that a case is the same work for every seed of its inputs.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
# query heads, kv heads, head dim, layers
GEOMETRY = {"qwen": (14, 2, 64, 24), "llama": (32, 8, 128, 32), "mqa": (12, 1, 64, 6), "mha": (5, 5, 128, 4)}


def _select(name, dtype, requests, beams, vocab, candidates, kind, lengths=1):
    return {"name": name, "op": "select", "dtype": dtype, "requests": requests, "beams": beams, "vocab": vocab,
            "candidates": candidates, "kind": kind, "lengths": lengths}


def _reorder(name, geometry, dtype, requests, beams, prompt, made, block=16, lengths=1):
    return {"name": name, "op": "reorder", "geometry": geometry, "dtype": dtype, "requests": requests, "beams": beams,
            "prompt": prompt, "made": made, "block": block, "lengths": lengths}


def _step(name, rows, cached, new, partition, group, block=16, lengths=1):
    return {"name": name, "op": "step", "rows": rows, "cached": cached, "new": new, "partition": partition,
            "group": group, "block": block, "lengths": lengths}


def _attend(name, geometry, dtype, requests, beams, prompt, made, block=16, lengths=1):
    return {"name": name, "op": "attend", "geometry": geometry, "dtype": dtype, "requests": requests, "beams": beams,
            "prompt": prompt, "made": made, "block": block, "lengths": lengths}


def listed():
    return [
        # one user's request with four beams, the model's float logits: latency
        _select("select one request", "float32", 1, 4, 151936, 8, "open", lengths=1),
        # a serving batch, the LM head's 16-bit logits, some beams ended
        _select("select 32 requests bf16", "bfloat16", 32, 8, 151936, 16, "ended", lengths=2),
        # a small model's odd vocabulary, constrained decoding: most tokens masked, some beams lost
        _select("select masked fp16", "float16", 7, 5, 50257, 10, "masked", lengths=3),
        # many beams of few requests, for reranking
        _select("select 48 beams wide", "float32", 4, 48, 128256, 96, "open", lengths=4),
        # one user's request in a small model's layers
        _reorder("reorder one request", "qwen", "bfloat16", 1, 4, "600:600", "47:47", lengths=5),
        # a serving batch in the small model's layers
        _reorder("reorder 32 requests", "qwen", "bfloat16", 32, 8, "100:2000", "3:200", lengths=6),
        # the layers of the 8B geometry
        _reorder("reorder 16 requests 8B", "llama", "bfloat16", 16, 4, "200:900", "3:200", lengths=7),
        # a decode step of the serving batch's beams
        _step("step 256 beams", 256, "512:4096", "1:1", 256, 1, lengths=8),
        # a step of prompts and chunks beside decoding rows
        _step("step 300 rows mixed", 300, "0:2000", "0:100", 256, 2, lengths=9),
        # the parity precision: a few short requests
        _attend("attend fp32 short", "qwen", "float32", 2, 3, "29:300", "1:40", lengths=10),
        # a serving batch over contexts of the headline decode step
        _attend("attend bf16 32 requests", "qwen", "bfloat16", 32, 8, "512:4096", "3:200", lengths=11),
        # long contexts at the 8B geometry
        _attend("attend bf16 8B long", "llama", "bfloat16", 24, 4, "lognormal:8192:0.5:1024:24000", "3:400", lengths=12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """A case of the ranges above: other batches, beams, vocabularies, lengths, geometries and
    types, each no more work than the largest above of its kind."""
    lengths = rng.randrange(1, 1 << 20)
    op = rng.choice(["select", "reorder", "step", "attend", "attend"])
    beams = _log_int(rng, 1, 24)
    block = rng.choice([16, 16, 32])
    if op == "select":
        vocab = rng.choice([151936, 128256, 50257, 32001, 32000, 257])
        requests = max(1, min(_log_int(rng, 1, 64), 36_000_000 // (vocab * beams), 400 // beams))
        c = _select("", rng.choice(["float32", "float32", "float16", "bfloat16"]), requests, beams, vocab,
                    min(rng.choice([beams, 2 * beams]), 96), rng.choice(["open", "ended", "masked"]), lengths)
    elif op == "reorder":
        g = rng.choice(["qwen", "llama", "mqa", "mha"])
        requests = max(1, min(_log_int(rng, 1, 40), (256 if g != "llama" else 64) // beams))
        hi = _log_int(rng, 5, 2000 if g != "llama" else 800)
        c = _reorder("", g, rng.choice(["bfloat16", "float16", "float32"]) if g != "llama" else "float16", requests,
                     beams, f"{max(1, hi // 6)}:{hi}", f"1:{_log_int(rng, 2, 200)}", block, lengths)
    elif op == "step":
        rows = _log_int(rng, 1, 300)
        hi = _log_int(rng, 1, 4000)
        new = rng.choice(["1:1", "0:1", f"0:{_log_int(rng, 2, 100)}"])
        c = _step("", rows, f"{rng.choice([0, hi // 2])}:{hi}", new, rng.choice([64, 256, 512]), rng.choice([1, 2, 4]),
                  block, lengths)
    else:
        g = rng.choice(["qwen", "qwen", "llama", "mqa", "mha"])
        hq, hkv, d, _ = GEOMETRY[g]
        dt = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
        hi = _log_int(rng, 9, 12000)
        made = _log_int(rng, 2, 300)
        # positions times query rows bounded, and the cache that the plain form lays out row by row
        most = (1_500_000_000 if dt != "float32" else 300_000_000) // (hkv * d * beams)
        requests = max(1, min(_log_int(rng, 1, 40), most // (hi + made), 400 // beams))
        c = _attend("", g, dt, requests, beams, f"{max(1, hi // 6)}:{hi}", f"1:{made}", block, lengths)
    c.pop("name")
    return c


# ---- what a case's sizes come to ------------------------------------------------
def _draws(rng, spec, n):
    if spec.startswith("lognormal:"):
        median, sigma, lo, hi = (float(x) for x in spec.split(":")[1:])
        return [int(min(hi, max(lo, round(median * math.exp(sigma * rng.gauss(0, 1)))))) for _ in range(n)]
    lo, hi = (int(x) for x in spec.split(":"))
    return [rng.randint(lo, hi) for _ in range(n)]


def _prompts(case):
    """Each request's prompt and how many tokens its beams have made since."""
    return list(zip(_draws(random.Random(case["lengths"]), case["prompt"], case["requests"]),
                    _draws(random.Random(case["lengths"] + 1), case["made"], case["requests"])))


def _parents(case):
    """The parents that a selection gave, best candidate first: good beams have several children."""
    rng = random.Random(case["lengths"] + 2)
    K = case["beams"]
    return [[min(int(K * rng.random() ** 1.5), K - 1) for _ in range(K)] for _ in range(case["requests"])]


def _ended(case):
    rng = random.Random(case["lengths"])
    share = 0.3 if case["kind"] == "ended" else 0.0
    return [[rng.random() < share for _ in range(case["beams"])] for _ in range(case["requests"])]


def _lost(case):
    """How many of a request's beams, its last, are lost."""
    return case["beams"] // 4 if case["kind"] == "masked" else 0


def _new_lens(case):
    """(cached, new) tokens of every row; rows of a wide range of new tokens are mostly decoding."""
    rng = random.Random(case["lengths"] + 1)
    cached, lo_hi = _draws(random.Random(case["lengths"]), case["cached"], case["rows"]), case["new"]
    lo, hi = (int(x) for x in lo_hi.split(":"))
    new = [rng.randint(lo, hi) if hi <= 1 or rng.random() < 0.5 else 1 for _ in cached]
    return cached, new


def _parts(case):
    """(work items, partitions, rows of several partitions) of a step."""
    P, group = case["partition"], case["group"]
    items = parts = split = 0
    for c, n in zip(*_new_lens(case)):
        i = 0
        while i < n:
            np_ = -(-(c + i + 1) // P)
            k = 1
            while i + k < n and k < group and -(-(c + i + k + 1) // P) == np_:
                k += 1
            items += np_
            parts += np_ * k
            split += k if np_ > 1 else 0
            i += k
    return items, parts, split


def work(case):
    if case["op"] == "select":
        # the beams that have ended or are lost need no look at their logits
        rows = sum(map(len, _ended(case))) - sum(map(sum, _ended(case))) - case["requests"] * _lost(case)
        return {"bytes": rows * case["vocab"] * DTYPES[case["dtype"]].itemsize, "flops": 2 * rows * case["vocab"]}
    bs = case["block"]
    if case["op"] == "step":
        cached, new = _new_lens(case)
        tokens, (items, parts, split) = sum(new), _parts(case)
        blocks = sum(-(-(c + n) // bs) - -(-c // bs) for c, n in zip(cached, new))
        return {"bytes": 16 * len(new) + 20 * tokens + 12 * blocks + 16 * (items + split), "flops": 0}
    hq, hkv, d, layers = GEOMETRY[case["geometry"]]
    b = DTYPES[case["dtype"]].itemsize
    if case["op"] == "reorder":
        moved = entries = 0
        for (p, m), parents in zip(_prompts(case), _parents(case)):
            moved += (len(parents) - len(set(parents))) * ((p + m) % bs)
            entries += len(parents) * -(-(p + m) // bs)
        return {"bytes": moved * layers * 2 * 2 * hkv * d * b + 2 * 4 * entries, "flops": 0}
    rows = case["requests"] * case["beams"]
    kv = pairs = 0
    for p, m in _prompts(case):
        shared = p // bs * bs
        kv += shared + case["beams"] * (p + m - shared)
        pairs += case["beams"] * (p + m)
    return {"bytes": kv * 2 * hkv * d * b + 2 * rows * hq * d * b, "flops": 4 * hq * d * pairs}


# ---- inputs -----------------------------------------------------------------------
def _dev():
    return torch.device("cuda", torch.cuda.current_device())


def _generator(seed):
    return torch.Generator(device=_dev()).manual_seed(int(seed))


def _tensor(values, dtype=torch.int64):
    return torch.tensor(values, dtype=dtype, device=_dev())


def _select_inputs(case, seed):
    """Logits [requests * beams, vocab], the beams' scores [requests, beams] (falling, -inf: a
    beam that is lost), and which have ended (None: not asked for)."""
    g = _generator(seed)
    R, K, V, dev = case["requests"], case["beams"], case["vocab"], _dev()
    logits = torch.randn(R * K, V, generator=g, device=dev) * 3
    scores = -(torch.rand(R, K, generator=g, device=dev) * 0.4).cumsum(1) - 20 * torch.rand(R, 1, generator=g, device=dev)
    ended = None
    if case["kind"] == "masked":
        # what the constraint allows: a few hundred tokens, the rest masked out
        allowed = torch.rand(R * K, V, generator=g, device=dev) < 300.0 / V
        logits.masked_fill_(~allowed, -math.inf)
        scores[:, K - _lost(case):] = -math.inf
    elif case["kind"] == "ended":
        ended = _tensor(_ended(case), torch.bool)
    return logits.to(DTYPES[case["dtype"]]), scores, ended


def _beams(case, seed, spare):
    """Block tables of every beam (the prompt's whole blocks shared, the rest its own) over a
    shuffled pool, the contexts, the free blocks (``spare`` of them), the pool's size."""
    bs, K = case["block"], case["beams"]
    prompts = _prompts(case)
    total = sum(p // bs + K * (-(-(p + m) // bs) - p // bs) for p, m in prompts) + spare
    ids = list(range(total))
    random.Random(int(seed) * 7919 + case["lengths"]).shuffle(ids)
    tables, at = [], 0
    for p, m in prompts:
        shared, mine = p // bs, -(-(p + m) // bs) - p // bs
        for k in range(K):
            first = at + shared + k * mine
            tables.append(ids[at:at + shared] + ids[first:first + mine])
        at += shared + K * mine
    return tables, [p + m for p, m in prompts for _ in range(K)], ids[at:], total


def _padded(rows, width, fill=-1):
    return [list(r) + [fill] * (width - len(r)) for r in rows]


def _step_inputs(case, seed):
    """The rows' tables, cached and new lengths, the free blocks and the pool's size."""
    bs = case["block"]
    cached, new = _new_lens(case)
    have = [-(-c // bs) for c in cached]
    want = sum(-(-(c + n) // bs) for c, n in zip(cached, new)) - sum(have)
    total = sum(have) + want + want // 8 + 7
    ids = list(range(total))
    random.Random(int(seed) * 7919 + case["lengths"]).shuffle(ids)
    tables, at = [], 0
    for k in have:
        tables.append(ids[at:at + k])
        at += k
    return tables, cached, new, ids[at:], total


def _step_sizes(case):
    """What a program sets a step's arrays to: tokens, work items, partitions, rows of several."""
    cached, new = _new_lens(case)
    items, parts, split = _parts(case)
    return {"tokens": sum(new) + 3, "items": items + 5, "parts": parts + 5, "split": split + 5,
            "width": max(-(-(c + n) // case["block"]) for c, n in zip(cached, new)) + 2}


def _paged(case, tables, lens, free, total, group, width):
    """The rows' paged state: with ``own`` the framework's, otherwise the same arrays."""
    if own:
        from tinybatch_amd import DeviceTables

        return DeviceTables.from_lists(tables, lens, free, max_blocks=width, block_size=case["block"],
                                       num_blocks=total, group_size=group, device=_dev())
    refs = np.zeros(total, dtype=np.int64)
    for t in tables:
        refs[t] += 1
    return {"tables": _tensor(_padded(tables, width), torch.int32), "lens": _tensor(lens, torch.int32),
            "refs": _tensor(refs.tolist(), torch.int32), "num_free": _tensor([len(free)], torch.int32),
            "free": _tensor(free + [0] * (total - len(free)), torch.int32),
            "shared": torch.zeros(len(lens) // group, dtype=torch.int32, device=_dev())}


@torch.no_grad()
def prepare(case, seed):
    """The inputs and the state that a search keeps from step to step."""
    state = {"case": case}
    if case["op"] == "select":
        state["logits"], state["scores"], state["ended"] = _select_inputs(case, seed)
        return state
    if case["op"] == "step":
        tables, cached, new, free, total = _step_inputs(case, seed)
        z = _step_sizes(case)
        state["new"] = _tensor(new, torch.int32)
        state["paged"] = _paged(case, tables, cached, free, total, 1, z["width"])
        if own:
            state["step"] = state["paged"].new_step(max_tokens=z["tokens"], partition_tokens=case["partition"],
                                                    rows_per_item=case["group"], max_items=z["items"],
                                                    max_partitions=z["parts"], max_split_rows=z["split"])
        else:
            state["items"] = torch.zeros(z["items"], 4, dtype=torch.int32, device=_dev())
            state["split"] = torch.zeros(z["split"], 4, dtype=torch.int32, device=_dev())
            state["tokens"] = z["tokens"]
        return state
    K = case["beams"]
    hq, hkv, d, layers = GEOMETRY[case["geometry"]]
    g, dt = _generator(seed), DTYPES[case["dtype"]]
    if case["op"] == "reorder":
        tables, lens, free, total = _beams(case, seed, case["requests"] * K)
        storage = torch.empty(layers, total, 2, hkv, case["block"], d, device=_dev(), dtype=dt)
        for layer in storage:
            layer.normal_(generator=g)
        state["storage"], state["parents"] = storage, _tensor(_parents(case), torch.int32)
        state["paged"] = _paged(case, tables, lens, free, total, K, max(map(len, tables)) + 1)
        return state
    state["q"], state["pool"], tables, lens = _attend_inputs(case, seed)
    if own:
        from tinybatch_amd import BeamPlan, DeviceTables

        paged = DeviceTables.from_lists(tables, lens, [], max_blocks=max(map(len, tables)), block_size=case["block"],
                                        num_blocks=state["pool"].shape[0], group_size=K, device=_dev())
        state["plan"] = BeamPlan(paged, num_heads=hq, num_kv_heads=hkv, head_dim=d, dtype=dt)
        state["plan"].build()
    else:
        state["tables"] = _tensor(_padded(tables, max(map(len, tables)), 0))
        state["lens"] = _tensor(lens)
    return state


def _attend_inputs(case, seed):
    g, dt = _generator(seed), DTYPES[case["dtype"]]
    hq, hkv, d, _ = GEOMETRY[case["geometry"]]
    tables, lens, _, total = _beams(case, seed, 3)
    q = torch.randn(len(lens), hq, d, generator=g, device=_dev()).to(dt)
    pool = torch.empty(total, 2, hkv, case["block"], d, device=_dev(), dtype=dt).normal_(generator=g)
    return q, pool, tables, lens


@torch.no_grad()
def run(state):
    case = state["case"]
    if own:
        from tinybatch_amd import beam_attention, build_device_step, reorder_beams, select_beams

        if case["op"] == "select":
            c = select_beams(state["logits"], state["scores"], num_candidates=case["candidates"],
                             finished=state["ended"], end_token=2)
            return {"scores": c.scores, "parents": c.parents, "tokens": c.tokens}
        if case["op"] == "attend":
            return beam_attention(state["q"], state["pool"], state["plan"])
        t = state["paged"]
        if case["op"] == "reorder":
            reorder_beams(state["storage"], t, state["parents"])
            return {"storage": state["storage"], "tables": t.block_tables, "lens": t.context_lens, "refs": t.ref_counts,
                    "free": t.free_blocks, "num_free": t.num_free, "shared": t.shared_blocks}
        s = build_device_step(t, state["new"], state["step"])
        return {"tables": t.block_tables, "refs": t.ref_counts, "num_free": s.num_free, "lens": s.context_lens,
                "starts": s.query_start_loc, "positions": s.positions, "slots": s.slot_mapping, "row_ctx": s.row_ctx,
                "offsets": s.row_part_offsets, "items": s.work_items, "split": s.split_rows, "counts": s.counts}
    if case["op"] == "select":
        return _plain_select(state)
    if case["op"] == "attend":
        return _plain_attend(state)
    return _plain_reorder(state) if case["op"] == "reorder" else _plain_step(state)


# ---- plain forms ------------------------------------------------------------------
def _plain_select(state):
    case, scores, ended = state["case"], state["scores"], state["ended"]
    R, K, V = case["requests"], case["beams"], case["vocab"]
    x = state["logits"].double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    m = x.amax(1, keepdim=True)
    y = torch.where(x == m, 0.0, x - m)                          # (-inf - -inf: a row without any)
    y = y - y.exp().sum(1, keepdim=True).log()
    c = scores.double().reshape(R * K, 1) + torch.where(x == -math.inf, -math.inf, y)
    if ended is not None:
        only = torch.full_like(c, -math.inf)
        only[:, 2] = scores.double().reshape(R * K)
        c = torch.where(ended.reshape(R * K, 1), only, c)
    c = torch.where(torch.isnan(c), -math.inf, c).reshape(R, K * V)
    best, at = torch.sort(c, dim=1, descending=True, stable=True)
    best, at = best[:, :case["candidates"]], at[:, :case["candidates"]]
    none = best == -math.inf
    return {"scores": best.float(), "parents": torch.where(none, -1, at // V).int(),
            "tokens": torch.where(none, -1, at % V)}


def _plain_reorder(state):
    case, s, storage, parents = state["case"], state["paged"], state["storage"], state["parents"].long()
    bs, (G, K) = case["block"], parents.shape
    R, dev = G * K, parents.device
    tables, lens, refs, free, num_free = s["tables"].long(), s["lens"].long(), s["refs"].long(), s["free"], s["num_free"]
    row = torch.arange(R, device=dev)
    src = (row // K * K) + parents.reshape(R).clamp(min=0)
    live = (parents.reshape(R) >= 0) & (lens[src] > 0)
    ctx = torch.where(live, lens[src], 0)
    # the block that is not full: the first child keeps it if nobody else holds it
    full, rest = ctx // bs, ctx % bs
    same = (parents[:, :, None] == parents[:, None, :]) & (row[:K, None] > row[None, :K])
    first = ~same.any(2).reshape(R)
    old = tables[src]
    open_block = old.gather(1, full.clamp(max=old.shape[1] - 1)[:, None])[:, 0]
    copies = live & (rest > 0) & ~(first & (refs[open_block.clamp(min=0)] == 1))
    place = copies.long().cumsum(0) - 1
    enough = copies.sum() <= num_free[0]
    copies = copies & enough
    fresh = free.long()[(num_free[0] - 1 - place).clamp(min=0)]
    # tables
    j = torch.arange(tables.shape[1], device=dev)[None, :]
    used = -(-ctx // bs)
    new = torch.where(j < used[:, None], old, -1)
    new = torch.where((j == full[:, None]) & copies[:, None], fresh[:, None], new)
    width = (-(-lens // bs)).reshape(G, K).amax(1).repeat_interleave(K)[:, None]
    new = torch.where((j < width) & enough, new, tables)
    # who holds what, before and after; the freed blocks in the order of (request, column, row)
    held = j < (-(-lens // bs))[:, None]
    n = refs.shape[0]
    before = torch.zeros(n + 1, dtype=torch.int64, device=dev)
    before.index_add_(0, torch.where(held, tables, n).reshape(-1), torch.ones(R * j.shape[1], dtype=torch.int64, device=dev))
    after = torch.zeros_like(before)
    mine = torch.where(j < torch.where(enough, used, -(-lens // bs))[:, None], new, n).reshape(-1)
    after.index_add_(0, mine, torch.ones_like(mine))
    got = refs - before[:n] + after[:n]
    new_block = torch.zeros(n + 1, dtype=torch.bool, device=dev)
    new_block[torch.where(copies, fresh, n)] = True
    got = torch.where(new_block[:n], 1, got)
    order = torch.full((n + 1,), R * j.shape[1], dtype=torch.int64, device=dev)
    at = (row[:, None] // K * j.shape[1] + j) * K + row[:, None] % K
    order.scatter_reduce_(0, torch.where(held, tables, n).reshape(-1), at.reshape(-1), "amin")
    gone = (before[:n] > 0) & (got == 0)
    rank = torch.argsort(torch.where(gone, order[:n], R * j.shape[1] + 1), stable=True)
    left = num_free[0] - copies.sum()
    push = torch.arange(n, device=dev)
    kept = push < gone.sum()
    spots = torch.where(kept, left + push, n)
    longer = torch.cat([free, free[:1]])
    longer[spots] = rank.int()
    # the copied positions, in every layer
    many = torch.arange(bs, device=dev)
    take = copies[:, None] & (many[None, :] < rest[:, None])
    r, p = take.nonzero(as_tuple=True)
    storage[:, fresh[r], :, :, p] = storage[:, open_block[r], :, :, p]
    # the leading blocks that all live beams of a request share
    lives = (torch.where(enough, ctx, lens) > 0).reshape(G, K)
    t3 = new.reshape(G, K, -1)
    one = t3.gather(1, lives.int().argmax(1)[:, None, None].expand(-1, 1, t3.shape[2]))
    whole = (torch.where(enough, ctx, lens) // bs).reshape(G, K, 1)
    agree = ((t3 == one) & (j[None] < whole)) | ~lives[:, :, None]
    shared = torch.where(lives.any(1), agree.all(1).long().cumprod(1).sum(1), 0)
    s["tables"].copy_(new)
    s["lens"].copy_(torch.where(enough, ctx, lens))
    s["refs"].copy_(torch.where(enough, got, refs))
    s["free"].copy_(longer[:n])
    s["num_free"].copy_(left + gone.sum())
    s["shared"].copy_(shared)
    return {"storage": storage, **s}


def _plain_step(state):
    case, s, T = state["case"], state["paged"], state["tokens"]
    bs, P, group = case["block"], case["partition"], case["group"]
    tables, cached, new, free = s["tables"].long(), s["lens"].long(), state["new"].long(), s["free"].long()
    dev, B = tables.device, cached.shape[0]
    ctx = cached + new
    have, need = -(-cached // bs), -(-ctx // bs)
    starts = torch.cat([new.new_zeros(1), new.cumsum(0)])
    base = (need - have).cumsum(0) - (need - have)               # of the blocks that are taken
    j = torch.arange(tables.shape[1], device=dev)[None, :]
    added = (j >= have[:, None]) & (j < need[:, None])
    taken = free[(s["num_free"] - 1 - (base[:, None] + j - have[:, None])).clamp(0, free.shape[0] - 1)]
    s["tables"].copy_(torch.where(added, taken, tables))
    refs = torch.cat([s["refs"], s["refs"][:1]])
    refs[torch.where(added, taken, refs.shape[0] - 1).reshape(-1)] = 1
    s["refs"].copy_(refs[:-1])
    # the new tokens' rows
    t = torch.arange(T, device=dev)
    inside = t < starts[-1]
    b = torch.searchsorted(starts[1:], t, right=True).clamp(max=B - 1)
    i = t - starts[b]
    pos = torch.where(inside, cached[b] + i, 0)
    block = s["tables"].long()[b, (pos // bs).clamp(max=tables.shape[1] - 1)]
    row_ctx = torch.where(inside, pos + 1, 0)
    parts = -(-row_ctx // P)
    offsets = torch.cat([parts.new_zeros(1), parts.cumsum(0)])
    # work items: rows of one partition count, `group` at a time, an item for each partition
    since = torch.maximum((parts - 1) * P - cached[b], torch.zeros_like(i))
    leads = inside & ((i - since) % group == 0)
    size = torch.minimum(torch.minimum(torch.full_like(i, group), new[b] - i), parts * P - pos)
    count = torch.where(leads, parts, 0)
    first = count.cumsum(0) - count
    w = torch.arange(state["items"].shape[0], device=dev)
    listed_ = w < count.sum()
    r = torch.searchsorted(first + count, w, right=True).clamp(max=T - 1)
    item = torch.stack([r, b[r], (w - first[r]) | ((size[r] - 1) << 24), row_ctx[r]], 1)
    state["items"].copy_(torch.where(listed_[:, None], item, state["items"]))
    many = parts > 1
    spot = torch.where(many, many.long().cumsum(0) - 1, state["split"].shape[0])
    longer = torch.cat([state["split"], state["split"][:1]])
    longer[spot] = torch.stack([t, offsets[:-1], parts, torch.zeros_like(t)], 1).int()
    state["split"].copy_(longer[:-1])
    counts = torch.stack([count.sum(), many.sum(), torch.zeros_like(count.sum()), offsets[-1]])
    return {"tables": s["tables"], "refs": s["refs"], "num_free": (s["num_free"] - (need - have).sum()).int(),
            "lens": ctx.int(), "starts": starts.int(), "positions": pos,
            "slots": torch.where(inside, block * bs + pos % bs, -1).int(), "row_ctx": row_ctx.int(),
            "offsets": offsets.int(), "items": state["items"], "split": state["split"], "counts": counts.int()}


def _plain_attend(state):
    hq, hkv, d, _ = GEOMETRY[state["case"]["geometry"]]
    q, table = state["q"], state["tables"]
    R, P = q.shape[0], table.shape[1] * state["case"]["block"]
    kv = state["pool"][table].permute(2, 0, 3, 1, 4, 5).reshape(2, R * hkv, P, d).float()
    s = torch.bmm(q.float().reshape(R * hkv, hq // hkv, d), kv[0].transpose(1, 2).contiguous()).div_(math.sqrt(d))
    hidden = torch.arange(P, device=q.device)[None, :] >= state["lens"][:, None]
    s = s.reshape(R, hq, P).masked_fill_(hidden[:, None], -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp_()
    p = p / p.sum(-1, keepdim=True)
    return torch.bmm(p.reshape(R * hkv, hq // hkv, P), kv[1].contiguous()).reshape(R, hq * d).to(q.dtype)


# ---- 64-bit results ----------------------------------------------------------------
@torch.no_grad()
def exact(case, seed):
    if case["op"] == "select":
        return _exact_select(case, seed)
    if case["op"] == "attend":
        return _exact_attend(case, seed)
    return None                                                  # whole numbers and moved rows: nothing is computed


def _exact_select(case, seed):
    """Request by request, on the host: every continuation's log-probability, the best in order."""
    logits, scores, ended = _select_inputs(case, seed)
    K, V, M = case["beams"], case["vocab"], case["candidates"]
    told = {"scores": [], "parents": [], "tokens": []}
    for r in range(case["requests"]):
        x = logits[r * K:(r + 1) * K].double().cpu().numpy()
        total = np.full((K, V), -np.inf)
        for k in range(K):
            s = float(scores[r, k])
            if ended is not None and bool(ended[r, k]):
                total[k, 2] = s
            elif np.isfinite(x[k]).any():
                top = x[k].max()
                total[k] = s + (x[k] - (top + np.log(np.exp(x[k] - top).sum())))
        flat = total.reshape(-1)
        worst = np.partition(flat, -M)[-M] if flat.size > M else -np.inf
        at = np.nonzero(flat >= worst)[0]
        at = at[np.argsort(-flat[at], kind="stable")][:M]
        there = np.isfinite(flat[at])
        told["scores"].append(flat[at])
        told["parents"].append(np.where(there, at // V, -1))
        told["tokens"].append(np.where(there, at % V, -1))
    return {"scores": _tensor(np.stack(told["scores"]), torch.float64),
            "parents": _tensor(np.stack(told["parents"]), torch.int32), "tokens": _tensor(np.stack(told["tokens"]))}


def _exact_attend(case, seed):
    hq, hkv, d, _ = GEOMETRY[case["geometry"]]
    rep = hq // hkv
    q, pool, tables, lens = _attend_inputs(case, seed)
    out = torch.empty(q.shape[0], hq, d, dtype=torch.float64, device=q.device)
    for r, (table, n) in enumerate(zip(tables, lens)):
        blocks = pool[_tensor(table)].double()                   # [blocks, 2, hkv, block, d]
        k, v = blocks.permute(1, 2, 0, 3, 4).reshape(2, hkv, -1, d)[:, :, :n].unbind(0)
        s = (q[r].double().reshape(hkv, rep, 1, d) * k[:, None]).sum(-1) / math.sqrt(d)
        p = torch.softmax(s, -1)
        out[r] = (p[..., None] * v[:, None]).sum(2).reshape(hq, d)
    return out.reshape(-1, hq * d)
