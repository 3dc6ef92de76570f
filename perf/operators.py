"""What is measured of the operators of speculative decoding: a step's drafted tokens form
a tree (a chain is the tree of one child each) that hangs below the last token a sequence
has emitted. Three operators serve the step:

* ``attend``: every node's attention over the sequence's cached positions and over its own
  ancestors among the step's nodes, whose K/V lie in the pages behind the cached ones
  (``tree_attention``);
* ``verify``: which drafted tokens the target's probabilities keep, by given random numbers,
  and the token that follows them (``verify_tree``), with the probabilities that the drafts
  were drawn from or without (drafts that were not drawn at random);
* ``commit``: the kept nodes' K/V rows moved to the positions they now have, in every layer
  (``commit_tree``).

Tree shapes and lengths are drawn from the case alone (``lengths`` seeds them), so that a
case is the same work for every seed of its inputs.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
# query heads, kv heads, head dim
GEOMETRY = {"qwen": (14, 2, 64), "llama": (32, 8, 128), "mqa": (12, 1, 64), "mha": (5, 5, 128)}


def _attend(name, geometry, dtype, seqs, nodes, shape, cached, block=16, lengths=1):
    return {"name": name, "op": "attend", "geometry": geometry, "dtype": dtype, "seqs": seqs, "nodes": nodes,
            "shape": shape, "cached": cached, "block": block, "lengths": lengths}


def _verify(name, dtype, seqs, nodes, shape, vocab, drafts, lengths=1):
    return {"name": name, "op": "verify", "dtype": dtype, "seqs": seqs, "nodes": nodes, "shape": shape,
            "vocab": vocab, "drafts": drafts, "lengths": lengths}


def _commit(name, geometry, dtype, layers, seqs, nodes, shape, cached, block=16, lengths=1):
    return {"name": name, "op": "commit", "geometry": geometry, "dtype": dtype, "layers": layers, "seqs": seqs,
            "nodes": nodes, "shape": shape, "cached": cached, "block": block, "lengths": lengths}


def listed():
    return [
        # one user's request some way into its answer, four drafted tokens in a row: latency
        _attend("attend bf16 one chain", "qwen", "bfloat16", 1, "5:5", "chain", "600:600", lengths=1),
        # the parity precision: a few short requests with small trees
        _attend("attend fp32 small trees", "qwen", "float32", 8, "7:13", "tree", "29:900", lengths=2),
        # a serving batch with trees of the usual size, contexts of the headline decode step
        _attend("attend fp16 32 trees", "qwen", "float16", 32, "20:30", "tree", "512:4096", lengths=3),
        # a large batch at the 8B geometry, short chains over long contexts: the cache's bytes count
        _attend("attend bf16 8B chains long", "llama", "bfloat16", 48, "4:8", "chain",
                "lognormal:8192:0.5:1024:32768", lengths=4),
        # large trees at the 8B geometry: the products count
        _attend("attend bf16 8B trees of 64", "llama", "bfloat16", 16, "60:64", "tree", "1000:8000", lengths=5),
        # one user's chain drawn from a draft model
        _verify("verify one chain", "float32", 1, "6:6", "chain", 151936, True, lengths=6),
        # one user's tree of a draft model's most likely tokens
        _verify("verify one tree top-k", "float32", 1, "60:60", "tree", 151936, False, lengths=7),
        # a serving batch of chains drawn from a draft model
        _verify("verify 64 chains", "float32", 64, "4:6", "chain", 151936, True, lengths=8),
        # a batch of trees whose children were drawn from a draft model: several rounds a node
        _verify("verify 16 trees drawn", "float32", 16, "12:20", "tree", 151936, True, lengths=9),
        # a serving batch of top-k trees, the probabilities kept in 16 bits
        _verify("verify 32 trees top-k bf16", "bfloat16", 32, "20:30", "tree", 128256, False, lengths=10),
        # one user's accepted path in a small model's layers
        _commit("commit one tree", "qwen", "bfloat16", 24, 1, "26:26", "tree", "600:600", lengths=11),
        # a serving batch's paths in the layers of the 8B geometry
        _commit("commit 64 trees 8B", "llama", "bfloat16", 32, 64, "20:60", "tree", "20:90", lengths=12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """A case of the ranges above: other batches, trees, contexts, vocabularies, geometries
    and types, each no more work than the largest above of its kind."""
    lengths = rng.randrange(1, 1 << 20)
    shape = rng.choice(["chain", "tree", "tree"])
    n_hi = _log_int(rng, 1, 12) if shape == "chain" else _log_int(rng, 4, 100)
    n_lo = max(1, n_hi // rng.randint(1, 4))
    op = rng.choice(["attend", "attend", "verify", "verify", "commit"])
    if op == "attend":
        g = rng.choice(["qwen", "qwen", "llama", "llama", "mqa", "mha"])
        hq, hkv, d = GEOMETRY[g]
        dt = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
        c_hi = _log_int(rng, 17, 16000)
        # positions times query rows bounded: by the products of the largest case, in fp32 less
        most = (2_000_000_000 if dt != "float32" else 150_000_000) // (hq * d * n_hi)
        seqs = max(1, min(_log_int(rng, 1, 64), most // c_hi, 400_000 // c_hi))
        c = _attend("", g, dt, seqs, f"{n_lo}:{n_hi}", shape, f"{rng.choice([0, c_hi // 8, c_hi // 2])}:{c_hi}",
                    block=rng.choice([16, 16, 32]), lengths=lengths)
    elif op == "verify":
        n_hi = min(n_hi, 60)
        vocab = rng.choice([151936, 128256, 50257, 32001, 32000])
        drafts = rng.random() < 0.5
        seqs = max(1, min(_log_int(rng, 1, 64), (800 if not drafts else 320) // n_hi))
        c = _verify("", rng.choice(["float32", "float32", "float16", "bfloat16"]), seqs, f"{min(n_lo, n_hi)}:{n_hi}",
                    shape, vocab, drafts, lengths=lengths)
    else:
        g = rng.choice(["qwen", "llama", "mqa"])
        c = _commit("", g, rng.choice(["bfloat16", "float16", "float32"]), rng.randint(1, 16),
                    _log_int(rng, 1, 64), f"{n_lo}:{n_hi}", shape, "0:90", block=rng.choice([16, 16, 32]),
                    lengths=lengths)
    c.pop("name")
    return c


# ---- what a case's sizes come to ------------------------------------------------
def _draws(rng, spec, n):
    if spec.startswith("lognormal:"):
        median, sigma, lo, hi = (float(x) for x in spec.split(":")[1:])
        return [int(min(hi, max(lo, round(median * math.exp(sigma * rng.gauss(0, 1)))))) for _ in range(n)]
    lo, hi = (int(x) for x in spec.split(":"))
    return [rng.randint(lo, hi) for _ in range(n)]


def _trees(case):
    """Each sequence's tree, as the parents of its nodes: node 0 is the root (parent -1)."""
    rng = random.Random(case["lengths"])
    sizes = _draws(rng, case["nodes"], case["seqs"])
    if case["shape"] == "chain":
        return [list(range(-1, n - 1)) for n in sizes]
    return [[-1] + [rng.randrange(i) for i in range(1, n)] for n in sizes]


def _cached(case):
    return _draws(random.Random(case["lengths"] + 1), case["cached"], case["seqs"])


def _paths(case):
    """A path from the root in each tree: the nodes that a verification kept."""
    rng = random.Random(case["lengths"] + 2)
    paths = []
    for parents in _trees(case):
        node, path = rng.randrange(len(parents)), []
        while node >= 0:
            path.append(node)
            node = parents[node]
        paths.append(path[::-1])
    return paths


def _depths(parents):
    d = []
    for p in parents:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def work(case):
    trees = _trees(case)
    if case["op"] == "verify":
        # the row that the next token is drawn from, and the draft's row where there is one
        rows = case["seqs"] * (2 if case["drafts"] else 1)
        return {"bytes": rows * case["vocab"] * DTYPES[case["dtype"]].itemsize, "flops": 0}
    hq, hkv, d = GEOMETRY[case["geometry"]]
    b = DTYPES[case["dtype"]].itemsize
    if case["op"] == "commit":
        moved = sum(1 for path in _paths(case) for j, i in enumerate(path) if i != j)
        return {"bytes": max(1, moved) * case["layers"] * 2 * 2 * hkv * d * b, "flops": 0}
    rows = sum(len(t) for t in trees)
    kv = sum(c + len(t) for c, t in zip(_cached(case), trees))
    pairs = sum(len(t) * c + sum(x + 1 for x in _depths(t)) for c, t in zip(_cached(case), trees))
    return {"bytes": kv * 2 * hkv * d * b + 2 * rows * hq * d * b, "flops": 4 * hq * d * pairs}


# ---- inputs -----------------------------------------------------------------------
def _dev():
    return torch.device("cuda", torch.cuda.current_device())


def _generator(seed):
    return torch.Generator(device=_dev()).manual_seed(int(seed))


def _tensor(values, dtype=torch.int64):
    return torch.tensor(values, dtype=dtype, device=_dev())


def _tables(case):
    """Block tables over a shuffled pool, and the pool's size (1 in 16 of it unused)."""
    need = [-(-(c + len(t)) // case["block"]) for c, t in zip(_cached(case), _trees(case))]
    total = sum(need) + sum(need) // 16 + 1
    ids = list(range(total))
    random.Random(case["lengths"] + 3).shuffle(ids)
    tables, at = [], 0
    for k in need:
        tables.append(ids[at:at + k])
        at += k
    return tables, total


def _padded(rows, fill=0):
    width = max(len(r) for r in rows)
    return [list(r) + [fill] * (width - len(r)) for r in rows]


def _starts(trees):
    at = [0]
    for t in trees:
        at.append(at[-1] + len(t))
    return at


def _attend_inputs(case, seed):
    """q [rows, hq, d] and the pool [blocks, 2, hkv, block, d], the nodes' K/V in it."""
    g = _generator(seed)
    hq, hkv, d = GEOMETRY[case["geometry"]]
    dt = DTYPES[case["dtype"]]
    tables, blocks = _tables(case)
    q = torch.randn(sum(len(t) for t in _trees(case)), hq, d, generator=g, device=_dev()).to(dt)
    pool = torch.empty(blocks, 2, hkv, case["block"], d, device=_dev(), dtype=dt).normal_(generator=g)
    return q, pool, tables


def _verify_inputs(case, seed):
    """The target's probabilities [rows, vocab], the draft's or None, the nodes' tokens and
    the random numbers: peaked distributions, the draft's a disturbed copy of the target's."""
    g = _generator(seed)
    trees = _trees(case)
    rows, vocab, dev = sum(len(t) for t in trees), case["vocab"], _dev()
    dt = DTYPES[case["dtype"]]
    logits = torch.randn(rows, vocab, generator=g, device=dev) * 5
    probs = torch.softmax(logits, dim=-1).to(dt)
    logits += torch.randn(rows, vocab, generator=g, device=dev)
    starts = _starts(trees)
    parent_row = _tensor([starts[b] + max(p, 0) for b, t in enumerate(trees) for p in t])
    rank = _tensor([t[:i].count(p) if p >= 0 else 0 for t in trees for i, p in enumerate(t)])
    if case["drafts"]:
        draft = torch.softmax(logits, dim=-1).to(dt)
        drawn = torch.multinomial(draft.float(), int(rank.max()) + 1, replacement=True, generator=g)
    else:
        draft, drawn = None, logits.topk(int(rank.max()) + 1, dim=-1).indices
    tokens = drawn[parent_row, rank]
    uniforms = torch.rand(rows, generator=g, device=dev)
    return probs, draft, tokens, uniforms


def _commit_inputs(case, seed):
    g = _generator(seed)
    hq, hkv, d = GEOMETRY[case["geometry"]]
    tables, blocks = _tables(case)
    storage = torch.empty(case["layers"], blocks, 2, hkv, case["block"], d, device=_dev(), dtype=DTYPES[case["dtype"]])
    for layer in storage:
        layer.normal_(generator=g)
    return storage, tables


def _metadata(case, tables=None, blocks=0):
    from tinybatch_amd import build_tree_metadata

    if tables is None:
        return build_tree_metadata(_trees(case)).to(_dev())
    hq, hkv, d = GEOMETRY[case["geometry"]]
    return build_tree_metadata(_trees(case), _cached(case), tables, block_size=case["block"], num_blocks=blocks,
                               num_heads=hq, num_kv_heads=hkv, head_dim=d, dtype=DTYPES[case["dtype"]]).to(_dev())


@torch.no_grad()
def prepare(case, seed):
    """The inputs, and the step's plan: with ``own`` the framework's, otherwise index tensors."""
    trees = _trees(case)
    state = {"case": case}
    if case["op"] == "verify":
        state["probs"], state["draft"], state["tokens"], state["uniforms"] = _verify_inputs(case, seed)
        state.update({"meta": _metadata(case)} if own else _verify_plan(trees))
        return state
    cached = _cached(case)
    if case["op"] == "commit":
        state["storage"], tables = _commit_inputs(case, seed)
        paths = _paths(case)
        state["accepted"] = _tensor([p + [-1] * (max(map(len, trees)) - len(p)) for p in paths], torch.int32)
        state["count"] = _tensor([len(p) for p in paths], torch.int32)
        if own:
            state["meta"] = _metadata(case, tables, state["storage"].shape[1])
        else:
            state["tables"], state["cached"] = _tensor(_padded(tables)), _tensor(cached)
        return state
    state["q"], state["pool"], tables = _attend_inputs(case, seed)
    if own:
        state["meta"] = _metadata(case, tables, state["pool"].shape[0])
    else:
        state.update(_attend_plan(case, trees, cached, tables))
    return state


@torch.no_grad()
def run(state):
    case = state["case"]
    if own:
        from tinybatch_amd import commit_tree, tree_attention, verify_tree

        if case["op"] == "attend":
            return tree_attention(state["q"], state["pool"], state["meta"])
        if case["op"] == "verify":
            v = verify_tree(state["meta"], state["tokens"], state["uniforms"], state["probs"], state["draft"])
            return {"accepted": v.accepted, "count": v.num_accepted, "tokens": v.tokens}
        commit_tree(state["storage"], state["meta"], state["accepted"], state["count"])
        return state["storage"]
    if case["op"] == "attend":
        return _plain_attend(state)
    if case["op"] == "verify":
        return _plain_verify(state)
    return _plain_commit(state)


# ---- plain forms ------------------------------------------------------------------
def _ancestors(parents, width):
    """[n, width]: node i's ancestors and itself."""
    rows = []
    for i, p in enumerate(parents):
        row = list(rows[p]) if p >= 0 else [False] * width
        row[i] = True
        rows.append(row)
    return rows


def _attend_plan(case, trees, cached, tables):
    """The sequences padded to one length: tables [B, blocks], hidden [B, nodes, positions]
    (not among a node's cached positions and ancestors), the rows' places in [B, nodes]."""
    width = max(len(t) for t in trees)
    visible = torch.zeros(len(trees), width, width, dtype=torch.bool)
    for b, t in enumerate(trees):
        visible[b, :len(t)] = torch.tensor(_ancestors(t, width))
    table = _tensor(_padded(tables))
    n = _tensor([len(t) for t in trees])
    c = _tensor(cached)
    pos = torch.arange(table.shape[1] * case["block"], device=_dev())
    node = pos[None, :] - c[:, None]                            # which node a position holds
    seen = torch.gather(visible.to(_dev()), 2,
                        node.clamp(0, width - 1)[:, None, :].expand(-1, width, -1))
    seen &= (node < n[:, None])[:, None, :]
    hidden = ~(seen | (node < 0)[:, None, :])
    place = torch.arange(width, device=_dev())[None, :] < n[:, None]
    return {"table": table, "hidden": hidden, "place": place.nonzero(as_tuple=True)}


def _plain_attend(state):
    hq, hkv, d = GEOMETRY[state["case"]["geometry"]]
    rep = hq // hkv
    hidden, (seq, node) = state["hidden"], state["place"]
    B, N, P = hidden.shape
    kv = state["pool"][state["table"]].permute(2, 0, 3, 1, 4, 5).reshape(2, B * hkv, P, d).float()
    q = torch.zeros(B, N, hq, d, device=kv.device)
    q[seq, node] = state["q"].float()
    q = q.reshape(B, N, hkv, rep, d).permute(0, 2, 3, 1, 4).reshape(B * hkv, rep * N, d)
    s = torch.bmm(q, kv[0].transpose(1, 2).contiguous()).div_(math.sqrt(d)).reshape(B, hkv * rep, N, P)
    s.masked_fill_(hidden[:, None], -math.inf)
    p = (s - s.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    p = p / p.sum(-1, keepdim=True)
    o = torch.bmm(p.reshape(B * hkv, rep * N, P), kv[1].contiguous())
    o = o.reshape(B, hkv, rep, N, d).permute(0, 3, 1, 2, 4).reshape(B, N, hq * d)
    return o[seq, node].to(state["q"].dtype)


def _verify_plan(trees):
    starts = _starts(trees)
    rows = starts[-1]
    parent, rank, seq = [], [], []
    path = torch.zeros(rows, rows, dtype=torch.bool)            # ancestors and itself, without the root
    earlier = torch.zeros(rows, rows, dtype=torch.bool)         # earlier children of the same parent
    for b, t in enumerate(trees):
        s = starts[b]
        path[s:s + len(t), s:s + len(t)] = torch.tensor(_ancestors(t, len(t)))
        path[s:s + len(t), s] = False
        siblings = {}
        for i, p in enumerate(t):
            before = siblings.setdefault(p, [])
            parent.append(s + p if p >= 0 else s)
            rank.append(len(before) if p >= 0 else -1)
            earlier[s + i, before] = True
            before.append(s + i)
            seq.append(b)
    ranks = torch.tensor(rank)
    return {"parent": _tensor(parent), "path": path.to(_dev()), "earlier": earlier.to(_dev()),
            "root": _tensor([r < 0 for r in rank], torch.bool), "seq": _tensor(seq), "start": _tensor(starts[:-1]),
            "by_rank": [(ranks == r).nonzero()[:, 0].to(_dev()) for r in range(int(ranks.max()) + 1)],
            "width": max(len(t) for t in trees)}


def _plain_verify(state):
    """Every node's test as if its parent were reached and its earlier siblings refused; a node
    is on the path where it and all its ancestors are the first of their siblings to pass."""
    probs, draft, tokens, u = state["probs"], state["draft"], state["tokens"], state["uniforms"].double()
    parent, earlier, root, start = state["parent"], state["earlier"], state["root"], state["start"]
    rows, vocab = probs.shape
    B, width = start.shape[0], state["width"]
    p = probs[parent, tokens].double()
    again = (earlier & (tokens[:, None] == tokens[None, :])).any(1)
    if draft is None:
        # a refused sibling's token leaves the distribution: what it held is gone from the whole
        p = p.masked_fill(again, 0.0)
        left = 1.0 - (earlier * p[None, :]).sum(1)
        passes = (p > 0) & (u * left < p)
    else:
        # after m refusals the distribution is max(p - a q, 0) / s with a = sum of the earlier s
        qv = draft[parent, tokens].double()
        a = torch.zeros(rows, dtype=torch.float64, device=probs.device)
        s = torch.ones_like(a)
        passes = torch.zeros(rows, dtype=torch.bool, device=probs.device)
        for nodes in state["by_rank"]:
            at = parent[nodes]
            passes[nodes] = u[nodes] * qv[nodes] * s[at] < p[nodes] - a[at] * qv[nodes]
            a[at] = a[at] + s[at]
            s[at] = (probs[at].double() - a[at, None] * draft[at].double()).clamp_(min=0).sum(1)
    taken = (passes & ~(earlier & passes[None, :]).any(1)) | root
    reached = (taken[None, :] | ~state["path"]).all(1)
    # the path's nodes in order: a node's ancestors come before it
    index = torch.arange(rows, device=probs.device)
    order = (state["path"] & reached[None, :]).sum(1)           # how deep a reached node lies
    count = torch.zeros(B, dtype=torch.int64, device=probs.device).index_add_(0, state["seq"], reached.long())
    last = torch.zeros_like(count).scatter_reduce_(0, state["seq"], torch.where(reached, index, -1), "amax")
    accepted = torch.full((B, width + 1), -1, dtype=torch.int64, device=probs.device)
    out = torch.full((B, width + 1), -1, dtype=torch.int64, device=probs.device)
    spare = torch.full_like(order, width)                       # nodes off the path write a spare column
    accepted[state["seq"], torch.where(reached, order, spare)] = index - start[state["seq"]]
    out[state["seq"], torch.where(reached & ~root, order - 1, spare)] = tokens
    # the token after the path, from what its last node's refused children leave
    whole = probs[last].double()
    children = (parent[None, :] == last[:, None]) & ~root[None, :]
    if draft is None:
        gone = torch.zeros_like(whole).scatter_add_(
            1, tokens[None, :].expand(B, -1), children.double())
        w = whole.masked_fill(gone > 0, 0.0)
    else:
        w = (whole - a[last, None] * draft[last].double()).clamp_(min=0)
    total = w.sum(1, keepdim=True)
    w = torch.where(total > 0, w, whole)
    cum = w.cumsum(1)
    nxt = (cum <= u[start, None] * cum[:, -1:]).sum(1).clamp_(max=vocab - 1)
    out[torch.arange(B, device=probs.device), count - 1] = nxt
    return {"accepted": accepted[:, :width].int(), "count": count.int(), "tokens": out[:, :width].contiguous()}


def _plain_commit(state):
    storage, accepted, count = state["storage"], state["accepted"].long(), state["count"]
    block = state["case"]["block"]
    j = torch.arange(accepted.shape[1], device=storage.device)[None, :]
    kept = j < count[:, None]
    to = state["cached"][:, None] + torch.where(kept, j, 0)
    frm = state["cached"][:, None] + torch.where(kept, accepted, 0)
    table = state["table"] if "table" in state else state["tables"]
    rows = storage[:, table.gather(1, frm // block), :, :, frm % block]
    storage[:, table.gather(1, to // block), :, :, to % block] = rows
    return storage


# ---- 64-bit results ----------------------------------------------------------------
@torch.no_grad()
def exact(case, seed):
    if case["op"] == "attend":
        return _exact_attend(case, seed)
    if case["op"] == "verify":
        return _exact_verify(case, seed)
    return None                                                  # rows are moved, nothing is computed


def _exact_attend(case, seed):
    hq, hkv, d = GEOMETRY[case["geometry"]]
    rep = hq // hkv
    q, pool, tables = _attend_inputs(case, seed)
    out = torch.empty(q.shape[0], hq, d, dtype=torch.float64, device=q.device)
    row = 0
    for parents, c, table in zip(_trees(case), _cached(case), tables):
        n = len(parents)
        blocks = pool[_tensor(table)].double()
        for h in range(hkv):
            k = blocks[:, 0, h].reshape(-1, d)[:c + n]
            v = blocks[:, 1, h].reshape(-1, d)[:c + n]
            for i0 in range(0, n, 16):
                i1 = min(n, i0 + 16)
                hide = torch.ones(i1 - i0, c + n, dtype=torch.bool)
                for i in range(i0, i1):
                    hide[i - i0, :c] = False
                    node = i
                    while node >= 0:
                        hide[i - i0, c + node] = False
                        node = parents[node]
                qs = q[row + i0:row + i1, h * rep:(h + 1) * rep].double()
                s = torch.tensordot(qs, k, dims=([2], [1])) * (1.0 / math.sqrt(d))
                s[hide.to(q.device)[:, None, :].expand_as(s)] = -math.inf
                out[row + i0:row + i1, h * rep:(h + 1) * rep] = torch.tensordot(torch.softmax(s, -1), v, dims=([2], [0]))
        row += n
    return out.reshape(-1, hq * d)


def _exact_verify(case, seed):
    """The rule as it is told: from the root on, try a reached node's children in order."""
    probs, draft, tokens, uniforms = _verify_inputs(case, seed)
    tok, u = tokens.tolist(), uniforms.tolist()
    trees = _trees(case)
    width = max(len(t) for t in trees)
    accepted, out, counts = [], [], []
    for parents, s in zip(trees, _starts(trees)):
        path, told, node = [0], [], 0
        while True:
            p = probs[s + node].double()
            rest, took = p.clone(), None
            for child in [i for i, x in enumerate(parents) if x == node and i > 0]:
                t = tok[s + child]
                if draft is None:
                    # `rest` sums to 1 less what refused tokens held
                    ok = float(rest[t]) > 0 and u[s + child] * (1.0 - float((p - rest).sum())) < float(rest[t])
                else:
                    q = draft[s + node].double()
                    ok = u[s + child] * float(q[t]) < float(rest[t])
                if ok:
                    took = child
                    break
                if draft is None:
                    rest[t] = 0.0
                else:
                    rest = (rest - q).clamp(min=0)
                    if float(rest.sum()) > 0:
                        rest = rest / rest.sum()
            if took is None:
                break
            node = took
            path.append(node)
            told.append(tok[s + node])
        if not float(rest.sum()) > 0:
            rest = probs[s + node].double()
        cum = rest.cumsum(0)
        told.append(min(int((cum <= u[s] * cum[-1]).sum()), case["vocab"] - 1))
        counts.append(len(path))
        accepted.append(path + [-1] * (width - len(path)))
        out.append(told + [-1] * (width - len(told)))
    return {"accepted": _tensor(accepted, torch.int32), "count": _tensor(counts, torch.int32), "tokens": _tensor(out)}
