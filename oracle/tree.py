"""Plain 64-bit forms of the operators on trees of drafted tokens (tinybatch_amd/tree.py).
The reference decodes without drafts; these restate the rules of include/tinybatch_amd.h."""
from __future__ import annotations

import math

import numpy as np
import torch


def visible(parents) -> np.ndarray:
    """[n, n] booleans: node i and its ancestors."""
    n = len(parents)
    v = np.zeros((n, n), dtype=bool)
    for i in range(n):
        j = i
        while j >= 0:
            v[i, j] = True
            j = parents[j]
    return v


def rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Rotate-half RoPE of [rows, heads, d] with fp32 tables' rows, each product rounded to fp32
    and the result to x's dtype."""
    half = x.shape[-1] // 2
    a, b = x[..., :half].float(), x[..., half:].float()
    c, s = cos[:, None, :], sin[:, None, :]
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1).to(x.dtype)


def attention(q, pool, seen, cached, tables, hq, scale=None):
    """(out, weight, spread) in 64 bits, [rows, hq, d] each but for spread [rows, hq]: the attention of
    every node, the sum of p |v| (what a relative error of the weights acts on), and the largest
    sum_d |q_d k_d| |scale| of a row's scores. seen[b]: [n, n] booleans. Positions a node does not see
    are left out of the sums."""
    nb, _, hkv, bs, d = pool.shape
    rep = hq // hkv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    rows = sum(s.shape[0] for s in seen)
    out, weight = torch.zeros(rows, hq, d, dtype=torch.float64), torch.zeros(rows, hq, d, dtype=torch.float64)
    spread = torch.zeros(rows, hq, dtype=torch.float64)
    at = 0
    for sees, c, table in zip(seen, cached, tables):
        n = sees.shape[0]
        pos = torch.arange(c + n)
        kv = pool[torch.as_tensor(list(table), dtype=torch.int64)[pos // bs], :, :, pos % bs].double()   # [P, 2, hkv, d]
        for i in range(n):
            keep = torch.cat([torch.ones(c, dtype=torch.bool), torch.from_numpy(sees[i].copy())])
            if not keep.any():
                continue
            k = kv[keep, 0].repeat_interleave(rep, dim=1)
            v = kv[keep, 1].repeat_interleave(rep, dim=1)
            x = q[at + i].double()
            p = torch.softmax((k * x[None]).sum(-1) * scale, dim=0)[:, :, None]
            out[at + i] = (p * v).sum(0)
            weight[at + i] = (p * v.abs()).sum(0)
            spread[at + i] = (k * x[None]).abs().sum(-1).max(0).values * abs(scale)
        at += n
    return out, weight, spread


def verify(parents, tokens, uniforms, probs, draft=None):
    """The walk as it is told, in numpy float64: (path, emitted tokens) of one sequence. The residual
    distribution is kept normalised, one refusal after the other."""
    p_all = np.asarray(probs, dtype=np.float64)
    node, path, told = 0, [0], []
    while True:
        whole = np.where(p_all[node] > 0, p_all[node], 0.0)
        rest, left, took = whole.copy(), 1.0, None
        for child in [i for i in range(1, len(parents)) if parents[i] == node]:
            t, u = int(tokens[child]), float(uniforms[child])
            known = 0 <= t < rest.size
            if draft is None:
                ok = known and rest[t] > 0 and u * left < rest[t]
            else:
                q = np.asarray(draft[node], dtype=np.float64)
                ok = known and u * q[t] < rest[t]
            if ok:
                took = child
                break
            if draft is None:
                if known:
                    left -= rest[t]
                    rest[t] = 0.0
            else:
                rest = np.maximum(rest - q, 0.0)
                if rest.sum() > 0:
                    rest = rest / rest.sum()
        if took is None:
            break
        node = took
        path.append(node)
        told.append(int(tokens[node]))
    if not rest.sum() > 0:
        rest = whole
    cum = np.cumsum(rest)
    if not cum[-1] > 0:
        told.append(-1)
    else:
        last = int(np.flatnonzero(rest > 0)[-1])
        told.append(min(int((cum <= float(uniforms[0]) * cum[-1]).sum()), last))
    return path, told
