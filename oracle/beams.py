"""Plain forms of beam search's operators and of steps built from lengths, in lists and 64 bits.

No counterpart in the reference; the rules are those of include/tinybatch_amd.h (tb_device_step,
tb_beam_select, tb_beam_reorder, tb_beam_attention)."""
from __future__ import annotations

import copy
import math

import numpy as np


class State:
    """Rows' block tables, lengths, reference counts and free blocks (handed out from the end)."""

    def __init__(self, tables, lens, free, num_blocks, block_size, beams, held=()):
        self.tables = [list(t[:-(-n // block_size)]) for t, n in zip(tables, lens)]
        self.lens, self.free, self.bs, self.beams, self.nb = list(lens), list(free), block_size, beams, num_blocks
        self.refs = [0] * num_blocks
        for t in self.tables:
            for b in t:
                self.refs[b] += 1
        for b in held:
            self.refs[b] += 1

    def clone(self):
        return copy.deepcopy(self)

    def shared(self):
        """Leading whole blocks that a request's rows with positions have in common."""
        out = []
        for g in range(0, len(self.lens), self.beams):
            live = [r for r in range(g, g + self.beams) if self.lens[r] > 0]
            n = min((self.lens[r] // self.bs for r in live), default=0)
            k = 0
            while k < n and len({self.tables[r][k] for r in live}) == 1:
                k += 1
            out.append(k)
        return out


def step(state: State, new_lens, padded=0):
    """The state with the new tokens' blocks, and (starts, positions, slots, row_ctx) of the flat rows."""
    s, starts, positions, slots, ctx = state.clone(), [0], [], [], []
    for b, n in enumerate(new_lens):
        for i in range(n):
            p = s.lens[b] + i
            if p // s.bs == len(s.tables[b]):
                blk = s.free.pop()
                s.tables[b].append(blk)
                s.refs[blk] = 1
            positions.append(p)
            slots.append(s.tables[b][p // s.bs] * s.bs + p % s.bs)
            ctx.append(p + 1)
        for _ in range(padded - n if padded else 0):
            positions.append(0), slots.append(-1), ctx.append(0)
        starts.append(len(positions))
    s.lens = [c + n for c, n in zip(s.lens, new_lens)]
    return s, starts, positions, slots, ctx


def reorder(state: State, parents):
    """(the state after, copies): copies as (source block, fresh block, positions)."""
    s, K, bs = state.clone(), state.beams, state.bs
    copies, tables, lens = [], [], []
    for r in range(len(s.lens)):
        g, p = r // K * K, parents[r]
        src = g + p
        if p < 0 or s.lens[src] == 0:
            tables.append([]), lens.append(0)
            continue
        n, t = s.lens[src], list(state.tables[src])
        if n % bs:
            open_block = t[n // bs]
            if not (p not in parents[g:r] and state.refs[open_block] == 1):
                t[n // bs] = s.free.pop()
                s.refs[t[n // bs]] = 1
                copies.append((open_block, t[n // bs], n % bs))
        tables.append(t), lens.append(n)
    fresh = {c[1] for c in copies}
    for t in state.tables:
        for b in t:
            s.refs[b] -= 1
    for t in tables:
        for b in t:
            s.refs[b] += b not in fresh
    gone = []
    for g in range(0, len(s.lens), K):
        rows = state.tables[g:g + K]
        for j in range(max(map(len, rows))):
            for t in rows:
                if j < len(t) and s.refs[t[j]] == 0 and t[j] not in gone:
                    gone.append(t[j])
    s.free += gone
    s.tables, s.lens = tables, lens
    return s, copies


def select(logits, scores, picks, finished=None, end_token=-1):
    """(scores, parents, tokens) [G, M] of float64 logits [G * K, V] and scores [G, K]. Among equal scores the smaller
    beam first, within a beam the larger logit (scores, rounded, may be equal where logits are not), then the smaller token."""
    G, K = scores.shape
    V = logits.shape[1]
    top = float(np.finfo(np.float32).max)
    out = np.full((G, picks), -np.inf), np.full((G, picks), -1), np.full((G, picks), -1)
    for g in range(G):
        c, logit = np.full((K, V), -np.inf), np.zeros((K, V))
        for k in range(K):
            s = float(scores[g, k])
            if finished is not None and finished[g, k]:
                if s > -math.inf:
                    c[k, end_token] = s
            elif s > -math.inf:
                x = np.minimum(np.where(np.isnan(logits[g * K + k]), -np.inf, logits[g * K + k]), top)
                m = x.max()
                if m > -math.inf:
                    c[k] = s + ((x - m) - np.log(np.exp(x - m).sum()))
                    logit[k] = x
        flat = c.reshape(-1)
        at = np.lexsort((-logit.reshape(-1), np.arange(K * V) // V, -flat))[:picks]
        at = at[flat[at] > -np.inf]
        out[0][g, :len(at)], out[1][g, :len(at)], out[2][g, :len(at)] = flat[at], at // V, at % V
    return out


def attention(q, pool, tables, lens, heads, scale=None):
    """[R, heads * D] in 64 bits, with the weights' and scores' sizes (for tolerances): row r over the first
    lens[r] positions of tables[r]; 0 for a row without positions."""
    R, d = len(lens), pool.shape[-1]
    hkv, bs = pool.shape[2], pool.shape[3]
    rep = heads // hkv
    scale = 1 / math.sqrt(d) if scale is None else scale
    out, weight, spread = np.zeros((R, heads, d)), np.zeros((R, heads, d)), np.zeros((R, heads))
    q = q.reshape(R, heads, d).astype(np.float64)
    for r, n in enumerate(lens):
        if n == 0:
            continue
        kv = np.concatenate([pool[b] for b in tables[r][:-(-n // bs)]], axis=2)[:, :, :n].astype(np.float64)
        for h in range(heads):
            k, v = kv[0, h // rep], kv[1, h // rep]
            s = scale * (k @ q[r, h])
            p = np.exp(s - s.max())
            p /= p.sum()
            out[r, h], weight[r, h] = p @ v, p @ np.abs(v)
            spread[r, h] = (abs(scale) * np.abs(k) @ np.abs(q[r, h])).max()
    return out, weight, spread
