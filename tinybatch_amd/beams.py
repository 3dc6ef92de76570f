"""Beam search over the paged cache, without the host between two steps.

The reference decodes one continuation per request (src/tinybatch/engine.py:99-159). Here a request
has ``group_size`` rows, its beams, whose paged state lives on the GPU (DeviceTables):

    build_device_step(tables, live, step)                        # one token per live beam (1; ended or lost: 0)
    plan.build(step.row_ctx)                                     # a BeamPlan, for all layers
    for layer in range(n_layers):
        ops.kv_append(cache.pools[layer], k, v, step.slot_mapping)
        attn = beam_attention(q, cache.pools[layer], plan)
    choice = select_beams(logits, scores, finished=finished, end_token=eos)
    reorder_beams(cache.storage, tables, choice.parents, step=step)
    # finished and live follow choice.parents and choice.tokens (BeamState.advance in beam_search.py)

Everything is enqueued on the tensors' device's current stream and nothing synchronises.
"""
from __future__ import annotations

import functools
import math
from typing import NamedTuple

import torch

from . import _lib
from .device_tables import MAX_BEAMS, DeviceStep, DeviceTables, _ints
from .ops import _check_pool, _rows_view
from .tree import _elsewhere, _scratch

MAX_CANDIDATES = 128         # TB_BEAM_CANDIDATES_MAX


class BeamChoice(NamedTuple):
    """A request's best continuations, best first, on the device."""
    scores: torch.Tensor     # [G, M] float32, -inf where no candidate is left
    parents: torch.Tensor    # [G, M] int32: the beam that is continued, -1 where none is left
    tokens: torch.Tensor     # [G, M] int64: with which token, -1 where none is left


def select_beams(logits: torch.Tensor, scores: torch.Tensor, *, num_candidates: int | None = None,
                 finished: torch.Tensor | None = None, end_token: int = -1) -> BeamChoice:
    """The ``num_candidates`` (by default as many as beams) best continuations of every request
    (tb_beam_select): candidate (k, v) is worth scores[g, k] + log_softmax(logits[g * K + k])[v]; among
    equals the smaller k first, within a beam the larger logit, then the smaller v.

    logits [G * K, vocab] (fp32, fp16 or bf16, contiguous rows); scores [G, K] float32, the beams' sums of
    log-probabilities (-inf: no beam). ``finished`` [G, K] bool: a beam that has ended stands for itself
    alone, with ``end_token`` at its score. NaN logits count as -inf.
    """
    _lib.require_gpu_tensor("logits", logits)
    device, code, shape = logits.device, _lib.DTYPE_CODE.get(logits.dtype), scores.shape
    if code is None:
        raise TypeError(f"unsupported logits dtype {logits.dtype}")
    if len(shape) != 2 or not 1 <= shape[1] <= MAX_BEAMS:
        raise ValueError(f"scores must be [requests, beams] with 1 .. {MAX_BEAMS} beams, got {tuple(shape)}")
    G, K = shape
    _ints("scores", scores, torch.float32, (G, K), device)
    rows, vocab = logits.shape if logits.dim() == 2 else (-1, 0)
    if rows != G * K or vocab < 1 or logits.stride(1) != 1:
        raise ValueError(f"logits must be [{G * K}, vocab] with contiguous rows, got {tuple(logits.shape)}")
    stride = logits.stride(0) if rows > 1 else vocab
    if stride < vocab:
        raise ValueError("logits' rows overlap")
    M = K if num_candidates is None else num_candidates
    if not 1 <= M <= MAX_CANDIDATES:
        raise ValueError(f"num_candidates must lie within 1 .. {MAX_CANDIDATES}")
    if vocab > 1 << 30 or rows > 65535:
        raise ValueError(f"{rows} rows of a vocabulary of {vocab}: at most 65535 and 2^30 are served")
    if finished is not None:
        _ints("finished", finished, torch.bool, (G, K), device)
        if not 0 <= end_token < vocab:
            raise ValueError(f"end_token {end_token} outside the vocabulary of {vocab}")
    if _elsewhere(device):
        with torch.cuda.device(device):
            return select_beams(logits, scores, num_candidates=M, finished=finished, end_token=end_token)
    best = torch.empty(G, M, dtype=torch.float32, device=device)
    parents = torch.empty(G, M, dtype=torch.int32, device=device)
    tokens = torch.empty(G, M, dtype=torch.int64, device=device)
    L, stream, need = _lib.lib(), _lib.stream_handle(device), _select_bytes(rows, vocab, M)
    lock, ws, ws_bytes, _, _ = _scratch(device, stream, need, 0)
    try:
        st = L.tb_beam_select(logits.data_ptr(), stride, vocab, code, scores.data_ptr(),
                              None if finished is None else finished.data_ptr(), end_token, rows, K, M,
                              best.data_ptr(), parents.data_ptr(), tokens.data_ptr(), ws.data_ptr(), ws_bytes, stream)
    finally:
        lock.release()
    _lib.check(st, "tb_beam_select")
    return BeamChoice(best, parents, tokens)


@functools.lru_cache(maxsize=256)
def _select_bytes(rows: int, vocab: int, picks: int) -> int:
    return _lib.lib().tb_beam_select_workspace_bytes(rows, vocab, picks)


@functools.lru_cache(maxsize=256)
def _reorder_bytes(rows: int, beams: int, max_blocks: int) -> int:
    return _lib.lib().tb_beam_reorder_workspace_bytes(rows, beams, max_blocks)


def reorder_beams(storage: torch.Tensor | None, tables: DeviceTables, parents: torch.Tensor,
                  step: DeviceStep | None = None) -> None:
    """The beams' paged states follow the selection, in place (tb_beam_reorder): row (g, k) continues row
    (g, parents[g, k]); -1 empties it. Whole blocks are shared, the block that is not full is kept by
    its row's first child and copied for the others, in every layer; blocks that no row holds any more are
    free again. storage: the layers' pools [layers, num_blocks, 2, kv_heads, block_size, head_dim]
    (PagedKVCache.storage), or None for the tables alone. parents [G, K] int32. ``step``: the step that
    has just run (its lengths become the state's); without it the state's own lengths. Where the free blocks do not
    suffice nothing is changed (tables.check() raises)."""
    device, K, G = tables.device, tables.group_size, tables.num_rows // tables.group_size
    _ints("parents", parents, torch.int32, (G, K), device)
    layers = stride = hkv = d = dtype = 0
    if storage is not None:
        _lib.require_gpu_tensor("storage", storage)
        if storage.dim() != 6 or storage.shape[2] != 2 or not storage.is_contiguous():
            raise ValueError("storage must be a contiguous [layers, num_blocks, 2, kv_heads, block_size, head_dim] tensor")
        if storage.dtype not in _lib.DTYPE_CODE:
            raise TypeError(f"unsupported pool dtype {storage.dtype}")
        if storage.device != device:
            raise ValueError(f"storage is on {storage.device}, the tables on {device}")
        if storage.shape[1] != tables.num_blocks or storage.shape[4] != tables.block_size:
            raise ValueError(f"tables are for {tables.num_blocks} blocks of {tables.block_size} positions")
        layers, hkv, d, dtype = storage.shape[0], storage.shape[3], storage.shape[5], _lib.DTYPE_CODE[storage.dtype]
        stride = storage.stride(0) * storage.element_size()
        if d * storage.element_size() % 16:
            raise ValueError(f"head_dim {d} is not served (rows of whole 16-byte pieces are)")
    if step is not None and (step.context_lens.device != device or step.context_lens.shape[0] != tables.num_rows):
        raise ValueError("the step was made for other tables (DeviceTables.new_step)")
    if _elsewhere(device):
        with torch.cuda.device(device):
            return reorder_beams(storage, tables, parents, step)
    p = tables._ptr
    lens, free = (p["context_lens"], p["num_free"]) if step is None else step._args[2:4]
    L, stream, need = _lib.lib(), _lib.stream_handle(device), _reorder_bytes(tables.num_rows, K, tables.max_blocks)
    lock, ws, ws_bytes, _, _ = _scratch(device, stream, need, 0)
    try:
        st = L.tb_beam_reorder(
            None if storage is None else storage.data_ptr(), layers, stride, tables.num_blocks, hkv, d,
            tables.block_size, dtype, p["block_tables"], tables.max_blocks, tables.num_rows, K, lens, p["context_lens"],
            p["ref_counts"], p["free_blocks"], free, p["num_free"], p["shared_blocks"], parents.data_ptr(), p["status"],
            ws.data_ptr(), ws_bytes, stream)
    finally:
        lock.release()
    _lib.check(st, "tb_beam_reorder")


class BeamPlan:
    """How a step's attention is cut over the GPU (tb_beam_plan), for one geometry: made on the GPU from
    the lengths that are there, once for all layers of a step. A plan belongs to its tables; build() it anew for every step,
    on the stream of the calls that use it."""

    def __init__(self, tables: DeviceTables, *, num_heads: int, num_kv_heads: int, head_dim: int, dtype: torch.dtype):
        if dtype not in _lib.DTYPE_CODE:
            raise TypeError(f"unsupported dtype {dtype}")
        if num_heads <= 0 or num_kv_heads <= 0 or num_heads % num_kv_heads or num_heads > 4096:
            raise ValueError(f"num_heads {num_heads} is not a multiple of kv heads {num_kv_heads} (of at most 4096)")
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim {head_dim} is not served (64 and 128 are)")
        if tables.block_size < 16:
            raise ValueError("blocks of fewer than 16 positions are not served")
        self.tables, self.num_heads, self.num_kv_heads = tables, num_heads, num_kv_heads
        self.head_dim, self.dtype = head_dim, dtype
        self.built = False
        L = _lib.lib()
        sizes = (tables.num_rows, tables.group_size, num_heads, num_kv_heads, head_dim, _lib.DTYPE_CODE[dtype])
        self.buffer = torch.zeros(max(16, L.tb_beam_plan_bytes(*sizes)), dtype=torch.uint8, device=tables.device)
        self.workspace_bytes = L.tb_beam_attention_workspace_bytes(*sizes)
        # of the usual call, once: a call is as short as its launches
        self._pool_shape = (tables.num_blocks, 2, num_kv_heads, tables.block_size, head_dim)
        self._q_shape = (tables.num_rows, num_heads, head_dim)
        self._scale, self._dtype_code = 1.0 / math.sqrt(head_dim), _lib.DTYPE_CODE[dtype]
        self._ptr, self._bytes = self.buffer.data_ptr(), self.buffer.numel()

    def build(self, row_ctx: torch.Tensor | None = None) -> "BeamPlan":
        """The plan for rows that see row_ctx [rows] int32 positions (0: none): a step's row_ctx
        (DeviceTables.new_step(padded=1)), by default the tables' lengths."""
        t = self.tables
        if row_ctx is None:
            row_ctx = t.context_lens
        _ints("row_ctx", row_ctx, torch.int32, (t.num_rows,), t.device)
        if _elsewhere(t.device):
            with torch.cuda.device(t.device):
                return self.build(row_ctx)
        st = _lib.lib().tb_beam_plan(row_ctx.data_ptr(), t._ptr["shared_blocks"], t.num_rows, t.group_size,
                                     t.max_blocks, self.num_heads, self.num_kv_heads, self.head_dim, t.block_size,
                                     self._dtype_code, self._ptr, self._bytes, _lib.stream_handle(t.device))
        _lib.check(st, "tb_beam_plan")
        self.built = True
        return self


def beam_attention(q: torch.Tensor, pool: torch.Tensor, plan: BeamPlan, *, scale: float | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per row (tb_beam_attention): row r over the positions of its table that the plan
    was built for, the blocks that a request's rows share read once for all of them. The new tokens' K/V
    must be in the pool (ops.kv_append, same stream).

    q: [rows, num_heads, head_dim] (after rotation) in the pool's dtype; returns [rows, num_heads *
    head_dim]. ``scale``: 1 / sqrt(head_dim) by default. A row that sees nothing gives 0."""
    device, dtype, t, hq, d, R = pool.device, plan.dtype, plan.tables, plan.num_heads, plan.head_dim, plan.tables.num_rows
    if not plan.built:
        raise ValueError("the plan has not been built (BeamPlan.build)")
    nb, qs, os_ = t.num_blocks, hq * d, hq * d
    if not (pool.shape == plan._pool_shape and q.shape == plan._q_shape and device == t.device == q.device
            and pool.dtype == q.dtype == dtype and pool.is_contiguous() and q.is_contiguous()):
        nb, qs = _check_attention(q, pool, plan)   # (what is not as usual)
    if out is not None:
        if out.dtype != dtype or out.shape[0] != R or out.device != device:
            raise ValueError("out must match q's dtype, device and row count")
        os_ = _rows_view("out", out, hq, d)
    if _elsewhere(device):
        with torch.cuda.device(device):
            return beam_attention(q, pool, plan, scale=scale, out=out)
    if out is None:
        out = torch.empty(R, hq * d, device=device, dtype=dtype)
    stream = _lib.stream_handle(device)
    lock, ws, ws_bytes, _, _ = _scratch(device, stream, plan.workspace_bytes, 0)
    try:
        st = _lib.lib().tb_beam_attention(
            q.data_ptr(), qs, pool.data_ptr(), nb, out.data_ptr(), os_, t._ptr["block_tables"], t.max_blocks, R,
            t.group_size, hq, plan.num_kv_heads, d, t.block_size, plan._scale if scale is None else float(scale),
            plan._dtype_code, plan._ptr, plan._bytes, ws.data_ptr(), ws_bytes, stream)
    finally:
        lock.release()
    _lib.check(st, "tb_beam_attention")
    return out


def _check_attention(q: torch.Tensor, pool: torch.Tensor, plan: BeamPlan) -> tuple[int, int]:
    """The pool's blocks and q's row stride, where both may serve the plan."""
    nb, hkv, bs, d = _check_pool(pool)
    device, dtype, t = pool.device, pool.dtype, plan.tables
    if q.device != device:
        _lib.require_gpu_tensor("q", q)
        raise ValueError(f"q is on {q.device}, the pool on {device}")
    if t.device != device:
        raise ValueError(f"the plan is on {t.device}, the pool on {device}")
    if q.dtype != dtype or plan.dtype != dtype:
        raise TypeError(f"q {q.dtype}, pool {dtype} and plan {plan.dtype} differ in dtype")
    if hkv != plan.num_kv_heads or d != plan.head_dim or bs != t.block_size or nb < t.num_blocks:
        raise ValueError(f"the plan is for {t.num_blocks} blocks of {t.block_size} positions, {plan.num_kv_heads} kv heads "
                         f"of {plan.head_dim}; the pool is {tuple(pool.shape)}")
    qs = _rows_view("q", q, plan.num_heads, d)
    if q.shape[0] != t.num_rows:
        raise ValueError(f"q has {q.shape[0]} rows, the tables {t.num_rows}")
    return nb, qs
