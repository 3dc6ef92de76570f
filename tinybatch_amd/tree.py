"""Speculative decoding over the paged cache: steps whose rows are trees of drafted tokens.

The reference decodes one token per sequence and step (src/tinybatch/engine.py:99-126); here a
step carries, for every sequence, the last token it emitted (the root) and drafted tokens
below it, each a child of an earlier node (a chain of drafts is the tree of one child each):

    meta = cache.tree_metadata(parents, cached_lens, block_tables, num_heads=n_heads)
    for layer in range(n_layers):                       # q, k, v of all nodes, before rotation
        cache.tree_append(layer, k, v, meta, rope=rope)
        attn = cache.tree_attention(layer, q, meta, rope=rope)
    verdict = verify_tree(meta, tokens, uniforms, probs, draft_probs)   # or verify_tree_greedy
    cache.commit_tree(meta, verdict.accepted, verdict.num_accepted)
    # sequence b has emitted verdict.tokens[b, :num_accepted[b]] and has
    # cached_lens[b] + num_accepted[b] positions in its cache; the last token is the next root

Everything is enqueued on the tensors' device's current stream, nothing synchronises; the
verdict stays on the device and the commit reads it there.
"""
from __future__ import annotations

import itertools
import math
import threading
from dataclasses import dataclass, field
from typing import NamedTuple

import numpy as np
import torch

from . import _lib
from .metadata import pad4
from .ops import Rope, _check_pool, _rows_view, kv_append

MAX_NODES = 1024             # TB_TREE_MAX_NODES
MAX_VOCAB = 64 * ((1 << 17) - 64)
_FAULT_PARENT, _FAULT_BLOCK, _FAULT_SLOTS, _FAULT_SHARED, _FAULT_CACHED = 1, 3, 4, 5, 6   # TB_TREE_FAULT_*
NUM_CUS, NUM_XCDS = 256, 8   # MI355X, for which the work lists are made


@dataclass
class TreeMetadata:
    """One step's trees: built by build_tree_metadata, uploaded by ``to`` and used by every
    layer's calls."""
    num_rows: int
    num_seqs: int
    max_nodes: int               # nodes of the largest tree
    max_refusals: int            # of a walk from the root, those that leave a sibling to test
    mask_words: int              # 32-bit words of a row's mask
    # the cache part (None / 0 without cached_lens)
    block_size: int
    num_blocks: int
    max_blocks_per_seq: int
    num_heads: int | None
    num_kv_heads: int | None
    head_dim: int | None
    dtype: torch.dtype | None
    # host copies
    parents_np: np.ndarray       # [T] inside the tree, -1 for a root
    row_starts_np: np.ndarray    # [B + 1]
    positions_np: np.ndarray     # [T] int64: cached + depth, the nodes' RoPE positions (no cache: the depth)
    mask_np: np.ndarray          # [T, mask_words] uint32
    row_seq_np: np.ndarray       # [T]
    cached_np: np.ndarray | None
    block_tables_np: np.ndarray | None
    slot_mapping_np: np.ndarray | None
    # tb_tree_attention's work list
    work_np: np.ndarray | None = None         # [n, 12]
    split_np: np.ndarray | None = None        # [rows of contexts cut into parts, 4]
    partial_slots: int = 0
    column_blocks: int = 1
    units: int = 0                            # arrival counters of a call that joins its parts itself
    # device views (one backing buffer)
    device: torch.device | None = None
    parents: torch.Tensor | None = None
    row_starts: torch.Tensor | None = None
    mask: torch.Tensor | None = None          # [T, mask_words] int32
    row_seq: torch.Tensor | None = None
    positions: torch.Tensor | None = None     # [T] int64
    cached: torch.Tensor | None = None
    block_tables: torch.Tensor | None = None
    slot_mapping: torch.Tensor | None = None
    work: torch.Tensor | None = None
    split: torch.Tensor | None = None
    addresses: tuple | None = None            # of the arrays, in the order that the calls take them
    longest: int = 0                          # the largest RoPE position, plus one
    verify_bytes: dict = field(default_factory=dict)   # workspace of verify_tree by vocabulary

    @property
    def depths_np(self) -> np.ndarray:
        """[T]: every node's depth in its tree."""
        return self.positions_np - (0 if self.cached_np is None else self.cached_np[self.row_seq_np])

    def to(self, device: torch.device) -> "TreeMetadata":
        """Upload every array with one host-to-device copy (views into one buffer)."""
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        has_cache = self.cached_np is not None
        parts = [("positions", self.positions_np.view(np.int32)), ("parents", self.parents_np),
                 ("row_starts", self.row_starts_np), ("mask", self.mask_np.view(np.int32).reshape(-1)),
                 ("row_seq", self.row_seq_np)]
        if has_cache:
            parts += [("cached", self.cached_np), ("block_tables", self.block_tables_np.reshape(-1)),
                      ("slot_mapping", self.slot_mapping_np), ("work", self.work_np.reshape(-1)),
                      ("split", self.split_np.reshape(-1))]
        host = np.zeros(sum(pad4(x.size) for _, x in parts), dtype=np.int32)
        at, spans = 0, {}
        for name, x in parts:
            host[at:at + x.size] = x
            spans[name] = (at, x.size)
            at += pad4(x.size)
        src = torch.from_numpy(host)
        if device.type == "cuda":
            src = src.pin_memory()
        buf = src.to(device, non_blocking=True)
        for name, (o, size) in spans.items():
            setattr(self, name, buf.narrow(0, o, size))
        self.positions = self.positions.view(torch.int64)
        self.mask = self.mask.view(-1, self.mask_words)
        if has_cache:
            self.block_tables = self.block_tables.view(-1, self.max_blocks_per_seq)
        self.device = device
        self.addresses = None
        if has_cache:
            self.addresses = (self.block_tables.data_ptr(), self.max_blocks_per_seq, self.row_starts.data_ptr(),
                              self.cached.data_ptr(), self.num_seqs, self.row_seq.data_ptr(), self.num_rows)
        return self


def _flat(lists, lens: np.ndarray, lo: int) -> np.ndarray:
    """The lists' integers one behind the other, what int32 does not hold at its ends."""
    flat = np.fromiter(itertools.chain.from_iterable(lists), np.int64, int(lens.sum()))
    return np.clip(flat, lo, np.iinfo(np.int32).max).astype(np.int32)


def _see(mask: np.ndarray, visible, row_starts: np.ndarray) -> None:
    """The sequences that name the nodes their rows see."""
    for b, v in enumerate(visible):
        if v is None:
            continue
        first, n = int(row_starts[b]), int(row_starts[b + 1] - row_starts[b])
        v = np.asarray(v, dtype=bool)
        if v.shape != (n, n):
            raise ValueError(f"visible[{b}] must be [{n}, {n}], got {v.shape}")
        rows = np.packbits(v, axis=1, bitorder="little")
        own = mask[first:first + n].view(np.uint8)
        own[:] = 0
        own[:, :rows.shape[1]] = rows


def _attach_work(meta: TreeMetadata) -> None:
    """The work list of the step's attention calls (tb_build_tree_work)."""
    L = _lib.lib()
    nodes = np.diff(meta.row_starts_np).astype(np.int32)
    counts = np.zeros(5, dtype=np.int32)
    head = (meta.cached_np.ctypes.data, nodes.ctypes.data, meta.num_seqs, meta.num_heads, meta.num_kv_heads,
            meta.head_dim, _lib.DTYPE_CODE[meta.dtype], NUM_CUS, NUM_XCDS)
    _lib.check(L.tb_build_tree_work(*head, None, 0, None, 0, counts.ctypes.data), "tb_build_tree_work")
    work, split = np.zeros((int(counts[0]), 12), dtype=np.int32), np.zeros((int(counts[1]), 4), dtype=np.int32)
    _lib.check(L.tb_build_tree_work(*head, work.ctypes.data, work.shape[0], split.ctypes.data, split.shape[0],
                                    counts.ctypes.data), "tb_build_tree_work")
    meta.work_np, meta.split_np = work, split
    meta.partial_slots, meta.column_blocks, meta.units = int(counts[2]), int(counts[3]), int(counts[4])


def build_tree_metadata(parents, cached_lens=None, block_tables=None, *, block_size: int = 0, num_blocks: int = 0,
                        num_heads: int | None = None, num_kv_heads: int | None = None, head_dim: int | None = None,
                        dtype: torch.dtype | None = None, visible=None) -> TreeMetadata:
    """The metadata of a step of trees (host lists in, ``to(device)`` uploads it).

    parents[b][i] is the parent of sequence b's node i inside its tree: -1 for node 0, the
    root, and an earlier node for every other (no nodes: a sequence without rows). The step's
    flat rows are the trees one behind the other. cached_lens[b] positions of sequence b are in
    the cache; block_tables[b] covers them and one position per node behind them (node i at
    cached_lens[b] + i). Without cached_lens the trees alone (verify_tree needs no more).

    A node sees the cached positions, itself and its ancestors, or the nodes that
    visible[b] ([nodes, nodes] booleans, row i for node i) names; a row that sees nothing
    gives 0.

    A table too short, or a block id outside the pool, raises IndexError; two nodes of the step
    in one slot raise ValueError.
    """
    parents = list(parents)
    B = len(parents)
    sizes = np.fromiter(map(len, parents), np.int64, B)
    T, max_nodes = int(sizes.sum()), int(sizes.max(initial=0))
    if max_nodes > MAX_NODES:
        raise ValueError(f"a tree of {max_nodes} nodes; at most {MAX_NODES} are served")
    if visible is not None and len(visible) != B:
        raise ValueError("visible needs one entry per sequence")
    words = max(1, -(-max_nodes // 32))
    row_starts = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    flat, mask = _flat(parents, sizes, -2), np.empty((T, words), dtype=np.uint32)
    positions, row_seq = np.empty(T, dtype=np.int64), np.empty(T, dtype=np.int32)
    cached = tables = slots = None
    max_nb = 0
    if cached_lens is None:
        if block_tables is not None:
            raise ValueError("block_tables without cached_lens")
    else:
        if block_tables is None or len(block_tables) != B or len(cached_lens) != B:
            raise ValueError("cached_lens and block_tables need one entry per sequence")
        if block_size <= 0 or block_size & (block_size - 1) or num_blocks <= 0:
            raise ValueError("block_size must be a power of two and num_blocks positive")
        if num_heads is None or num_kv_heads is None or head_dim is None or dtype not in _lib.DTYPE_CODE:
            raise ValueError("num_heads, num_kv_heads, head_dim and dtype (fp32, fp16, bf16) describe the attention's calls")
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim {head_dim} is not served (64 and 128 are)")
        if num_heads <= 0 or num_kv_heads <= 0 or num_heads % num_kv_heads:
            raise ValueError(f"num_heads {num_heads} is not a multiple of kv heads {num_kv_heads}")
        ends = np.fromiter(cached_lens, np.int64, B) + sizes
        if B and ((ends < sizes).any() or ends.max() > (1 << 30)):
            raise ValueError("cached_lens must be >= 0 (and a context at most 2^30 positions)")
        cached = (ends - sizes).astype(np.int32)
        need, lens = -(-ends // block_size), np.fromiter(map(len, block_tables), np.int64, B)
        if (lens < need).any():
            b = int(np.argmax(lens < need))
            raise IndexError(f"sequence {b} needs {need[b]} blocks for {ends[b]} positions, table has {lens[b]}")
        max_nb = max(1, int(need.max(initial=0)))
        tables = np.full((B, max_nb), -1, dtype=np.int32)            # -1: no block
        if (lens <= 2 * need + 64).all():
            ids, at = _flat(block_tables, lens, -1), np.cumsum(lens) - lens
        else:                                                        # tables made longer than they are used
            ids, at = _flat([t[:k] for t, k in zip(block_tables, need)], need, -1), np.cumsum(need) - need
        inside = np.arange(max_nb) < need[:, None]
        tables[inside] = ids[(at[:, None] + np.arange(max_nb))[inside]]
        slots = np.empty(T, dtype=np.int32)
    info = np.zeros(4, dtype=np.int32)
    st = _lib.lib().tb_build_tree_rows(
        flat.ctypes.data, row_starts.ctypes.data, B, None if cached is None else cached.ctypes.data,
        None if cached is None else tables.ctypes.data, max_nb, block_size, num_blocks, mask.ctypes.data, words,
        positions.ctypes.data, row_seq.ctypes.data, None if cached is None else slots.ctypes.data, info.ctypes.data)
    if st != _lib.TB_OK:
        fault, where = int(info[2]), int(info[3])
        if fault == _FAULT_PARENT:
            b = int(np.searchsorted(row_starts, where, side="right")) - 1
            i = where - int(row_starts[b])
            raise ValueError(f"parents[{b}][{i}] is {parents[b][i]}: node 0 has parent -1, every other node an earlier one")
        if fault == _FAULT_BLOCK:
            raise IndexError(f"block_tables[{where}] holds a block id outside the pool of {num_blocks} blocks")
        if fault == _FAULT_SLOTS:
            raise ValueError("a pool of more than 2^31 slots")
        if fault == _FAULT_SHARED:
            raise ValueError(f"two nodes of the step share a pool slot (block {where}): give each tree blocks of its own")
        if fault == _FAULT_CACHED:
            raise ValueError(f"a tree's nodes fall on another sequence's cached positions (block {where}): give each tree "
                             "blocks of its own behind a shared prefix of whole blocks")
        _lib.check(st, "tb_build_tree_rows")
    if visible is not None:
        _see(mask, visible, row_starts)
    meta = TreeMetadata(
        num_rows=T, num_seqs=B, max_nodes=max_nodes, max_refusals=int(info[0]), mask_words=words, block_size=block_size,
        num_blocks=num_blocks, max_blocks_per_seq=max_nb, num_heads=num_heads, num_kv_heads=num_kv_heads,
        head_dim=head_dim, dtype=dtype, parents_np=flat, row_starts_np=row_starts, positions_np=positions, mask_np=mask,
        row_seq_np=row_seq, cached_np=cached, block_tables_np=tables, slot_mapping_np=slots, longest=int(info[1]))
    if cached is None:
        return meta
    _attach_work(meta)
    return meta


class _Scratch:
    """What the calls on one stream of one device share, since they are ordered: a workspace, and
    arrival counters (zero between calls: every call leaves them zero). A call holds the lock until
    its launches are on the stream: those of another thread do not come between them."""

    def __init__(self, device: torch.device):
        self.lock = threading.RLock()
        self.workspace = torch.empty(1 << 20, dtype=torch.uint8, device=device)
        self.arrivals = torch.zeros(4096, dtype=torch.int32, device=device)


_SCRATCH: dict[tuple[int, int], _Scratch] = {}
_SCRATCH_LOCK = threading.RLock()
_KEPT_BYTES = 32 << 20       # larger workspaces are allocated call by call


def _scratch(device: torch.device, stream: int, nbytes: int, units: int):
    """(lock to release after the launches, workspace, its bytes, arrival counters or None, their number)
    of a call on the current stream. A call that is being captured gets a workspace of its own and no
    counters: its graph may be replayed beside anything."""
    if torch._C._cuda_isCurrentStreamCapturing():
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        _SCRATCH_LOCK.acquire()
        return _SCRATCH_LOCK, ws, nbytes, None, 0
    s = _SCRATCH.get((device.index, stream))
    if s is None:
        with _SCRATCH_LOCK:
            s = _SCRATCH.setdefault((device.index, stream), _Scratch(device))
    s.lock.acquire()
    try:
        if s.arrivals.shape[0] < units:
            s.arrivals = torch.zeros(2 * units, dtype=torch.int32, device=device)
        if nbytes > _KEPT_BYTES:
            return s.lock, torch.empty(nbytes, dtype=torch.uint8, device=device), nbytes, s.arrivals, units
        if s.workspace.shape[0] < nbytes:
            s.workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
    except BaseException:
        s.lock.release()
        raise
    return s.lock, s.workspace, nbytes, s.arrivals, units


def _elsewhere(device: torch.device) -> bool:
    """Whether the tensors' device is not the current one."""
    return device.index != torch._C._cuda_getDevice()


def _check_meta(meta: TreeMetadata, device: torch.device, cache: bool) -> None:
    if meta.device is None:
        raise ValueError("metadata has not been uploaded (call meta.to(device))")
    if meta.device != device:
        raise ValueError(f"metadata is on {meta.device}, the tensors on {device}")
    if cache and meta.cached is None:
        raise ValueError("metadata was built without cached_lens and block_tables")


def _check_rope(rope: Rope, meta: TreeMetadata, head_dim: int, device: torch.device) -> None:
    rope.check(head_dim, device)
    if rope.max_position < meta.longest:
        raise IndexError(f"rope tables of {rope.max_position} positions, the step's nodes reach {meta.longest}")


def tree_append(pool: torch.Tensor, k: torch.Tensor, v: torch.Tensor, meta: TreeMetadata,
                rope: Rope | None = None) -> None:
    """The nodes' K/V rows [T, kv_heads, head_dim] into their slots (ops.kv_append); with ``rope``
    k is the projection before rotation, rotated at cached + depth on the way."""
    _lib.require_gpu_tensor("pool", pool)
    _check_meta(meta, pool.device, True)
    if pool.dim() == 5 and (pool.shape[3] != meta.block_size or pool.shape[0] < meta.num_blocks):
        raise ValueError(f"metadata is for {meta.num_blocks} blocks of {meta.block_size} positions")
    if rope is not None:
        _check_rope(rope, meta, pool.shape[-1], pool.device)
    with torch.cuda.device(pool.device):
        kv_append(pool, k, v, meta.slot_mapping, rope=rope, positions=meta.positions if rope is not None else None)


def tree_attention(q: torch.Tensor, pool: torch.Tensor, meta: TreeMetadata, *, scale: float | None = None,
                   out: torch.Tensor | None = None, rope: Rope | None = None,
                   mask: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of every node of the step over its sequence's cached positions and the nodes it
    sees (tb_tree_attention); the nodes' K/V must be in the pool (tree_append, same stream).

    q: [T, num_heads, head_dim] in the pool's dtype; returns [T, num_heads * head_dim]. ``scale``:
    1 / sqrt(head_dim) by default. With ``rope`` q is the projection before rotation. ``mask``
    ([T, meta.mask_words] int32 on the GPU, bit j % 32 of word j / 32: node j is seen) replaces the
    metadata's, for masks made on the device. A row that sees nothing gives 0.
    """
    nb, hkv, bs, d = _check_pool(pool)
    device, dtype = pool.device, pool.dtype
    if q.device != device:
        _lib.require_gpu_tensor("q", q)
        raise ValueError(f"q is on {q.device}, the pool on {device}")
    _check_meta(meta, device, True)
    if q.dtype != dtype or meta.dtype != dtype:
        raise TypeError(f"q {q.dtype}, pool {dtype} and metadata {meta.dtype} differ in dtype")
    if hkv != meta.num_kv_heads or d != meta.head_dim or bs != meta.block_size or nb < meta.num_blocks:
        raise ValueError(f"metadata is for {meta.num_blocks} blocks of {meta.block_size} positions, "
                         f"{meta.num_kv_heads} kv heads of {meta.head_dim}; the pool is {tuple(pool.shape)}")
    if _elsewhere(device):
        with torch.cuda.device(device):
            return tree_attention(q, pool, meta, scale=scale, out=out, rope=rope, mask=mask)
    hq, T = meta.num_heads, meta.num_rows
    qs = _rows_view("q", q, hq, d)
    if q.shape[0] != T:
        raise ValueError(f"q has {q.shape[0]} rows, metadata describes {T}")
    if out is None:
        out, os_ = torch.empty(T, hq * d, device=device, dtype=dtype), hq * d
    else:
        if out.dtype != dtype or out.shape[0] != T or out.device != device:
            raise ValueError("out must match q's dtype, device and row count")
        os_ = _rows_view("out", out, hq, d)
    if mask is None:
        mask = meta.mask
    elif (mask.dtype != torch.int32 or mask.device != device or mask.shape != (T, meta.mask_words)
          or not mask.is_contiguous()):
        raise TypeError(f"mask must be a contiguous int32 [{T}, {meta.mask_words}] tensor on {device}")
    cos = sin = positions = None
    longest = 0
    if rope is not None:
        _check_rope(rope, meta, d, device)
        cos, sin, longest = rope.cos.data_ptr(), rope.sin.data_ptr(), rope.max_position
        positions = meta.positions.data_ptr()
    stream = _lib.stream_handle(device)
    slots, units = meta.partial_slots, meta.units
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    lock = ws = arrivals = None
    ws_bytes = 0
    if slots:
        lock, ws, ws_bytes, arrivals, units = _scratch(device, stream, slots * hq * (d + 2) * 4, units)
    try:
        st = _lib.lib().tb_tree_attention(
            q.data_ptr(), qs, pool.data_ptr(), nb, out.data_ptr(), os_, *meta.addresses, mask.data_ptr(),
            meta.mask_words, meta.work.data_ptr(), meta.work_np.shape[0], meta.column_blocks, meta.split.data_ptr(),
            meta.split_np.shape[0], slots, None if ws is None else ws.data_ptr(), ws_bytes,
            None if arrivals is None or not units else arrivals.data_ptr(), units, hq, hkv, d, bs, scale,
            _lib.DTYPE_CODE[dtype], positions, cos, sin, longest, stream)
    finally:
        if lock is not None:
            lock.release()
    _lib.check(st, "tb_tree_attention")
    return out


class TreeVerdict(NamedTuple):
    """What a verification kept, on the device."""
    accepted: torch.Tensor       # [B, max_nodes] int32: the path's nodes from the root on, then -1
    num_accepted: torch.Tensor   # [B] int32: how many (0 for a sequence without rows)
    tokens: torch.Tensor         # [B, max_nodes] int64: num_accepted tokens emitted (the last one drawn), then -1


def _verdict(meta: TreeMetadata, device: torch.device) -> TreeVerdict:
    width = max(meta.max_nodes, 1)
    return TreeVerdict(torch.empty(meta.num_seqs, width, dtype=torch.int32, device=device),
                       torch.empty(meta.num_seqs, dtype=torch.int32, device=device),
                       torch.empty(meta.num_seqs, width, dtype=torch.int64, device=device))


def _vocab_rows(name: str, t: torch.Tensor, rows: int) -> int:
    """The row stride of a [rows, vocab] tensor of contiguous rows."""
    if t.dim() != 2 or t.shape[0] != rows or t.shape[1] < 1 or t.stride(1) != 1:
        raise ValueError(f"{name} must be [{rows}, vocab] with contiguous rows, got {tuple(t.shape)}")
    return t.stride(0) if rows > 1 else t.shape[1]


def _node_values(name: str, t: torch.Tensor, dtype: torch.dtype, rows: int, device: torch.device) -> None:
    if t.dtype != dtype or t.device != device or t.shape != (rows,) or not t.is_contiguous():
        raise TypeError(f"{name} must be a contiguous {dtype} [{rows}] tensor on {device}")


def verify_tree(meta: TreeMetadata, tokens: torch.Tensor, uniforms: torch.Tensor, probs: torch.Tensor,
                draft_probs: torch.Tensor | None = None) -> TreeVerdict:
    """Which drafts the target's probabilities keep, and the token after them (tb_tree_verify;
    the rule is written there): the emitted tokens follow the target's distribution.

    probs [T, vocab] (fp32, fp16 or bf16, rows that sum to 1): row r the target's distribution
    after node r. tokens [T] int64. uniforms [T] fp32 in [0, 1): one random number per node; the
    root's serves the token drawn at the end. draft_probs, in probs' dtype: row r the distribution
    that node r's children were drawn from, each independently; None for drafts that were not
    drawn at random (a draft model's most likely tokens).
    """
    device, T, dtype = probs.device, meta.num_rows, probs.dtype
    _lib.require_gpu_tensor("probs", probs)
    _check_meta(meta, device, False)
    if dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"unsupported probs dtype {dtype}")
    stride = _vocab_rows("probs", probs, T)
    vocab = probs.shape[1]
    draft, draft_stride = None, 0
    if draft_probs is not None:
        if draft_probs.dtype != dtype or draft_probs.device != device:
            raise TypeError("draft_probs must share probs' dtype and device")
        draft_stride = _vocab_rows("draft_probs", draft_probs, T)
        if draft_probs.shape[1] != vocab:
            raise ValueError(f"draft_probs must be [{T}, {vocab}], got {tuple(draft_probs.shape)}")
        draft = draft_probs.data_ptr()
    if vocab > MAX_VOCAB:
        raise ValueError(f"a vocabulary of {vocab} tokens; at most {MAX_VOCAB} are served")
    _node_values("tokens", tokens, torch.int64, T, device)
    _node_values("uniforms", uniforms, torch.float32, T, device)
    if _elsewhere(device):
        with torch.cuda.device(device):
            return verify_tree(meta, tokens, uniforms, probs, draft_probs)
    v = _verdict(meta, device)
    if T == 0:
        return v._replace(accepted=v.accepted.fill_(-1), num_accepted=v.num_accepted.zero_(), tokens=v.tokens.fill_(-1))
    L, B, width = _lib.lib(), meta.num_seqs, meta.max_nodes
    stream = _lib.stream_handle(device)
    need = meta.verify_bytes.get(vocab)
    if need is None:
        need = meta.verify_bytes[vocab] = L.tb_tree_verify_workspace_bytes(B, vocab, width)
    lock, ws, ws_bytes, arrivals, units = _scratch(device, stream, need, B)
    try:
        st = L.tb_tree_verify(
            probs.data_ptr(), stride, draft, draft_stride, vocab, _lib.DTYPE_CODE[dtype], tokens.data_ptr(),
            uniforms.data_ptr(), meta.parents.data_ptr(), meta.row_starts.data_ptr(), B, meta.max_refusals,
            v.accepted.data_ptr(), v.num_accepted.data_ptr(), v.tokens.data_ptr(), width, ws.data_ptr(), ws_bytes,
            None if arrivals is None else arrivals.data_ptr(), units, stream)
    finally:
        lock.release()
    _lib.check(st, "tb_tree_verify")
    return v


def verify_tree_greedy(meta: TreeMetadata, tokens: torch.Tensor, target_ids: torch.Tensor) -> TreeVerdict:
    """verify_tree for greedy decoding: target_ids [T] int64 is the target's choice after each node
    (layer_ops.linear_argmax, or an argmax of the logits); a child that holds it is kept."""
    _lib.require_gpu_tensor("target_ids", target_ids)
    device, T = target_ids.device, meta.num_rows
    _check_meta(meta, device, False)
    _node_values("target_ids", target_ids, torch.int64, T, device)
    _node_values("tokens", tokens, torch.int64, T, device)
    if _elsewhere(device):
        with torch.cuda.device(device):
            return verify_tree_greedy(meta, tokens, target_ids)
    v = _verdict(meta, device)
    st = _lib.lib().tb_tree_verify_greedy(
        meta.row_starts.data_ptr() if T == 0 else target_ids.data_ptr(),     # no rows: nothing is read
        meta.row_starts.data_ptr() if T == 0 else tokens.data_ptr(), meta.parents.data_ptr(),
        meta.row_starts.data_ptr(), meta.num_seqs, v.accepted.data_ptr(), v.num_accepted.data_ptr(),
        v.tokens.data_ptr(), v.accepted.shape[1], _lib.stream_handle(device))
    _lib.check(st, "tb_tree_verify_greedy")
    return v


def commit_tree(storage: torch.Tensor, meta: TreeMetadata, accepted: torch.Tensor,
                num_accepted: torch.Tensor) -> None:
    """The kept nodes' K/V rows to the positions they now have, in every layer (tb_tree_commit):
    position cached + accepted[b][j] to cached + j. storage: the layers' pools
    [layers, num_blocks, 2, kv_heads, block_size, head_dim] (PagedKVCache.storage); accepted
    and num_accepted as verify_tree gives them (nodes rising along a row)."""
    _lib.require_gpu_tensor("storage", storage)
    if storage.dim() != 6 or storage.shape[2] != 2 or not storage.is_contiguous():
        raise ValueError("storage must be a contiguous [layers, num_blocks, 2, kv_heads, block_size, head_dim] tensor")
    if storage.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"unsupported pool dtype {storage.dtype}")
    device = storage.device
    _check_meta(meta, device, True)
    layers, nb, _, hkv, bs, d = storage.shape
    if bs != meta.block_size or nb < meta.num_blocks:
        raise ValueError(f"metadata is for {meta.num_blocks} blocks of {meta.block_size} positions")
    B = meta.num_seqs
    if (accepted.dtype != torch.int32 or accepted.device != device or accepted.dim() != 2
            or accepted.shape[0] != B or accepted.shape[1] < 1 or not accepted.is_contiguous()):
        raise TypeError(f"accepted must be a contiguous int32 [{B}, nodes] tensor on {device}")
    _node_values("num_accepted", num_accepted, torch.int32, B, device)
    if _elsewhere(device):
        with torch.cuda.device(device):
            return commit_tree(storage, meta, accepted, num_accepted)
    st = _lib.lib().tb_tree_commit(
        storage.data_ptr(), layers, storage.stride(0) * storage.element_size(), nb, meta.addresses[0],
        meta.max_blocks_per_seq, meta.addresses[3], B, accepted.data_ptr(), accepted.shape[1],
        num_accepted.data_ptr(), hkv, d, bs, _lib.DTYPE_CODE[storage.dtype], _lib.stream_handle(device))
    _lib.check(st, "tb_tree_commit")
