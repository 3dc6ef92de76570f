"""Block tables, lengths and free blocks on the GPU, and steps built there.

The reference builds every step on the host: the block manager's lists give tables and slots
(src/tinybatch/block_manager.py:117-156, engine.py:99-126). Where the next step's rows are only known on
the GPU (beams that follow their parents, loops that run several steps ahead) the same arrays are
built from lengths that live there:

    tables = DeviceTables.from_lists(block_tables, context_lens, free_blocks, max_blocks=..., ...)
    step = tables.new_step(padded=1)                  # one token per row and step
    build_device_step(tables, new_lens, step)         # takes blocks, gives positions, slots, lengths
    ops.kv_append(pool, k, v, step.slot_mapping)      # and attention over step.row_ctx
    tables.take(step)                                 # the step has run: its lengths are the cached ones

Everything is enqueued on the current stream and nothing synchronises; what goes wrong on the GPU (no
free block left, a row's table full) leaves the state as it was, makes the step an empty one and
adds a bit to ``tables.status``, which ``tables.check()`` reads and raises.
"""
from __future__ import annotations

import itertools
from dataclasses import dataclass, field

import numpy as np
import torch

from . import _lib
from .block_manager import OutOfBlocks
from .metadata import StepMetadata
from .tree import _elsewhere, _scratch

MAX_BEAMS = 64               # TB_BEAMS_MAX
_OUT_OF_BLOCKS, _ROW_FULL, _BAD_PARENT, _TOO_MANY_TOKENS, _BAD_LENGTH, _TOO_MUCH_WORK = 1, 2, 4, 8, 16, 32  # TB_TABLES_*
_MOST = 1 << 24


def _ints(name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple, device: torch.device) -> None:
    if t.dtype != dtype or t.device != device or tuple(t.shape) != shape or not t.is_contiguous():
        raise TypeError(f"{name} must be a contiguous {dtype} {list(shape)} tensor on {device}")


@dataclass
class DeviceStep:
    """One step's arrays on the GPU (tb_beam_step), allocated once (DeviceTables.new_step) and
    filled by build_device_step: they may be written to, not replaced."""
    max_tokens: int
    padded: int                        # > 0: row b's tokens are the flat rows from b * padded on
    partition_tokens: int              # 0: no work items
    rows_per_item: int
    context_lens: torch.Tensor         # [rows] int32: cached + new
    num_free: torch.Tensor             # [1] int32: free blocks after the step
    query_start_loc: torch.Tensor      # [rows + 1] int32
    positions: torch.Tensor            # [max_tokens] int64
    slot_mapping: torch.Tensor         # [max_tokens] int32, -1: no token
    row_ctx: torch.Tensor              # [max_tokens] int32: positions the flat row sees, 0: no token
    row_part_offsets: torch.Tensor | None = None   # [max_tokens + 1] int32
    work_items: torch.Tensor | None = None         # [max_items, 4] int32
    split_rows: torch.Tensor | None = None         # [max_split_rows, 4] int32
    counts: torch.Tensor | None = None             # [4] int32: items, split rows, 0, partitions
    max_partitions: int = 0
    _counted: torch.Tensor | None = field(default=None, repr=False)   # context_lens and num_free, one behind the other
    _args: tuple = field(default=(), repr=False)   # tb_beam_step's arguments from pad_tokens to counts

    def metadata(self, tables: "DeviceTables") -> StepMetadata:
        """The step as ops.paged_attention and ops.kv_append take it: the arrays above, sized to their
        capacities, with the counts read on the device (no fused append)."""
        if not self.partition_tokens:
            raise ValueError("the step was made without work items (new_step's partition_tokens)")
        e = np.zeros(0, np.int32)
        most = -(-tables.max_blocks * tables.block_size // self.partition_tokens)
        m = StepMetadata(num_tokens=self.max_tokens, num_seqs=tables.num_rows, block_size=tables.block_size,
                         partition_tokens=self.partition_tokens, max_blocks_per_seq=tables.max_blocks,
                         num_work_items=self.work_items.shape[0], total_partitions=self.max_partitions,
                         max_parts_per_row=most, decode_only=False, rows_per_item=self.rows_per_item,
                         num_prefill_tiles=0, num_split_rows=self.split_rows.shape[0] if most > 1 else 0,
                         slot_mapping_np=e, block_tables_np=e, work_np=e, row_part_off_np=e, row_ctx_np=e,
                         prefill_tiles_np=e, split_rows_np=e, superseded=False, num_blocks=tables.num_blocks)
        m.slot_mapping, m.block_tables = self.slot_mapping, tables.block_tables
        m.work, m.row_part_off = self.work_items, self.row_part_offsets
        m.split_rows = m.prefill_tiles = self.split_rows
        m.device_counts = self.counts
        return m


class DeviceTables:
    """The paged state of ``num_rows`` rows on the GPU: block tables, lengths, reference counts and
    the free blocks. Rows g * group_size .. belong to request g (its beams). Its arrays are allocated
    once: they may be written to, not replaced (who writes lengths or tables sets shared_blocks, the leading whole blocks
    that all of a request's rows with positions have in common, to what holds: 0 always does)."""

    def __init__(self, num_rows: int, *, max_blocks: int, block_size: int, num_blocks: int, device,
                 group_size: int = 1, _arrays=None):
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("DeviceTables needs a GPU device (no CPU fallback)")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        _check_sizes(num_rows, max_blocks, block_size, num_blocks, group_size)
        self.num_rows, self.max_blocks, self.block_size = num_rows, max_blocks, block_size
        self.num_blocks, self.group_size, self.device = num_blocks, group_size, device
        # one buffer, so that a state from lists is one copy; each array begins at a multiple of 256 bytes
        sizes = (num_rows + 1, num_rows * max_blocks, num_blocks, num_blocks, num_rows // group_size, 1)
        begins = np.cumsum([0] + [-(-n // 64) * 64 for n in sizes]).tolist()
        if _arrays is None:
            self._buffer = torch.zeros(begins[-1], dtype=torch.int32, device=device)
        else:
            host = np.zeros(begins[-1], np.int32)
            for at, x in zip(begins, _arrays):
                host[at:at + x.size] = x.reshape(-1)
            self._buffer = torch.from_numpy(host).to(device)
        parts = [self._buffer[at:at + n] for at, n in zip(begins, sizes)]
        self._counted, self.ref_counts, self.free_blocks, self.shared_blocks, self.status = parts[0], *parts[2:]
        self.context_lens, self.num_free = self._counted[:num_rows], self._counted[num_rows:]
        self.block_tables = parts[1].view(num_rows, max_blocks)
        if _arrays is None:
            self.block_tables.fill_(-1)
        # addresses, taken once: a step's calls are short, and every data_ptr() is a part of them
        self._ptr = {name: getattr(self, name).data_ptr() for name in
                     ("block_tables", "context_lens", "num_free", "ref_counts", "free_blocks", "shared_blocks", "status")}

    @classmethod
    def from_lists(cls, block_tables, context_lens, free_blocks, *, max_blocks: int, block_size: int, num_blocks: int,
                   device, group_size: int = 1, held=()) -> "DeviceTables":
        """The state that the host's lists describe: row b has context_lens[b] positions in the
        blocks of block_tables[b] (rows may share blocks), free_blocks are handed out from
        the end (BlockManager.free_ids). ``held``: blocks that someone else holds too (a prefix
        cache), once for every holder."""
        rows = len(block_tables)
        arrays = _state_arrays(block_tables, context_lens, free_blocks, max_blocks, block_size, num_blocks, group_size, held)
        return cls(rows, max_blocks=max_blocks, block_size=block_size, num_blocks=num_blocks, device=device,
                   group_size=group_size, _arrays=arrays)

    def new_step(self, *, max_tokens: int | None = None, padded: int = 0, partition_tokens: int = 0,
                 rows_per_item: int = 1, max_items: int | None = None, max_partitions: int | None = None,
                 max_split_rows: int | None = None) -> DeviceStep:
        """The arrays of a step of up to ``max_tokens`` new tokens, one row's behind the other's; with
        ``padded`` every row has that many flat rows, used or not. With ``partition_tokens``
        (ops.partition_tokens) also tb_paged_attention's work items, of up to ``rows_per_item`` rows
        (ops.rows_per_item); their capacities are by default what max_tokens rows of full tables need."""
        if padded < 0 or (padded and max_tokens not in (None, padded * self.num_rows)):
            raise ValueError("padded steps have padded * num_rows flat rows")
        if padded:
            max_tokens = padded * self.num_rows
        if max_tokens is None or not 0 <= max_tokens < _MOST:
            raise ValueError(f"max_tokens must be given, below {_MOST}")
        i32 = dict(dtype=torch.int32, device=self.device)
        counted = torch.zeros(self.num_rows + 1, **i32)
        s = DeviceStep(max_tokens, padded, partition_tokens, rows_per_item, counted[:self.num_rows],
                       counted[self.num_rows:], torch.zeros(self.num_rows + 1, **i32),
                       torch.zeros(max_tokens, dtype=torch.int64, device=self.device),
                       torch.full((max_tokens,), -1, **i32), torch.zeros(max_tokens, **i32), _counted=counted)
        if partition_tokens:
            if partition_tokens < 0 or not 1 <= rows_per_item <= 16:
                raise ValueError("partition_tokens must be positive and rows_per_item within 1 .. 16")
            most = max_tokens * -(-self.max_blocks * self.block_size // partition_tokens)
            sizes = [most if n is None else n for n in (max_items, max_partitions)]
            sizes.append(max_tokens if max_split_rows is None else max_split_rows)
            if not all(0 <= n < _MOST for n in sizes):
                raise ValueError(f"work items, partitions and split rows must stay below {_MOST}: give their capacities")
            s.row_part_offsets = torch.zeros(max_tokens + 1, **i32)
            s.work_items, s.split_rows = torch.zeros(sizes[0], 4, **i32), torch.zeros(sizes[2], 4, **i32)
            s.max_partitions = sizes[1]
            s.counts = torch.zeros(4, **i32)
        ptr = lambda t: None if t is None else t.data_ptr()
        entries = lambda t: 0 if t is None else t.shape[0]
        s._args = (padded, max_tokens, s.context_lens.data_ptr(), s.num_free.data_ptr(), s.query_start_loc.data_ptr(),
                   s.positions.data_ptr(), s.slot_mapping.data_ptr(), s.row_ctx.data_ptr(), partition_tokens, rows_per_item,
                   ptr(s.row_part_offsets), ptr(s.work_items), entries(s.work_items), s.max_partitions, ptr(s.split_rows),
                   entries(s.split_rows), ptr(s.counts))
        return s

    def take(self, step: DeviceStep) -> None:
        """The step has run: its lengths and free blocks are the state's."""
        self._counted.copy_(step._counted)

    def check(self) -> None:
        """Raise what a call could not do since the last check (waits for the current stream, which is to be the calls')."""
        st = int(self.status.item())
        if not st:
            return
        self.status.zero_()
        if st & _OUT_OF_BLOCKS:
            raise OutOfBlocks(f"a step needed more KV blocks than are free ({self.num_blocks} in all)")
        if st & _ROW_FULL:
            raise IndexError(f"a row needed more than {self.max_blocks} blocks")
        if st & _BAD_PARENT:
            raise IndexError(f"a parent outside [-1, {self.group_size})")
        if st & _TOO_MANY_TOKENS:
            raise ValueError("more new tokens than the step has flat rows for")
        if st & _BAD_LENGTH:
            raise ValueError("a length below 0, or beyond its row's blocks")
        raise ValueError("more work items, partitions or split rows than the step has room for")


def _check_sizes(num_rows, max_blocks, block_size, num_blocks, group_size) -> None:
    if num_rows < 0 or max_blocks <= 0 or num_blocks <= 0:
        raise ValueError("max_blocks and num_blocks must be positive and num_rows not negative")
    if block_size <= 0 or block_size & (block_size - 1):
        raise ValueError("block_size must be a power of two")
    if not 1 <= group_size <= MAX_BEAMS or num_rows % group_size:
        raise ValueError(f"group_size must divide the rows and lie within 1 .. {MAX_BEAMS}")
    if num_blocks * block_size >= 1 << 31 or max_blocks * block_size >= 1 << 31 or max_blocks > _MOST:
        raise ValueError("a pool or a table of more than 2^31 slots")


def _state_arrays(block_tables, context_lens, free_blocks, max_blocks, block_size, num_blocks, group_size, held):
    """(context_lens and num_free, tables, reference counts, free blocks, shared blocks) of the host's lists."""
    rows = len(block_tables)
    _check_sizes(rows, max_blocks, block_size, num_blocks, group_size)
    if len(context_lens) != rows:
        raise ValueError("block_tables and context_lens need one entry per row")
    lens = np.fromiter(context_lens, np.int64, rows)
    if rows and lens.min() < 0:
        raise ValueError(f"context_lens[{int(lens.argmin())}] is {lens.min()}")
    need, have = -(-lens // block_size), np.fromiter(map(len, block_tables), np.int64, rows)
    if (need > max_blocks).any():
        b = int(np.argmax(need > max_blocks))
        raise IndexError(f"row {b} needs {need[b]} blocks, its table holds {max_blocks}")
    if (have < need).any():
        b = int(np.argmax(have < need))
        raise IndexError(f"row {b} needs {need[b]} blocks for {lens[b]} positions, table has {have[b]}")
    used = block_tables if (have == need).all() else [t[:n] for t, n in zip(block_tables, need)]
    tables = np.full((rows, max_blocks), -1, dtype=np.int32)
    ids = _ids("block_tables", itertools.chain.from_iterable(used), num_blocks)
    tables[np.arange(max_blocks) < need[:, None]] = ids
    refs = np.bincount(ids, minlength=num_blocks) + np.bincount(_ids("held", held, num_blocks), minlength=num_blocks)
    free = _ids("free_blocks", free_blocks, num_blocks)
    if free.size and (np.bincount(free).max() > 1 or (refs[free] > 0).any()):
        raise ValueError("free_blocks must be distinct blocks that no row holds")
    counted, stack = np.zeros(rows + 1, dtype=np.int32), np.zeros(num_blocks, dtype=np.int32)
    counted[:rows], counted[rows], stack[:free.size] = lens, free.size, free
    # leading whole blocks that the rows of a group with positions have in common
    groups = tables.reshape(rows // group_size, group_size, max_blocks)
    live = (lens > 0).reshape(rows // group_size, group_size)
    first = groups[np.arange(groups.shape[0]), live.argmax(1)]
    whole = np.where(live, lens.reshape(rows // group_size, group_size) // block_size, max_blocks).min(1, initial=max_blocks)
    agree = ((groups == first[:, None]) | ~live[:, :, None]).all(1) & (np.arange(max_blocks) < whole[:, None])
    shared = np.where(live.any(1), np.cumprod(agree, axis=1).sum(1), 0)
    return counted, tables, refs.astype(np.int32), stack, shared.astype(np.int32)


def _ids(name: str, x, num_blocks: int) -> np.ndarray:
    a = np.fromiter(x, np.int64)
    if a.size and (a.min() < 0 or a.max() >= num_blocks):
        raise IndexError(f"{name} holds a block id outside [0, {num_blocks})")
    return a


def build_device_step(tables: DeviceTables, new_lens: torch.Tensor, step: DeviceStep) -> DeviceStep:
    """Row b gets new_lens[b] (int32, on the GPU) tokens behind its cached positions: the blocks they need
    are taken from the free blocks, and the step's arrays are filled (tb_beam_step). ``tables`` keeps
    its lengths and free blocks until tables.take(step) or reorder_beams(..., step=step), so a step may be
    built again; a request of which an empty row gets tokens shares no block from here to its next reordering.
    Where something does not fit the step is empty (tables.check() raises)."""
    device, rows = tables.device, tables.num_rows
    _ints("new_lens", new_lens, torch.int32, (rows,), device)
    if step.context_lens.device != device or step.context_lens.shape[0] != rows:
        raise ValueError("the step was made for other tables (DeviceTables.new_step)")
    if _elsewhere(device):
        with torch.cuda.device(device):
            return build_device_step(tables, new_lens, step)
    L, stream, p = _lib.lib(), _lib.stream_handle(device), tables._ptr
    need = L.tb_device_step_workspace_bytes(rows)
    lock = ws = None
    if need:
        lock, ws, _, _, _ = _scratch(device, stream, need, 0)
    try:
        st = L.tb_beam_step(p["block_tables"], tables.max_blocks, p["context_lens"], new_lens.data_ptr(), rows,
                            p["shared_blocks"], tables.group_size, p["ref_counts"], p["free_blocks"], p["num_free"],
                            tables.num_blocks, tables.block_size, *step._args, p["status"],
                            None if ws is None else ws.data_ptr(), need, stream)
    finally:
        if lock is not None:
            lock.release()
    _lib.check(st, "tb_beam_step")
    return step
