"""Beam search on the model over the paged cache (LLMEngine.beam_search).

The reference samples one continuation per request (src/tinybatch/engine.py:145-159). Here every prompt
is prefilled once, its ``num_beams`` best first tokens become its beams, and each step continues them
by one token: the operators of beams.py, with nothing read back between two steps. A beam that has
ended stays among the candidates with its score, which live beams of any length are measured against as it is (length_penalty
orders the results alone), so that the search may end early only when every beam has.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
import torch.nn.functional as F

from . import layer_ops, ops
from .beams import BeamPlan, beam_attention, reorder_beams, select_beams
from .block_manager import BlockManager, OutOfBlocks
from .device_tables import MAX_BEAMS, DeviceTables, build_device_step
from .kv_cache import PagedKVCache
from .model import Qwen2Paged

CHECK_EVERY = 16             # steps between two looks at whether every beam has ended


class BeamResult(NamedTuple):
    token_ids: list[int]     # the continuation, with its end token if it has ended
    score: float             # the sum of its tokens' log-probabilities
    value: float             # score / length ** length_penalty, by which a request's results are ordered


class BeamState:
    """The beams of some requests between two steps, all on the GPU."""

    def __init__(self, model: Qwen2Paged, cache: PagedKVCache, tables: DeviceTables, choice, eos_ids, max_new: int):
        c = model.cfg
        self.model, self.cache, self.tables, self.eos_ids = model, cache, tables, tuple(eos_ids)
        self.served = c.head_dim in (64, 128) and cache.block_size >= 16
        # geometries that beam_attention does not serve take paged_attention's work items, built on the GPU as well
        self.step = tables.new_step(padded=1, partition_tokens=0 if self.served else cache.partition_tokens)
        self.plan = BeamPlan(tables, num_heads=c.n_heads, num_kv_heads=c.n_kv_heads, head_dim=c.head_dim,
                             dtype=cache.dtype) if self.served else None
        shape, dev = choice.tokens.shape, choice.tokens.device
        self.tokens, self.scores = choice.tokens.clone(), choice.scores.clone()
        self.finished = self._ends(choice.tokens)
        self.hist_tokens = torch.full((max_new, *shape), -1, dtype=torch.int64, device=dev)
        self.hist_parents = torch.full((max_new, *shape), -1, dtype=torch.int32, device=dev)
        self.hist_tokens[0], self.hist_parents[0] = choice.tokens, choice.parents
        self.at = torch.ones(1, dtype=torch.int64, device=dev)

    def _ends(self, tokens: torch.Tensor) -> torch.Tensor:
        ends = torch.zeros_like(tokens, dtype=torch.bool)
        for e in self.eos_ids:
            ends |= tokens == e
        return ends

    def live(self) -> torch.Tensor:
        """[G, K]: beams that are there and have not ended."""
        return ~self.finished & (self.scores > -float("inf"))

    @torch.inference_mode()
    def advance(self) -> None:
        """One token for every live beam; the states follow the selection. Can be captured."""
        m, c, t, step = self.model, self.model.cfg, self.tables, self.step
        build_device_step(t, self.live().view(-1).to(torch.int32), step)
        if self.served:
            self.plan.build(step.row_ctx)
        meta = None if self.served else step.metadata(t)

        def attention(i, q, k, v):
            ops.kv_append(self.cache.pools[i], k, v, step.slot_mapping)
            if self.served:
                return beam_attention(q, self.cache.pools[i], self.plan)
            out = torch.zeros(q.shape[0], c.n_heads * c.head_dim, dtype=q.dtype, device=q.device)
            return ops.paged_attention(q, self.cache.pools[i], meta, num_heads=c.n_heads, out=out)

        x = m.run_layers(self.tokens.view(-1).clamp(min=0), step.positions, attention)
        logits = layer_ops.linear(x, m.lm_head) if m._streamed(x) and c.vocab_size % 16 == 0 else F.linear(x, m.lm_head)
        choice = select_beams(logits, self.scores, finished=self.finished,
                              end_token=self.eos_ids[0] if self.eos_ids else 0)
        reorder_beams(self.cache.storage, t, choice.parents, step)
        parents = choice.parents.clamp(min=0).long()
        self.finished.copy_(self.finished.gather(1, parents) & (choice.parents >= 0) | self._ends(choice.tokens))
        self.tokens.copy_(choice.tokens)
        self.scores.copy_(choice.scores)
        self.hist_tokens.index_copy_(0, self.at, choice.tokens[None])
        self.hist_parents.index_copy_(0, self.at, choice.parents[None])
        self.at.add_(1)

    def run(self, steps: int, graph: bool) -> None:
        """``steps`` further tokens, fewer where every beam has ended; from the second on as replays of one captured step."""
        captured = None
        for i in range(steps):
            if i % CHECK_EVERY == 0 and not bool(self.live().any()):
                return
            if captured is not None:
                captured.replay()
                continue
            self.advance()
            # (a capture takes 3 to 5 ms, a replay saves 1 to 1.5: on the 0.5B model a search of 6 tokens, one prompt of 4 beams,
            # 12.8 ms captured and 13.9 not, of 8 tokens 15.0 and 18.1; 32 prompts of 8 beams 29.9 and 31.0, 36.2 and 40.5)
            if graph and steps - i > 4:
                stream = torch.cuda.Stream(device=self.tables.device)
                torch.cuda.synchronize(self.tables.device)
                captured = torch.cuda.CUDAGraph()
                with torch.cuda.graph(captured, stream=stream):
                    self.advance()                 # recorded, not run

    def results(self, length_penalty: float, count: int) -> list[list[BeamResult]]:
        """The ``count`` best of every request's beams (synchronises)."""
        self.tables.check()
        steps = int(self.at)
        tokens, parents = self.hist_tokens[:steps].cpu(), self.hist_parents[:steps].cpu()
        scores = self.scores.cpu()
        out = []
        for g in range(scores.shape[0]):
            found = []
            for k in range(scores.shape[1]):
                if scores[g, k] == -float("inf"):
                    continue
                ids, at = [], k
                for t in range(steps - 1, -1, -1):
                    ids.append(int(tokens[t, g, at]))
                    at = int(parents[t, g, at])
                ids.reverse()
                end = next((i for i, x in enumerate(ids) if x in self.eos_ids), len(ids) - 1)
                ids, score = ids[:end + 1], float(scores[g, k])
                found.append(BeamResult(ids, score, score / len(ids) ** length_penalty))
            found.sort(key=lambda r: -r.value)     # (stable: the search's own order among equals)
            out.append(found[:count])
        return out


def prefill(model: Qwen2Paged, cache: PagedKVCache, prompts, tables, cached, budget: int) -> torch.Tensor:
    """Logits [prompts, vocab] after every prompt, its K/V in the cache: prompts of up to ``budget`` new tokens together."""
    device, rows, at = cache.device, [], 0
    guard = ops.decode_device(device)
    while at < len(prompts):
        end, new = at, 0
        while end < len(prompts) and (end == at or new + len(prompts[end]) - cached[end] <= budget):
            new += len(prompts[end]) - cached[end]
            end += 1
        ids, pos, slices = [], [], []
        for p, c in zip(prompts[at:end], cached[at:end]):
            slices.append((len(ids), len(ids) + len(p) - c))
            ids += p[c:]
            pos += range(c, len(p))
        ids, positions = torch.tensor(ids).to(device), torch.tensor(pos).to(device)
        ctx, hq = [len(p) for p in prompts[at:end]], model.cfg.n_heads
        for attempt in range(2):                   # (as the engine's eager step: in-launch merges may report an error)
            cache.step_metadata(positions, slices, tables[at:end], ctx, cache.rows_per_item(hq), host_positions=pos,
                                num_heads=hq)
            logits = model.forward(ids, positions, slices, tables[at:end], ctx, cache)
            if guard.errors() == 0:
                break
            if attempt:
                raise RuntimeError("attention kept reporting merge errors with in-launch merges switched off")
            guard.disable_merges()
            cache.clear_metadata()
        rows.append(logits)
        at = end
    return torch.cat(rows)


def beam_search(model: Qwen2Paged, cache: PagedKVCache, blocks: BlockManager, prompts, *, num_beams: int, max_new: int,
                eos_ids=(), length_penalty: float = 1.0, num_return: int = 1, budget: int = 2048,
                graph: bool = True) -> list[list[BeamResult]]:
    """The ``num_return`` best of ``num_beams`` beams for every prompt (token ids), of up to ``max_new`` tokens. Blocks
    for the beams come from ``blocks`` and go back to it; as many prompts as its free blocks allow are searched together. A
    prompt that does not fit by itself raises OutOfBlocks before anything is computed."""
    if not 1 <= num_beams <= MAX_BEAMS or not 1 <= num_return <= num_beams or max_new < 1:
        raise ValueError(f"1 .. {MAX_BEAMS} beams, of which as many are returned at most, and one new token at least")
    vocab = model.cfg.vocab_size
    if any(not 0 <= e < vocab for e in eos_ids):
        raise ValueError("an end token outside the vocabulary")
    if any(not len(p) for p in prompts):
        raise ValueError("empty prompt")
    # a beam's own blocks: its tokens', the copy of the prompt's last block, and one more while a selection copies
    own = blocks.blocks_needed(max_new) + 2
    needs = [blocks.blocks_needed(len(p)) + num_beams * own for p in prompts]
    for p, need in zip(prompts, needs):            # (every turn gives its blocks back: what fits now fits then)
        if need > blocks.num_free():
            raise OutOfBlocks(f"a prompt of {len(p)} tokens with {num_beams} beams needs {need} blocks, "
                              f"{blocks.num_free()} are free")
    done: list[list[BeamResult]] = []
    while len(done) < len(prompts):
        some, tables, cached, spare, made = [], [], [], [], []
        written = False
        try:
            for p, need in zip(prompts[len(done):], needs[len(done):]):
                if need > blocks.num_free() or (len(some) + 1) * num_beams > 65535:
                    break
                table, n = blocks.allocate_prompt(list(p))
                tables.append(table)
                made.append(table[n // blocks.block_size:])
                spare.append(blocks.allocate_private(num_beams * own, []))
                some.append(list(p))
                cached.append(min(n, len(p) - 1))
            logits = prefill(model, cache, some, tables, cached, budget)
            written = True
            rows, lens = [], []
            for t, p in zip(tables, some):         # the prompt in a request's first row; its beams follow from there
                rows += [t] + [[]] * (num_beams - 1)
                lens += [len(p)] + [0] * (num_beams - 1)
            longest = max(map(len, some)) + max_new
            state = DeviceTables.from_lists(rows, lens, [b for s in reversed(spare) for b in reversed(s)],
                                            max_blocks=blocks.blocks_needed(longest), block_size=cache.block_size,
                                            num_blocks=cache.num_blocks, device=cache.device, group_size=num_beams,
                                            held=[b for t in tables for b in t])
            first = select_beams(logits, torch.zeros(len(some), 1, device=cache.device), num_candidates=num_beams)
            reorder_beams(cache.storage, state, first.parents)
            search = BeamState(model, cache, state, first, eos_ids, max_new)
            search.run(max_new - 1, graph)
            done += search.results(length_penalty, num_return)
        finally:
            if not written:                        # nobody may find the prompts' blocks, whose K/V are not there
                for t in made:
                    blocks.unpublish(t)
            for t in tables + spare:
                blocks.free_table(t)
    return done
