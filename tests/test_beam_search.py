"""Beam search's bookkeeping (tinybatch_amd/beam_search.py) without a GPU: the block manager before and after searches that
fail, with a prefill that stands in for the model's."""
from types import SimpleNamespace

import pytest

from tinybatch_amd import beam_search as bs
from tinybatch_amd.block_manager import BlockManager, OutOfBlocks


class Failed(Exception):
    pass


def search(blocks, prompts, num_beams=3, max_new=8, **kw):
    model = SimpleNamespace(cfg=SimpleNamespace(vocab_size=500))
    cache = SimpleNamespace(block_size=blocks.block_size, num_blocks=blocks.num_blocks, device="cpu")
    return bs.beam_search(model, cache, blocks, prompts, num_beams=num_beams, max_new=max_new, **kw)


def fail(*_, **__):
    raise Failed


PROMPT = list(range(70))


def test_a_failed_prefill_leaves_nothing_in_the_prefix_cache(monkeypatch):
    """Full blocks are found by their tokens before they are written: where they never were, nobody may find them."""
    blocks = BlockManager(100, 16)
    other, _ = blocks.allocate_prompt(PROMPT[:32])                    # served to its end: found before and after
    blocks.free_table(other)
    monkeypatch.setattr(bs, "prefill", fail)
    # (the second prompt finds the first one's blocks, the third its own prefix alone)
    with pytest.raises(Failed):
        search(blocks, [PROMPT, PROMPT[:64] + [7] * 20, PROMPT[:48] + [9] * 20])
    assert blocks.num_free() == 100 and sorted(blocks.cache.values()) == sorted(other[:2])
    assert all(b.prefix_hash is None for b in blocks.blocks if b.block_id not in other)
    hits = blocks.prefix_hits
    table, cached = blocks.allocate_prompt(PROMPT)
    assert cached == 32 and blocks.prefix_hits == hits + 2
    blocks.free_table(table)


def test_blocks_that_others_found_first_stay_theirs(monkeypatch):
    """A request in flight holds the prompt's first blocks: they stay in the cache and in its table."""
    blocks = BlockManager(60, 16)
    held, _ = blocks.allocate_prompt(PROMPT[:33])
    monkeypatch.setattr(bs, "prefill", fail)
    for _ in range(3):
        with pytest.raises(Failed):
            search(blocks, [PROMPT])
    assert [blocks.blocks[b].ref_count for b in held] == [1, 1, 1]
    assert sorted(blocks.cache.values()) == sorted(held[:2])
    blocks.free_table(held)
    assert blocks.num_free() == 60


def test_a_search_that_fails_behind_its_prefill_keeps_the_prompts(monkeypatch):
    """The prompts' K/V are there: what is found by them is right."""
    blocks = BlockManager(100, 16)
    monkeypatch.setattr(bs, "prefill", lambda *_: None)
    monkeypatch.setattr(bs.DeviceTables, "from_lists", fail)
    with pytest.raises(Failed):
        search(blocks, [PROMPT])
    assert blocks.num_free() == 100 and blocks.allocate_prompt(PROMPT)[1] == 64


def test_unpublish():
    blocks = BlockManager(10, 4)
    table, _ = blocks.allocate_prompt(list(range(10)))
    blocks.unpublish(table)                                           # two full blocks and one that is not
    assert not blocks.cache and [blocks.blocks[b].ref_count for b in table] == [1, 1, 1]
    again, cached = blocks.allocate_prompt(list(range(10)))
    assert cached == 0 and not set(again) & set(table)
    blocks.unpublish(table)                                           # whose tokens another block is found by: that one stays
    assert sorted(blocks.cache.values()) == sorted(again[:2])
    blocks.free_table(table)
    blocks.free_table(again)
    assert blocks.num_free() == 10 and len(blocks.free_ids) == 8


def test_a_prompt_that_can_never_fit_is_told_before_any_search(monkeypatch):
    """Behind prompts that fit, which are searched in turns: nothing is computed and thrown away."""
    blocks, calls = BlockManager(40, 16), []
    monkeypatch.setattr(bs, "prefill", lambda *_: calls.append(1))
    monkeypatch.setattr(bs.DeviceTables, "from_lists", fail)
    with pytest.raises(OutOfBlocks, match="prompt of 560 tokens"):
        search(blocks, [PROMPT, PROMPT[:20], list(range(560))], num_beams=4)
    assert not calls and blocks.num_free() == 40 and not blocks.cache
    with pytest.raises(Failed):                                       # 36 of 40 blocks: searched
        search(blocks, [list(range(24 * 16))], num_beams=4)
    assert calls == [1] and blocks.num_free() == 40
