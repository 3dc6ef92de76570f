"""Steps that make a prefix and read it (two prompts on one prefix, admitted together): which ones the builder tells
(StepMetadata.reads_new), and that they take the separate append."""
import numpy as np
import pytest

from tinybatch_amd.block_manager import BlockManager
from tinybatch_amd.kv_cache import PagedKVCache
from tinybatch_amd.metadata import PrefillRoute, build_step_metadata


def step(seqs, bs=16, nb=64, route=None):
    """seqs: (table, cached positions, new rows)."""
    pos, slices = [], []
    for _, c, n in seqs:
        slices.append((len(pos), len(pos) + n))
        pos += range(c, c + n)
    return build_step_metadata(pos, slices, [t for t, _, _ in seqs], [c + n for _, c, n in seqs], block_size=bs, num_blocks=nb,
                               partition_tokens=256, prefill_route=route)


ROUTE = PrefillRoute(2, 64, 576)


@pytest.mark.parametrize("told,seqs", [
    (True, [([0, 1, 2], 0, 40), ([0, 1, 3, 4], 32, 20)]),              # a prefix that the first sequence makes
    (True, [([0, 1, 3, 4], 32, 20), ([0, 1, 2], 0, 40)]),              # in either order
    (True, [([0, 1, 2], 16, 24), ([0, 1, 3, 4], 32, 20)]),             # the second block of it
    (True, [([0, 1], 0, 32), ([0, 1, 2], 32, 1)]),                     # read by one row
    (True, [([0, 1], 16, 1), ([0, 1], 17, 1)]),                        # a shared block that is not full
    (False, [([0, 1], 17, 1), ([0, 1], 16, 1)][:1]),
    (False, [([0, 1, 2], 32, 8), ([0, 1, 3, 4], 32, 20)]),             # a prefix that was there
    (False, [([0, 1, 2], 0, 40), ([3, 4, 5], 0, 40)]),
    (False, [([0, 1, 2], 0, 40)]),
    (False, [([0, 1, 2, 9], 40, 20), ([3, 1, 2], 16, 0)]),             # no new rows: reads nothing
    (False, [([0, 1, 2, 9], 37, 20), ([3, 4, 5, 6], 37, 20)]),         # own blocks that are not full
    (True, [([0, 1], 16, 9), ([2, 1, 3], 32, 3)]),                     # a block of it at another place
])
def test_steps_that_read_what_they_write(told, seqs):
    for route in (None, ROUTE):
        m = step(seqs, route=route)
        assert m.reads_new is told
        assert not (told and PagedKVCache._fusable(m))
    if len(seqs) > 1 and not told and all(n >= 16 for _, _, n in seqs):
        assert PagedKVCache._fusable(step(seqs, route=ROUTE))


def test_blocks_of_one_position():
    assert step([([0, 1, 2], 2, 1), ([0, 1, 2, 3], 3, 1)], bs=1).reads_new
    assert not step([([0, 1, 2], 2, 1), ([0, 1, 4, 3], 3, 1)], bs=1).reads_new


def test_prompts_of_the_block_manager():
    """Two prompts on one prefix in one step, then in two; a prompt that was there whole (its last position is written again)."""
    bm = BlockManager(64, 16)
    prefix = list(range(48))
    a, na = bm.allocate_prompt(prefix + [1] * 20)
    b, nb = bm.allocate_prompt(prefix + [2] * 30)
    assert (na, nb) == (0, 48)
    assert step([(a, 0, 68), (b, 48, 30)]).reads_new
    assert not step([(a, 0, 68)]).reads_new and not step([(b, 48, 30)]).reads_new
    c, nc = bm.allocate_prompt(prefix)
    assert nc == 48 and step([(c, 47, 1), (b, 78, 1)]).reads_new and not step([(a, 68, 1), (b, 78, 1)]).reads_new


@pytest.mark.parametrize("seed", range(30))
def test_random_steps(seed):
    """Against a look at every slot."""
    g = np.random.default_rng(seed)
    bs, seqs = int(g.choice([1, 2, 16])), []
    for _ in range(int(g.integers(2, 5))):
        c, n = int(g.integers(0, 5 * bs)), int(g.integers(0, 3 * bs))
        seqs.append((g.permutation(40)[:-(-(c + n) // bs) + 1].tolist(), c, n))
    slot = lambda t, p: t[p // bs] * bs + p % bs
    writes = [{slot(t, p) for p in range(c, c + n)} for t, c, n in seqs]
    reads = [{slot(t, p) for p in range(c)} if n else set() for t, c, n in seqs]
    want = any(reads[i] & writes[j] for i in range(len(seqs)) for j in range(len(seqs)))
    assert step(seqs, bs).reads_new is want
