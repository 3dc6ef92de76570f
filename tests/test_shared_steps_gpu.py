"""Steps that make a prefix and read it: prompts on one prefix, admitted together, give what they give one after the other."""
import pytest
import torch

from test_beams_gpu import check_attention
from test_engine_gpu import small_cfg
from tinybatch_amd import PagedKVCache, ops
from tinybatch_amd.config import EngineConfig
from tinybatch_amd.engine import LLMEngine

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def rows(seqs):
    pos, slices = [], []
    for _, c, n in seqs:
        slices.append((len(pos), len(pos) + n))
        pos += range(c, c + n)
    return torch.tensor(pos, device=DEV), slices, [t for t, _, _ in seqs], [c + n for _, c, n in seqs]


# (table, cached positions, new rows): prompts on the first one's prefix; the same, read by single rows; beside a decoding row
STEPS = {
    "prefills": [(list(range(20)), 0, 310), (list(range(19)) + [30, 31], 304, 25), (list(range(10)) + list(range(40, 46)), 160, 90)],
    "single rows": [(list(range(8)), 0, 128), (list(range(8)) + [30], 128, 1), (list(range(4)) + [31], 64, 1)],
    "mixed": [([50, 51, 52], 40, 1), (list(range(12)), 16, 170), (list(range(11)) + [30, 31], 176, 17)],
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("name", STEPS)
def test_a_step_that_makes_a_prefix_and_reads_it(name, hq, hkv, d, dtype):
    seqs = STEPS[name]
    g = torch.Generator().manual_seed(hq)
    T = sum(n for _, _, n in seqs)
    q, k, v = (torch.randn(T, h, d, generator=g).to(dtype).to(DEV) for h in (hq, hkv, hkv))
    cache = PagedKVCache(1, 64, 16, hkv, d, DEV, dtype)
    # (what is there before: the cached positions that no row of the step makes; large, so that a stale read is seen)
    cache.pools[0].copy_((torch.randn(64, 2, hkv, 16, d, generator=g) * 50).to(dtype))
    start = cache.pools[0].clone()
    pos, slices, tables, ctx = rows(seqs)
    got = cache.append_attention(0, q, k, v, pos, slices, tables, ctx)
    want = start.clone()
    slots = torch.tensor([t[p // 16] * 16 + p % 16 for t, c, n in seqs for p in range(c, c + n)], dtype=torch.int32, device=DEV)
    ops.kv_append(want, k, v, slots)
    assert torch.equal(cache.pools[0], want)
    flat = [(t, p + 1) for t, c, n in seqs for p in range(c, c + n)]
    check_attention(got, q, want.cpu(), [t for t, _ in flat], [n for _, n in flat], hq)
    meta = cache.step_metadata(pos, slices, tables, ctx, cache.rows_per_item(hq), num_heads=hq)
    assert meta.reads_new
    if name == "prefills" and dtype != torch.float32:      # (at head dim 128 longer than the kernel that appends holds)
        with pytest.raises(ValueError, match="earlier positions" if d == 64 else "fused append"):
            ops.paged_attention(q, cache.pools[0], meta, num_heads=hq, k_new=k, v_new=v)
        assert torch.equal(cache.pools[0], want)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_requests_on_one_prefix_admitted_together(dtype):
    """K/V of all three prompts as a search or the engine's own requests leave them, against prompts served one at a time: two
    runs' K/V of a position differ by their products' roundings, a stale one by its whole size."""
    prefix = torch.randint(0, 500, (160,), generator=torch.Generator().manual_seed(1)).tolist()
    prompts = [prefix + [7] * 20, prefix + [9] * 40, prefix[:96] + [11] * 33]

    def kv(run):
        eng = LLMEngine(EngineConfig(dtype=dtype, seed=3, num_blocks=200, max_model_len=300, max_batch_tokens=1024),
                        small_cfg(layers=3, heads=4, kv_heads=2, vocab=500))
        run(eng)
        out = []
        for p in prompts:
            table, cached = eng.block_manager.allocate_prompt(p)      # (their full blocks are found)
            assert cached == len(p) // 16 * 16
            out.append(torch.stack([torch.cat([pool[b] for b in table[:cached // 16]], dim=2) for pool in eng.kv_cache.pools]))
        return [x.float().cpu() for x in out]

    alone = kv(lambda eng: [eng.generate([p], max_new_tokens=1) for p in prompts])
    for run in (lambda eng: eng.generate(prompts, max_new_tokens=1),
                lambda eng: eng.beam_search(prompts, num_beams=2, max_new_tokens=2)):
        for a, b in zip(alone, kv(run)):
            # a layer's K and V are sums over d_model products of rounded values, some tens of roundings in all; unwritten: 0
            assert (a - b).abs().max() <= 64 * torch.finfo(getattr(torch, dtype)).eps * a.abs().max()
