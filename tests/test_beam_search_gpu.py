"""Beam search on the engine (tinybatch_amd/beam_search.py): the operators run together, step after step, against a plain
search that runs the CPU restatement of the model on every beam's whole sequence."""
import math

import pytest
import torch

from oracle import model_reference as mref
from test_engine_gpu import cpu_weights, small_cfg
from tinybatch_amd.block_manager import OutOfBlocks
from tinybatch_amd.config import EngineConfig
from tinybatch_amd.engine import LLMEngine

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def engine(dtype="float32", seed=3, mc=None, **kw):
    kw = {"num_blocks": 400, "max_model_len": 300, "max_batch_tokens": 512, **kw}
    return LLMEngine(EngineConfig(dtype=dtype, seed=seed, **kw), mc or small_cfg(layers=2, heads=4, kv_heads=2, vocab=500))


def sharpen(eng, by=40.0):
    """Weights that give logits of some spread: the candidates' gaps are then far above fp32's errors."""
    eng.model.norm.mul_(by)
    return eng


def log_probs(w, mc, sequences):
    """[n, vocab]: log-probabilities after every sequence, each run whole over a pool of its own."""
    out = []
    for ids in sequences:
        nb = -(-len(ids) // 16)
        pools = [torch.zeros(nb, 2, mc.n_kv_heads, 16, mc.head_dim) for _ in range(mc.n_layers)]
        logits = mref.forward(w, mc, torch.tensor(ids), torch.arange(len(ids)), [(0, len(ids))], [list(range(nb))],
                              [len(ids)], pools, 16)
        out.append(torch.log_softmax(logits[0].double(), -1))
    return torch.stack(out)


def plain_search(w, mc, prompt, K, max_new, eos=()):
    """[(tokens, score)], best first: beams that have ended stand with their score."""
    beams = [([], 0.0)]
    for _ in range(max_new):
        if all(b[0] and b[0][-1] in eos for b in beams):
            break
        found = []
        for k, (ids, s) in enumerate(beams):
            if ids and ids[-1] in eos:
                found.append((-s, k, eos[0], ids, s))
                continue
            lp = log_probs(w, mc, [prompt + ids])[0]
            for v in lp.topk(min(2 * K, lp.numel())).indices.tolist():
                found.append((-(s + float(lp[v])), k, v, ids + [v], s + float(lp[v])))
        found.sort(key=lambda x: x[:3])
        beams = [(ids, s) for _, _, _, ids, s in found[:K]]
    return beams


def check(eng, prompts, K, max_new, eos=(), penalty=1.0):
    w, mc = cpu_weights(eng.model), eng.model.cfg
    free = eng.block_manager.num_free()
    got = eng.beam_search(prompts, num_beams=K, max_new_tokens=max_new, length_penalty=penalty, num_return=K)
    for prompt, found in zip(prompts, got):
        want = plain_search(w, mc, prompt, K, max_new, eos)
        want = sorted(want, key=lambda x: -(x[1] / len(x[0]) ** penalty))
        assert [r.token_ids for r in found] == [ids for ids, _ in want]
        # a step's log-probabilities are fp32 logits of two layers' sums apart: 2e-4 a token as the engine's other tests
        assert all(abs(r.score - s) <= 2e-3 * len(ids) for r, (ids, s) in zip(found, want))
        assert all(abs(r.value - r.score / len(r.token_ids) ** penalty) < 1e-9 for r in found)
    assert eng.block_manager.num_free() == free
    return got


def random_prompts(seed, lens, vocab=500):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g).tolist() for n in lens]


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("K,by", [(1, 40.0), (3, 10.0), (4, 40.0), (6, 12.0)])
def test_search_follows_the_plain_one(K, by, graphs):
    """Prompts that end inside a block, on its end and of one token; tokens past two blocks."""
    eng = sharpen(engine(decode_graphs=graphs), by)
    check(eng, random_prompts(K, [5, 32, 1, 47]), K, 20)


def test_search_with_end_tokens_and_penalties():
    eng = sharpen(engine())
    prompts = random_prompts(9, [12, 30])
    plain = eng.beam_search(prompts, num_beams=4, max_new_tokens=12, num_return=4)
    ends = tuple({plain[0][0].token_ids[3], plain[1][1].token_ids[5]})
    eng.eos_ids, eng.cfg.stop_token_ids = set(ends), ends
    for penalty in (0.0, 1.0, 2.0):
        got = check(eng, prompts, 4, 12, ends, penalty)
        assert any(len(r.token_ids) < 12 for found in got for r in found)


def test_search_that_ends_early():
    """Every token ends a beam: after the first one nothing is left to do."""
    eng = sharpen(engine())
    eng.eos_ids, eng.cfg.stop_token_ids = set(range(500)), tuple(range(500))
    got = eng.beam_search(random_prompts(2, [7]), num_beams=3, max_new_tokens=40, num_return=3)
    assert [len(r.token_ids) for r in got[0]] == [1, 1, 1]


def test_more_beams_than_tokens():
    mc = small_cfg(layers=1, heads=2, kv_heads=1, vocab=5)
    eng = sharpen(engine(mc=mc))
    check(eng, [[1, 2, 3]], 5, 4)
    got = eng.beam_search([[1, 2, 3]], num_beams=8, max_new_tokens=1, num_return=8)
    assert len(got[0]) == 5                        # the others found nothing left


def test_searches_that_share_the_prefix_cache():
    """Prompts on one prefix, found in the cache from the second on; the engine's own requests between."""
    eng = sharpen(engine())
    prefix = random_prompts(4, [64])[0]
    prompts = [prefix + p for p in random_prompts(5, [3, 16, 1])]
    check(eng, prompts, 3, 8)
    hits = eng.block_manager.prefix_hits
    outs = eng.generate([prefix + [7]], max_new_tokens=3)
    assert eng.block_manager.prefix_hits > hits and len(outs[0]) == 3
    check(eng, prompts, 3, 8)


def test_search_in_the_blocks_there_are():
    """More prompts than the free blocks allow at once are searched in turn; one that does not fit is refused."""
    eng = sharpen(engine(num_blocks=30))
    check(eng, random_prompts(6, [20, 33, 16, 40]), 4, 10)
    with pytest.raises(OutOfBlocks):
        eng.beam_search(random_prompts(6, [20]), num_beams=8, max_new_tokens=100)
    assert eng.block_manager.num_free() == 30
    for bad in (dict(num_beams=0), dict(num_beams=65), dict(num_beams=2, num_return=3), dict(max_new_tokens=0),
                dict(max_new_tokens=290)):
        with pytest.raises(ValueError):
            eng.beam_search([[1] * 20], **{"num_beams": 2, "max_new_tokens": 4, **bad})
    with pytest.raises(ValueError):
        eng.beam_search([[]], num_beams=2, max_new_tokens=4)
    assert eng.beam_search([], num_beams=2, max_new_tokens=4) == []


@pytest.mark.parametrize("block_size", [8, 16])
def test_search_in_small_blocks(block_size):
    """Blocks that beam_attention does not serve take the work items of the step that was built on the GPU."""
    eng = sharpen(engine(block_size=block_size))
    check(eng, random_prompts(8, [9, 24]), 3, 12)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_search_in_16_bits(dtype):
    """Scores of the tokens that were found, by the model on the whole sequence: within the logits' rounding (2^-8 or 2^-11 of
    their size, twice a token for the two runs)."""
    # (a prompt found in the cache is prefilled by another kernel, whose roundings differ: none here)
    eng = sharpen(engine(dtype=dtype, enable_prefix_caching=False), 10.0)
    prompts = random_prompts(11, [17, 40])
    step = 2.0 ** (-8 if dtype == "bfloat16" else -11)
    for graphs in (False, True):
        eng.cfg.decode_graphs = graphs
        got = eng.beam_search(prompts, num_beams=4, max_new_tokens=10, num_return=4)
        w = cpu_weights(eng.model)
        for prompt, found in zip(prompts, got):
            assert len({tuple(r.token_ids) for r in found}) == 4
            assert [r.score for r in found] == sorted((r.score for r in found), reverse=True)
            for r in found:
                score = 0.0
                for i in range(len(r.token_ids)):
                    lp = log_probs(w, eng.model.cfg, [prompt + r.token_ids[:i]])[0]
                    score += float(lp[r.token_ids[i]])
                assert abs(score - r.score) <= 2 * step * 40 * len(r.token_ids), (score, r.score)
        if graphs:
            assert got == first
        first = got


def test_prompts_of_a_search_that_failed_are_not_found(monkeypatch):
    """The second of two prompts' forward passes fails: the next calls compute both prompts again, to the right tokens."""
    eng = sharpen(engine(max_batch_tokens=64))
    prompts = random_prompts(13, [50, 64])
    forward, calls = eng.model.forward, []

    def failing(*args):
        calls.append(args)
        if len(calls) == 2:
            raise RuntimeError("out of memory")
        return forward(*args)

    monkeypatch.setattr(eng.model, "forward", failing)
    with pytest.raises(RuntimeError, match="out of memory"):
        eng.beam_search(prompts, num_beams=3, max_new_tokens=6)
    assert len(calls) == 2 and eng.block_manager.num_free() == 400
    out = eng.generate([prompts[1]], max_new_tokens=2)
    assert eng.block_manager.prefix_hits == 0
    assert out[0][0] == int(log_probs(cpu_weights(eng.model), eng.model.cfg, [prompts[1]])[0].argmax())
    check(eng, prompts, 3, 6)
    assert eng.block_manager.prefix_hits == 4      # the second prompt's blocks, which generate() wrote


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_loop_of_ones_own(dtype):
    """The loop of the integration notes on the model's layers, its requests with beams that end on the way: the engine's search."""
    from tinybatch_amd import BeamPlan, DeviceTables, beam_attention, build_device_step, ops, reorder_beams, select_beams

    eng = sharpen(engine(dtype, decode_graphs=False, enable_prefix_caching=False), 12.0)
    m, cache, mc, K, new = eng.model, eng.kv_cache, eng.model.cfg, 3, 14
    prompts = random_prompts(21, [30, 45])
    plain = eng.beam_search(prompts, num_beams=K, max_new_tokens=new, num_return=K)
    eos = plain[0][0].token_ids[4]
    eng.eos_ids, eng.cfg.stop_token_ids = {eos}, (eos,)
    want = eng.beam_search(prompts, num_beams=K, max_new_tokens=new, num_return=K, length_penalty=0.0)
    assert any(len(r.token_ids) < new for found in want for r in found)
    blocks, logits = [], []
    for p in prompts:
        table = eng.block_manager.allocate_private(-(-len(p) // 16), p)
        blocks.append(table)
        logits.append(m.forward(torch.tensor(p, device=DEV), torch.arange(len(p), device=DEV), [(0, len(p))], [table], [len(p)], cache))
    free = eng.block_manager.allocate_private(40, [])
    tables = DeviceTables.from_lists([t for b in blocks for t in (b, [], [])], [n for p in prompts for n in (len(p), 0, 0)], free,
                                     max_blocks=6, block_size=16, num_blocks=cache.num_blocks, group_size=K, device=DEV)
    step = tables.new_step(padded=1)
    plan = BeamPlan(tables, num_heads=mc.n_heads, num_kv_heads=mc.n_kv_heads, head_dim=mc.head_dim, dtype=cache.dtype)
    choice = select_beams(torch.cat(logits), torch.zeros(2, 1, device=DEV), num_candidates=K)
    reorder_beams(cache.storage, tables, choice.parents)
    finished = choice.tokens == eos
    told = [choice]
    for _ in range(new - 1):
        live = ~finished & (choice.scores > -float("inf"))
        build_device_step(tables, live.view(-1).int(), step)
        plan.build(step.row_ctx)

        def attention(i, q, k, v):
            ops.kv_append(cache.pools[i], k, v, step.slot_mapping)
            return beam_attention(q, cache.pools[i], plan)

        x = m.run_layers(choice.tokens.view(-1).clamp(min=0), step.positions, attention)
        choice = select_beams((x @ m.lm_head.T).float(), choice.scores, finished=finished, end_token=eos)
        reorder_beams(cache.storage, tables, choice.parents, step)
        finished = finished.gather(1, choice.parents.clamp(min=0).long()) & (choice.parents >= 0) | (choice.tokens == eos)
        told.append(choice)
    tables.check()
    for g, found in enumerate(want):
        got = []
        for k in range(K):
            ids, at = [], k
            for c in reversed(told):
                ids.append(int(c.tokens[g, at]))
                at = int(c.parents[g, at])
            ids.reverse()
            got.append((float(choice.scores[g, k]), ids[:ids.index(eos) + 1] if eos in ids else ids))
        if dtype == "float32":
            assert [ids for _, ids in got] == [r.token_ids for r in found]
            assert all(abs(s - r.score) <= 2e-3 * len(ids) for (s, ids), r in zip(got, found))
        else:                                      # (other products of the LM head: near candidates may change places)
            assert max(s for s, _ in got) >= found[0].score - 2 * 2.0 ** -8 * 40 * new
