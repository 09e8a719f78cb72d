"""Forked requests on the CPU: shared pages and their counts, the copied page, and several completions of one prompt."""
import random

import pytest
import torch

import kv4_plain as P
from configs import TINY_B
from iitj_llm_coopt_b200 import EngineConfig, LLM, LlamaConfig, SamplingParams, build_engine
from iitj_llm_coopt_b200.cache import CacheManager, OutOfPages
from iitj_llm_coopt_b200.cache.manager import CacheError
from iitj_llm_coopt_b200.config.specs import CacheNeed

FULL = CacheNeed("paged_kv", kv_heads=2, head_dim=32)
WIN = CacheNeed("paged_kv", kv_heads=2, head_dim=32, window=6)


def test_a_fork_holds_the_same_full_pages_and_a_copy_of_the_last():
    cm = CacheManager([FULL, FULL], 4, 10, 3)
    cm.admit("a")
    cm.ensure("a", 11)
    cm.advance("a", 11)
    copies = cm.fork("a", "b", 10)
    a, b = cm.table(0, "a"), cm.table(0, "b")
    assert b[:2] == a[:2] and b[2] not in a and copies == [(0, a[2], b[2])]
    assert cm.num_tokens("b") == 10 and cm.num_free == 10 - 4
    cm.check()
    assert cm.release("a") == 1                       # only its own last page: the fork still holds the others
    cm.check()
    cm.ensure("b", 13)
    cm.advance("b", 13)
    assert cm.release("b") == 4 and cm.num_free == 10
    cm.check()


def test_a_fork_at_a_page_end_copies_nothing():
    cm = CacheManager([FULL], 4, 4, 3)
    cm.admit(0)
    cm.ensure(0, 8)
    cm.advance(0, 8)
    assert cm.fork(0, 1, 8) == [] and cm.table(0, 1) == cm.table(0, 0)
    assert cm.fork(1, 2, 4) == [] and cm.table(0, 2) == cm.table(0, 0)[:1]
    cm.check()
    with pytest.raises(CacheError, match="fork shares"):
        cm.truncate(0, 6)                             # the next token would be written where request 1 reads
    cm.truncate(0, 4)
    cm.check()
    for r in (0, 2, 1):
        cm.release(r)
    assert cm.num_free == 4


def test_what_cannot_be_forked_is_refused_and_changes_nothing():
    cm = CacheManager([FULL], 4, 3, 2)
    cm.admit(0)
    cm.ensure(0, 9)
    cm.advance(0, 9)
    assert not cm.can_fork(0, 9) and not cm.can_fork(0, 10) and not cm.can_fork(0, 0) and not cm.can_fork("x", 1)
    with pytest.raises(CacheError, match="cannot be forked"):
        cm.fork(0, 1, 9)                              # no page for the copy
    assert cm.can_fork(0, 8)
    cm.fork(0, 1, 8)
    with pytest.raises(CacheError, match="already admitted"):
        cm.fork(0, 1, 8)
    assert not cm.can_fork(0, 4)                      # no slot
    cm.check()
    state = CacheManager([FULL, CacheNeed("state", state_shape=(2,))], 4, 8, 3)
    state.admit(0)
    state.ensure(0, 8)
    state.advance(0, 8)
    assert not state.can_fork(0, 8)                   # a state holds all tokens: it cannot be shared
    win = CacheManager([FULL, WIN], 4, 16, 3)
    win.admit(0)
    win.ensure(0, 16)
    win.advance(0, 16)
    assert win.can_fork(0, 16) and win.can_fork(0, 15) and not win.can_fork(0, 12)     # pages that its window passed are gone
    win.fork(0, 1, 15)
    win.check()
    win.ensure(1, 20)
    win.advance(1, 20)
    win.check()
    win.release(0)
    win.check()
    win.release(1)
    assert win.num_free == 16


@pytest.mark.parametrize("seed", range(4))
def test_random_forks_lose_no_page(seed):
    rng = random.Random(seed)
    cm = CacheManager([FULL, WIN, FULL], 4, 40, 8, max_step_tokens=12)
    sizes = {g: cm.groups[g].pool.num_pages for g in cm.paged}
    live, nxt = {}, 0
    for _ in range(400):
        op = rng.random()
        if op < 0.2 and len(live) < 8:
            cm.admit(nxt)
            live[nxt] = 0
            nxt += 1
        elif op < 0.45 and live and len(live) < 8:
            parent = rng.choice(list(live))
            n = rng.randint(1, max(1, live[parent]))
            if cm.can_fork(parent, n):
                for g, src, dst in cm.fork(parent, nxt, n):
                    assert src != dst and cm.groups[g].pool.holders[dst] == 1
                live[nxt] = n
                nxt += 1
        elif op < 0.85 and live:
            r = rng.choice(list(live))
            n = live[r] + rng.randint(1, 6)
            try:
                cm.ensure(r, n)
                # nothing is ever written in a page that another table holds
                for g in cm.paged:
                    for p in range(live[r] // 4, -(-n // 4)):
                        assert cm.groups[g].pool.holders[cm.table(g, r)[p]] == 1
                cm.advance(r, n)
                live[r] = n
            except OutOfPages:
                pass
        elif live:
            r = rng.choice(list(live))
            cm.release(r)
            del live[r]
        cm.check()
    for r in live:
        cm.release(r)
    assert all(cm.groups[g].pool.num_free == sizes[g] for g in cm.paged)


def engine(kv_cache="model", kernels=None, **kw):
    opts = dict(dtype="float32", page_size=8, num_pages=48, device="cpu", max_num_seqs=6, max_num_batched_tokens=32, kv_cache=kv_cache)
    return build_engine(None, EngineConfig(**{**opts, **kw}), config=LlamaConfig.from_dict(TINY_B), random_seed=3,
                        kernels=kernels or P.PackedTorchKernels())


def run(eng, groups):
    """groups: [(n, prompt, max_tokens, temperature, seed)]; the sequences' generated tokens, group by group."""
    seqs = [eng.new_sequences(n, p, m, t, True, s) for n, p, m, t, s in groups]
    while eng.has_work():
        assert eng.step()
        eng.cache.check()
    assert all(g.pool.num_free == g.pool.num_pages for g in (eng.cache.groups[i] for i in eng.cache.paged))
    assert all(s.finished for group in seqs for s in group)
    return [[s.tokens[s.prompt_len:] for s in group] for group in seqs]


@pytest.mark.parametrize("kv_cache", ["model", "int4"])
@pytest.mark.parametrize("length", [1, 2, 8, 9, 21, 45])
def test_completions_of_one_prompt_are_those_of_separate_requests(kv_cache, length):
    prompt = [(5 * i + 11) % 320 for i in range(length)]
    kernels = P.PackedTorchKernels()
    together = run(engine(kv_cache, kernels), [(4, prompt, 6, 0.8, 70)])
    apart = run(engine(kv_cache), [(1, prompt, 6, 0.8, 70 + i) for i in range(4)])
    assert together[0] == [g[0] for g in apart]
    assert len({tuple(t) for t in together[0]}) > 1
    assert len(kernels.copied) == (3 if (length - 1) % 8 else 0)
    greedy = run(engine(kv_cache), [(3, prompt, 5, 0.0, None)])[0]
    assert greedy[0] == greedy[1] == greedy[2]


def test_forks_hold_the_prompts_pages_once():
    eng = engine()
    eng.new_sequences(4, [(5 * i + 11) % 320 for i in range(33)], 6, 0.9, True, 1)
    used = 0
    while eng.has_work():
        eng.step()
        used = max(used, eng.cache.groups[0].pool.num_pages - eng.cache.num_free)
    assert used == 4 + 4                              # 33 + 5 tokens: four pages of the prompt shared, one page each


@pytest.mark.parametrize("kw", [dict(max_num_seqs=2), dict(num_pages=9), dict(max_num_batched_tokens=7), dict(num_pages=14, max_num_seqs=5)])
def test_completions_without_room_to_fork_are_computed_one_by_one(kw):
    prompt = [(5 * i + 11) % 320 for i in range(26)]
    groups = [(4, prompt, 9, 0.8, 70), (2, prompt[:13], 4, 0.8, 9)]
    want = run(engine(num_pages=96), groups)
    assert run(engine(**kw), groups) == want


def test_a_completion_that_ends_at_once_leaves_the_others_to_run():
    prompt = [(5 * i + 11) % 320 for i in range(19)]
    got = run(engine(), [(3, prompt, 1, 0.0, None)])[0]
    assert got[0] == got[1] == got[2] and len(got[0]) == 1


def test_generate_returns_every_completion_in_order():
    llm = LLM(config=LlamaConfig.from_dict(TINY_B), random_seed=3, dtype="float32", page_size=8, num_pages=64, device="cpu", max_num_seqs=8,
              kernels=P.PackedTorchKernels(), kv_cache="int4")
    outs = llm.generate([[4, 5, 6, 7], [9, 8, 7]], [SamplingParams(max_tokens=3, temperature=0.7, seed=5, n=3), SamplingParams(max_tokens=2)])
    assert [o.prompt_token_ids for o in outs] == [[4, 5, 6, 7]] * 3 + [[9, 8, 7]]
    assert [len(o.token_ids) for o in outs] == [3, 3, 3, 2]
