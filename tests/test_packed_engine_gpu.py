"""The engine on the GPU with a packed cache and with several completions of a prompt: steps cut anywhere, captured graphs,
preemption, both types."""
import pytest
import torch

import kv4_plain as P
from configs import TINY_B, TINY_C, TINY_D
from iitj_llm_coopt_b200 import EngineConfig, LLM, LlamaConfig, SamplingParams, build_engine
from iitj_llm_coopt_b200.engine import StepEntry

pytestmark = pytest.mark.gpu


def engine(cfg, device="cuda:0", kernels=None, **kw):
    opts = dict(dtype="float32", page_size=8, num_pages=96, device=device, max_num_seqs=8, max_num_batched_tokens=256, kv_cache="int4")
    return build_engine(None, EngineConfig(**{**opts, **kw}), config=LlamaConfig.from_dict(cfg), random_seed=3, kernels=kernels)


def shared_weights(a, b):
    """Gives engine b (on the CPU) the weights of engine a."""
    for pa, pb in zip(a.runner.model.all_parts(), b.runner.model.all_parts()):
        for name, t in vars(pa).items():
            if isinstance(t, torch.Tensor):
                setattr(pb, name, t.float().cpu() if t.is_floating_point() else t.cpu())


@pytest.mark.parametrize("cfg,page", [(TINY_B, 8), (TINY_C, 16), (TINY_D, 16), (TINY_C, 4)])
def test_steps_against_the_plain_double(cfg, page):
    gpu = engine(cfg, page_size=page)
    cpu = engine(cfg, device="cpu", kernels=P.PackedTorchKernels(), page_size=page)
    shared_weights(gpu, cpu)
    toks = [(7 * i + 3) % cfg["vocab_size"] for i in range(150)]
    # request 0 in portions, request 1 joins, both decode
    steps = [[(0, toks[:70], [69])], [(0, toks[70:71], [0]), (1, toks[:33], [0, 32])], [(0, toks[71:90], [18]), (1, toks[33:34], [0])],
             [(0, toks[90:91], [0]), (1, toks[34:35], [0])], [(0, toks[91:92], [0]), (1, toks[35:36], [0])]]
    for eng in (gpu, cpu):
        for r in (0, 1):
            eng.cache.admit(r)
    for entries in steps:
        got, want = (eng.runner.step([StepEntry(*e) for e in entries]).float().cpu() for eng in (gpu, cpu))
        norm = want.norm(dim=-1)
        off = ((got - want).norm(dim=-1) / norm).max().item()
        # sums in another order, and the code beside it where a number lies that near a border: one number of thousands moves by a
        # fifteenth of its group's spread
        assert off < 5e-3, off
    gpu.sampler.k.check_health()


@pytest.mark.parametrize("cfg", [TINY_C, TINY_D])
def test_the_first_layers_cache_of_a_bfloat16_engine(cfg):
    """What a bfloat16 engine keeps of its first layer (whose keys and values no attention has touched) against float32 arithmetic.

    The normed row x is rounded to bfloat16 (u S of a sum of products with S = sum |x| |w|), the product and the rotated number are
    (2 u S), a rotation mixes two such numbers, and a code is off by half a step and 15 s 2^-8 (s rounded) on top."""
    eng = engine(cfg, dtype="bfloat16", page_size=16)
    toks = [(7 * i + 3) % cfg["vocab_size"] for i in range(90)]
    eng.cache.admit(0)
    for lo, hi in ((0, 61), (61, 62), (62, 63), (63, 90)):
        eng.runner.step([StepEntry(0, toks[lo:hi], [])])
    kept = eng.runner.read_cache(0, 0).cpu().double()
    parts = eng.runner.model.layers[0].parts()
    mixer, D, kv = parts["mixer"], cfg["head_dim"], cfg["num_key_value_heads"]
    x = eng.runner.model.embedding.weight[torch.tensor(toks, device="cuda")].double().cpu()
    x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + cfg["rms_norm_eps"]) * parts["mixer_norm"].weight.double().cpu()
    w = mixer.qkv.double().cpu()[mixer.heads * D:]
    k, v = (x @ w.T).view(90, 2, kv, D).unbind(1)
    sk, sv = (x.abs() @ w.abs().T).view(90, 2, kv, D).unbind(1)
    angle = torch.arange(90).float()[:, None] * mixer.position.inv_freq.cpu()          # (float32 angles, as the engine's)
    c, s = angle.double().cos()[:, None], angle.double().sin()[:, None]
    a, b = k.chunk(2, -1)
    k = torch.cat([a * c - b * s, b * c + a * s], -1)
    both = sum(sk.chunk(2, -1))
    sk = torch.cat([both, both], -1)
    for got, want, spread in ((kept[:, 0], k, sk), (kept[:, 1], v, sv)):
        err = 3 * P.U16 * spread
        # the step of the engine's group: its own spread, which the same errors move
        _, step, _ = P.pack(want.float())
        step = step.double() + 2 * err.unflatten(-1, (-1, 32)).amax(-1) / 15
        tol = err.unflatten(-1, (-1, 32)) + ((0.5 + 15 * 2.0 ** -8) * 1.01 * step)[..., None] + 1e-6
        assert bool(((got - want).abs().unflatten(-1, (-1, 32)) <= tol).all())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_graphs_and_lookahead_change_nothing(dtype):
    prompts = [[(3 * i + j) % 500 for i in range(n)] for j, n in enumerate((5, 40, 77, 1, 16))]
    got = []
    for kw in (dict(cuda_graphs=True, lookahead=True), dict(cuda_graphs=False, lookahead=False)):
        llm = LLM(config=LlamaConfig.from_dict(TINY_C), random_seed=2, dtype=dtype, num_pages=64, max_num_seqs=8, kv_cache="int4", **kw)
        got.append([o.token_ids for o in llm.generate(prompts, SamplingParams(max_tokens=40, temperature=0.7, seed=4, ignore_eos=True))])
    assert got[0] == got[1]


@pytest.mark.parametrize("kv_cache", ["model", "int4"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_completions_share_a_prompt(kv_cache, dtype):
    prompt = [(5 * i + 11) % 500 for i in range(101)]
    llm = LLM(config=LlamaConfig.from_dict(TINY_C), random_seed=2, dtype=dtype, num_pages=64, max_num_seqs=8, kv_cache=kv_cache)
    outs = llm.generate([prompt, prompt[:9]], SamplingParams(max_tokens=24, temperature=0.9, seed=50, n=3, ignore_eos=True))
    assert len(outs) == 6 and all(len(o.token_ids) == 24 for o in outs)
    assert len({tuple(o.token_ids) for o in outs[:3]}) == 3
    cache = llm.engine.cache
    cache.check()
    assert cache.num_free == cache.num_pages
    if dtype == "float32":
        alone = LLM(config=LlamaConfig.from_dict(TINY_C), random_seed=2, dtype=dtype, num_pages=64, max_num_seqs=8, kv_cache=kv_cache)
        for i in range(3):
            one = alone.generate([prompt], SamplingParams(max_tokens=24, temperature=0.9, seed=50 + i, ignore_eos=True))[0]
            assert one.token_ids == outs[i].token_ids


def test_a_fork_goes_on_from_a_copy_of_its_own():
    """What parent and child store after the fork does not reach the other."""
    eng = engine(TINY_C, dtype="bfloat16", page_size=16)
    toks = [(7 * i + 3) % 500 for i in range(60)]
    eng.cache.admit("a")
    eng.runner.step([StepEntry("a", toks[:43], [42])])
    eng.runner.fork("a", "b", 42)
    before = eng.runner.read_cache("a", 1).clone()
    assert torch.equal(eng.runner.read_cache("b", 1), before[:42])
    eng.runner.step([StepEntry("b", [9, 8, 7, 6], [3]), StepEntry("a", toks[43:47], [3])])
    assert torch.equal(eng.runner.read_cache("a", 1)[:43], before) and torch.equal(eng.runner.read_cache("b", 1)[:42], before[:42])
    assert not torch.equal(eng.runner.read_cache("b", 1)[42:46], eng.runner.read_cache("a", 1)[42:46])
    eng.cache.release("a")
    eng.cache.admit("c")
    eng.runner.step([StepEntry("c", toks[:16 * 4], [])])          # takes what "a" gave back
    assert torch.equal(eng.runner.read_cache("b", 1)[:42], before[:42])
    eng.cache.check()


def test_preemption_with_forks_and_a_packed_cache():
    prompt = [(5 * i + 11) % 500 for i in range(70)]
    groups = [(3, prompt, 30), (2, prompt[:40], 30), (1, prompt[:25], 20)]
    got = []
    for pages in (200, 14):
        eng = engine(TINY_C, num_pages=pages, page_size=8, max_num_seqs=6)
        seqs = [s for n, p, m in groups for s in eng.new_sequences(n, p, m, 0.8, True, 7)]
        eng.run_until_done()
        eng.cache.check()
        got.append([s.tokens for s in seqs])
        assert eng.cache.num_free == pages
    assert eng.counters["num_preemptions_total"] > 0
    assert got[0] == got[1]
