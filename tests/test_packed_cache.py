"""The packed key/value cache on the CPU: the format, its page sizes and budgets, what a configuration refuses, the C entry points'
refusals, and the engine end to end on the plain kernel double."""
import ctypes
import dataclasses
import io
import json
import math

import pytest
import torch

import kv4_plain as P
from configs import TINY_A, TINY_B, TINY_C
from iitj_llm_coopt_b200 import EngineConfig, LlamaConfig, SamplingParams, build_engine
from iitj_llm_coopt_b200.cache import CacheManager
from iitj_llm_coopt_b200.config.errors import ConfigError
from iitj_llm_coopt_b200.config.specs import CacheNeed
from iitj_llm_coopt_b200.engine import StepEntry


def packed_engine(cfg, kv_cache="int4", kernels=None, **kw):
    opts = dict(dtype="float32", page_size=8, num_pages=48, device="cpu", max_num_seqs=4, max_num_batched_tokens=64, kv_cache=kv_cache)
    ec = EngineConfig(**{**opts, **kw})
    return build_engine(None, ec, config=LlamaConfig.from_dict(cfg), random_seed=3, kernels=kernels or P.PackedTorchKernels())


@pytest.mark.parametrize("D", [32, 64, 96, 128, 256])
def test_every_number_has_a_nibble_of_its_own(D):
    for place in (P.key_place, P.value_place):
        places = {place(D, c) for c in range(D)}
        assert len(places) == D and all(0 <= b < D // 2 and s in (0, 4) for b, s in places)


def test_a_number_is_off_by_half_a_step_at_most():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(200, 3, 64, generator=g) * torch.logspace(-20, 20, 200)[:, None, None]
    x[7] = 0.75                                        # a constant group is its zero point
    x[8, :, ::2] += 1000.0                             # a spread that one number makes
    x = x.bfloat16().float()
    cache = torch.full((26, 3 * 8 * 2 * 40), 0xff, dtype=torch.uint8)
    slots = torch.randperm(208, generator=g)[:200]
    P.store(cache, slots, x, -x, 8)
    z, sn = P.numbers(cache, slots, 3, 8, 64)
    for got, want in ((z + sn)[:, 0], x), ((z + sn)[:, 1], -x):
        _, s, zero = P.pack(want)
        # half a step; s is rounded to bfloat16, which moves the top number's place by at most 15 s 2^-8, and 15.06 is still coded as 15
        tol = (0.5 + 15 * 2.0 ** -8) * s.double() + 4 * 2.0 ** -24 * (zero.abs() + 16 * s).double()
        assert bool(((got - want.double()).abs().unflatten(-1, (-1, 32)) <= tol[..., None]).all())
    assert bool(((z + sn)[7] == torch.tensor([0.75, -0.75]).view(2, 1, 1)).all())


@pytest.mark.parametrize("what", ["nan key", "inf key", "-inf value", "spread"])
def test_a_token_that_is_not_finite_is_a_key_of_nan_and_a_value_of_zero(what):
    k, v = torch.randn(3, 2, 64), torch.randn(3, 2, 64)
    if what == "nan key":
        k[1, 0, 40] = math.nan
    elif what == "inf key":
        k[1, 0, 3] = math.inf
    elif what == "-inf value":
        v[1, 0, 63] = -math.inf
    else:
        v[1, 0, 0], v[1, 0, 1] = 3e38, -3e38           # more than float32 spans
    cache = torch.zeros(1, 2 * 4 * 80, dtype=torch.uint8)
    P.store(cache, torch.tensor([0, 1, 2]), k, v, 4)
    z, sn = P.numbers(cache, torch.tensor([0, 1, 2]), 2, 4, 64)
    x = z + sn
    assert bool(x[1, 0, 0].isnan().all()) and bool((x[1, 1, 0] == 0).all())
    x[1, :, 0] = 0
    assert bool(x.isfinite().all())


def test_packed_pages_take_five_sixteenths_of_bfloat16():
    need = CacheNeed("paged_kv", kv_heads=8, head_dim=128)
    packed = dataclasses.replace(need, bits=4)
    assert need.page_bytes(16, 2) == 65536 and packed.page_bytes(16, 2) == packed.page_bytes(16, 4) == 65536 * 5 // 16
    many = CacheManager.pages_for_bytes([packed] * 4, 16, 1 << 28, 2, 8, 64)
    assert CacheManager.bytes_for([packed] * 4, 16, many, 2, 8, 64) <= 1 << 28 < CacheManager.bytes_for([packed] * 4, 16, many + 1, 2, 8, 64)
    cm = CacheManager([packed] * 2, 16, 5, 2, dtype=torch.bfloat16, device="cpu")
    assert cm.view(1)[1].shape == (6, 65536 * 5 // 16) and cm.view(1)[1].dtype == torch.uint8


def test_configurations_that_cannot_be_packed_are_refused():
    with pytest.raises(ValueError, match="kv_cache 'fp8' is not known"):
        EngineConfig(kv_cache="fp8")
    with pytest.raises(ConfigError, match="head_dim 16"):
        packed_engine(TINY_A)
    with pytest.raises(ConfigError, match="page_size 6"):
        packed_engine(TINY_C, page_size=6)
    from iitj_llm_coopt_b200.config.registry import architecture_for
    from iitj_llm_coopt_b200.presets import shape_config
    for name in ("lifusun-toy", "fomerax-toy", "kobolix-toy"):
        raw = shape_config(name)
        with pytest.raises(ConfigError, match="kv_cache 'int4'"):
            build_engine(None, EngineConfig(num_pages=8, device="cpu", kv_cache="int4"), random_seed=0, kernels=P.PackedTorchKernels(),
                         config=architecture_for(raw).config_class.from_dict(raw))


def test_c_entry_points_refuse_before_they_touch_the_device():
    from iitj_llm_coopt_b200.csrc import build
    from iitj_llm_coopt_b200.kernels import _SIGNATURES
    lib = ctypes.CDLL(build.library_path(verbose=False))
    lib.llm_last_error.restype = ctypes.c_char_p
    at = ctypes.c_void_p(4096)                          # never followed: every call below is refused

    def call(name, *args):
        fn = getattr(lib, name)
        fn.argtypes, fn.restype = _SIGNATURES[name], ctypes.c_int
        return fn(*args), lib.llm_last_error().decode()

    def store(head_dim=64, rotary=64, page=16, heads=4, kv=2, rows=at, splits=0, stride=0):
        return call("llm_rope_store_kv4", rows, at, splits, stride, at, 512, at, at, at, at, 1, 3, heads, kv, head_dim, rotary, page, None)
    for bad in (dict(head_dim=48), dict(head_dim=288), dict(page=6), dict(page=0), dict(rotary=12), dict(rotary=72), dict(heads=0),
                dict(rows=None, splits=9), dict(rows=None, splits=2, stride=6)):
        rc, text = store(**bad)
        assert rc == -1 and "rope_store_kv4" in text, bad
    assert call("llm_kv4_read", at, at, at, 0, 3, 2, 40, 16, None)[0] == -1
    assert call("llm_attention_kv4_general", at, 256, at, at, 4, None, 3, at, at, at, 256, 1, 5, 2, 64, 16, 0, 0.1, 1, None, None)[0] == -1     # 5 heads over 2
    for splits in (0, -1, 2):                           # none, and two without a place for their sums
        assert call("llm_attention_kv4_general", at, 256, at, at, 4, None, 3, at, at, at, 256, 1, 4, 2, 64, 16, 0, 0.1, splits, None, None)[0] == -1
    assert call("llm_attention_kv4_single", at, 256, at, at, 4, at, 3, at, at, None, None, at, 256, 4, 2, 96, 16, 0, 0.1, 6, 1, None)[0] == -1
    assert call("llm_attention_kv4_single", at, 256, at, at, 4, at, 3, at, at, None, None, at, 256, 4, 2, 64, 12, 0, 0.1, 6, 1, None)[0] == -1
    assert call("llm_attention_kv4_single", at, 256, at, at, 4, at, 3, at, at, None, None, at, 256, 4, 2, 64, 16, 0, 0.1, 6, 2, None)[0] == -1     # no scratch
    assert call("llm_attention_kv4_single", at, 252, at, at, 4, at, 3, at, at, None, None, at, 256, 4, 2, 64, 16, 0, 0.1, 6, 1, None)[0] == -1
    assert call("llm_attention_kv4_prompt", at, 256, 9, at, at, 4, at, 1, at, 256, 4, 2, 96, 16, 0, 0.1, 1, None, None, None)[0] == -1
    assert call("llm_attention_kv4_f32_tiles", at, 256, at, at, 4, at, 1, at, 256, 4, 2, 64, 6, 0, 0.1, None)[0] == -1
    pairs = (ctypes.c_int * 4)(0, 1, 2, 8)
    rc, text = call("llm_copy_pages", at, 2, 8, 1024, pairs, 2, None)
    assert rc == -1 and "page 8" in text
    for bad, text in (((0, 1, 2, 1), "page 1 is the destination of two copies"), ((0, 1, 1, 2), "page 1 is the source of one copy"),
                      ((3, 3, 0, 1), "page 3 is the source of one copy"), ((5, 6, 6, 6), "page 6 is the")):
        rc, said = call("llm_copy_pages", at, 2, 8, 1024, (ctypes.c_int * 4)(*bad), 2, None)
        assert rc == -1 and text in said
    many = [x for i in range(400) for x in (i, 1000 + i)] + [1399, 999]          # the last pair reads what the one before writes
    rc, said = call("llm_copy_pages", at, 2, 2000, 1024, (ctypes.c_int * len(many))(*many), 401, None)
    assert rc == -1 and "page 1399 is the source of one copy" in said
    # nothing to do is no error
    assert call("llm_copy_pages", at, 2, 8, 1024, pairs, 0, None)[0] == 0


def test_whole_prompts_and_portions_read_the_same_packed_keys():
    """The logits do not depend on how a prompt is cut, and they are near those of an unpacked cache."""
    toks = [(7 * i + 3) % 300 for i in range(41)]
    rows = {}
    for name, kv_cache, cuts in (("packed", "int4", [41]), ("cut", "int4", [1, 9, 16, 3, 12]), ("model", "model", [41])):
        eng = packed_engine(TINY_B, kv_cache)
        eng.cache.admit("r")
        at = 0
        for n in cuts:
            out = eng.runner.step([StepEntry("r", toks[at:at + n], [n - 1])])
            at += n
        rows[name] = out[-1]
        if kv_cache == "int4":
            kept = eng.runner.read_cache("r", 1)
            assert kept.shape == (41, 2, 1, 32) and torch.equal(kept[5:9], eng.runner.read_cache("r", 1, 5, 9))
    assert torch.allclose(rows["packed"], rows["cut"], atol=1e-4 * rows["packed"].abs().max().item())
    # a key or value number is off by up to 1/30 of its group's spread: logits move, and stay recognisable
    assert torch.nn.functional.cosine_similarity(rows["packed"], rows["model"], dim=0) > 0.98


def test_the_cache_reads_back_what_an_unpacked_one_holds_but_for_the_codes():
    toks = list(range(5, 30))
    got = {}
    for kv_cache in ("int4", "model"):
        eng = packed_engine(TINY_C, kv_cache, page_size=4)
        eng.cache.admit(0)
        eng.runner.step([StepEntry(0, toks, [24])])
        got[kv_cache] = eng.runner.read_cache(0, 0)           # the first layer's keys and values do not depend on the cache
        with pytest.raises(ValueError, match="not among the 25"):
            eng.runner.read_cache(0, 0, 3, 26)
    a, b = got["int4"].double(), got["model"].double()
    _, s, z = P.pack(b.float())
    tol = (0.5 + 15 * 2.0 ** -8) * s.double() + 2.0 ** -7 * z.abs().double()       # (z itself is rounded down to a bfloat16)
    assert bool(((a - b).abs().unflatten(-1, (-1, 32)) <= tol[..., None]).all())


def test_trace_replay_with_a_packed_cache(tmp_path):
    from iitj_llm_coopt_b200 import replay
    from iitj_llm_coopt_b200.weights import write_model_dir
    write_model_dir(TINY_B, str(tmp_path / "m"), 1)
    lines = [json.dumps({"step": 0, "entries": [{"id": 1, "tokens": [5, 6, 7], "want": [2]}]}),
             json.dumps({"step": 1, "entries": [{"id": 1, "tokens": [8], "want": [0]}], "end": [1]})]
    args = replay.parse_args(["--model", str(tmp_path / "m"), "--dtype", "float32", "--out", str(tmp_path / "o"), "--max-tokens", "64",
                              "--page-size", "8", "--device", "cpu", "--kv-cache", "int4"])
    assert replay.run(args, lines, out=io.StringIO(), kernels=P.PackedTorchKernels()) == 0
    assert (tmp_path / "o" / "1.f32").stat().st_size == 4 * 320


def test_sampling_params_refuse_no_completion():
    with pytest.raises(ValueError, match="n must be"):
        SamplingParams(n=0)
