"""The kernels of the packed key/value cache against their plain restatement (tests/kv4_plain.py): codes to the bit, attention within
the bound that its roundings allow, at the sizes, pages and masks where it can go wrong."""
import math
from types import SimpleNamespace

import pytest
import torch

import kv4_plain as P

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from iitj_llm_coopt_b200 import kernels
    return kernels.load()


def rnd(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def page_bytes(kv, page, D):
    return kv * page * (D // 32) * 40


# ---- storing and reading back ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,heads,kv,D,page,rot", [(1, 4, 2, 128, 16, 128), (9, 6, 2, 64, 8, 64), (3, 5, 5, 32, 4, 32), (17, 3, 1, 96, 12, 96),
                                                   (5, 2, 1, 160, 16, 64), (6, 4, 2, 256, 64, 256), (4, 8, 8, 64, 16, 0), (2, 40, 20, 32, 16, 16),
                                                   (130, 32, 8, 128, 16, 128)])
def test_store_packs_to_the_bit(K, dtype, T, heads, kv, D, page, rot):
    qkv = rnd(T, heads + 2 * kv, D, seed=1)
    qkv[:, heads:heads + kv, ::7] *= 9.0
    qkv = qkv.flatten(1).to(dtype)
    angle = rnd(T, max(rot // 2, 1), seed=2) * 40
    tables = (angle.cos(), angle.sin()) if rot else None
    pages = -(-T // page) + 2
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(3))[:T].int()
    if T > 2:
        slots[1] = -1                                  # not stored
    want_cache = torch.full((pages, page_bytes(kv, page, D)), 0xa5, dtype=torch.uint8)
    cache = want_cache.cuda()
    want_qkv = qkv.clone()
    P.PackedTorchKernels().rope_store_kv4(want_qkv, tables, slots, want_cache, heads, kv, D, rot)
    dev_tables = tuple(t.cuda() for t in tables) if rot else None
    got = qkv.cuda()
    assert K.rope_store_kv4(got, dev_tables, slots.cuda(), cache, heads, kv, D, rot).data_ptr() == got.data_ptr()
    assert torch.equal(cache.cpu(), want_cache)        # rows that no slot names stay as they were
    assert torch.equal(got.cpu(), want_qkv)
    # queries into a tensor of their own; nothing stored
    q_out, again = torch.empty(T, heads * D, dtype=dtype, device="cuda"), qkv.cuda()
    K.rope_store_kv4(again, dev_tables, None, None, heads, kv, D, rot, q_out=q_out)
    assert torch.equal(q_out.cpu(), want_qkv[:, :heads * D]) and torch.equal(again.cpu(), qkv) and torch.equal(cache.cpu(), want_cache)
    # and back as numbers
    kept = torch.empty(T, 2, kv, D, device="cuda")
    K.kv4_read(cache, slots.cuda(), kept, kv, D)
    z, sn = P.numbers(want_cache, slots.clamp(min=0), kv, page, D)
    want = (z + sn).float()
    want[slots < 0] = 0
    assert torch.equal(kept.cpu(), want)
    half = torch.empty(T, 2, kv, D, device="cuda", dtype=torch.bfloat16)
    assert torch.equal(K.kv4_read(cache, slots.cuda(), half, kv, D).cpu(), want.bfloat16())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_store_of_odd_numbers(K, dtype, D):
    """Constants, tiny and huge spreads, zeros of either sign, what is not finite."""
    T, kv, page = 16, 2, 4
    x = rnd(T, 3 * kv, D, seed=4)
    x[0] = 0.0
    x[1] = -0.0
    x[2] = 3.25
    x[3] *= 1e-38
    x[4] *= 1e-42
    x[5] *= 1e37
    x[6, :, 0], x[6, :, 1] = 3.3e38, -3.3e38           # spans more than float32 does
    x[7, kv, 33] = math.nan
    x[8, 2 * kv, D - 1] = math.inf
    x[9, kv + 1, 0] = -math.inf
    x[10] = x[10] * 1e-3 + 100.0
    x[11, :, 5] = 1e30
    x[12, :, :32] = -3.38e38                           # (a float32 whose bfloat16 below it is -inf, in float32)
    x[12, :, 1] = -3.4e38
    qkv = x.flatten(1).to(dtype)
    slots = torch.arange(T, dtype=torch.int32)
    want = torch.zeros(4, page_bytes(kv, page, D), dtype=torch.uint8)
    P.PackedTorchKernels().rope_store_kv4(qkv.clone(), None, slots, want, kv, kv, D, 0)
    cache = torch.zeros_like(want).cuda()
    K.rope_store_kv4(qkv.cuda(), None, slots.cuda(), cache, kv, kv, D, 0)
    z, sn = P.numbers(cache.cpu(), slots, kv, page, D)
    wz, wsn = P.numbers(want, slots, kv, page, D)
    assert torch.equal((z + sn).nan_to_num(nan=7e77), (wz + wsn).nan_to_num(nan=7e77))      # (the zero's sign may differ)
    nan = (z + sn)[:, 0].isnan().all(-1)
    assert bool(nan[6].all()) and nan[7].tolist() == [True, False] and nan[8].tolist() == [True, False] and nan[9].tolist() == [False, True]
    assert bool(((z + sn)[:, 1][nan] == 0).all()) and bool((z + sn)[:, 1].isfinite().all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("splits", [1, 3, 8])
def test_store_adds_partial_sums(K, dtype, splits):
    from iitj_llm_coopt_b200.kernels import PartialSums
    T, heads, kv, D, page = 5, 8, 2, 128, 16
    parts = rnd(splits, T, (heads + 2 * kv) * D, seed=6)
    total = parts[0].clone()
    for i in range(1, splits):
        total += parts[i]                              # in the order of the splits, in float32
    angle = rnd(T, D // 2, seed=7) * 9
    tables = (angle.cos(), angle.sin())
    slots = torch.tensor([3, 17, 40, 41, 0], dtype=torch.int32)
    want = torch.zeros(3, page_bytes(kv, page, D), dtype=torch.uint8)
    # the sums are rotated in float32 and rounded to the engine's type once, as the unpacked store does
    x = total.view(T, -1, D)
    c, s = tables[0][:, None], tables[1][:, None]
    a, b = x[:, :heads + kv, :D // 2], x[:, :heads + kv, D // 2:]
    rot = torch.cat([a * c - b * s, b * c + a * s], -1).to(dtype)
    P.store(want, slots, rot[:, heads:], x[:, heads + kv:].to(dtype), page)
    cache, out = torch.zeros_like(want).cuda(), torch.zeros(T, (heads + 2 * kv) * D, dtype=dtype, device="cuda")
    q = K.rope_store_kv4(PartialSums(K, parts.cuda(), out), tuple(t.cuda() for t in tables), slots.cuda(), cache, heads, kv, D, D)
    assert q.data_ptr() == out.data_ptr() and torch.equal(q.cpu()[:, :heads * D], rot[:, :heads].flatten(1))
    assert torch.equal(cache.cpu(), want)


# ---- attention -----------------------------------------------------------------------------------------------------------
def case(seed, lens, news, heads, kv, D, page, dtype, wide=0, spoil=True):
    """Packed pages in random order.  Everything that no sequence owns (rows behind the last token, other pages) is 0xff: z and s
    that are NaN.  q rows are `wide` numbers wider than the queries."""
    need = [-(-n // page) for n in lens]
    pool = sum(need) + 3
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed))
    table = torch.zeros(len(lens), max(need) + 2, dtype=torch.int32)
    cache = torch.full((pool, page_bytes(kv, page, D)), 0xff if spoil else 0, dtype=torch.uint8)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].int()
        at += n
        p = torch.arange(lens[b])
        k, v = rnd(lens[b], kv, D, seed=seed * 100 + b), rnd(lens[b], kv, D, seed=seed * 100 + 50 + b)
        k[:, :, ::11] *= 4.0
        P.store(cache, table[b].long()[p // page] * page + p % page, k.to(dtype), v.to(dtype), page)
    T = sum(news)
    q = rnd(T, heads * D + wide, seed=seed + 9).to(dtype)
    request = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(news)).int()
    position = torch.cat([torch.arange(n - m, n) for n, m in zip(lens, news)]).int()
    meta = SimpleNamespace(block_table=table.cuda(), token_request=request.cuda(), positions=position.cuda(), query_lens=list(news),
                           seq_lens_host=list(lens))
    return q, cache, table, meta


def check(K, seed, lens, news, heads, kv, D, page, dtype, window=0, scale=0.0, wide=0):
    q, cache, table, meta = case(seed, lens, news, heads, kv, D, page, dtype, wide)
    want, tol = P.attend(q[:, :heads * D], cache, table, lens, news, heads, kv, page, D, window, scale,
                         P.U16 if dtype == torch.bfloat16 else P.U32)
    out = torch.full((q.shape[0], heads * D), 7.0, dtype=dtype, device="cuda")
    K.attention_kv4(q.cuda(), cache.cuda(), meta, out, heads, kv, D, window=window, scale=scale)
    K.check_health()
    got = out.cpu().double()
    worst = ((got - want).abs() / tol).max().item()
    assert worst <= 1.0 and bool(got.isfinite().all()), worst
    return got, want


DTYPES = [torch.bfloat16, torch.float32]
LENS = [1, 2, 15, 16, 17, 31, 33, 64, 65, 127, 128, 129, 255, 300]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,D,page", [(4, 2, 64, 16), (4, 1, 128, 16), (6, 2, 128, 4), (9, 1, 64, 8), (16, 1, 128, 64), (3, 3, 64, 32),
                                             (2, 1, 128, 12), (4, 2, 32, 16), (6, 3, 96, 20), (4, 1, 256, 16), (12, 1, 160, 48), (5, 1, 64, 128)])
def test_single_tokens(K, dtype, heads, kv, D, page):
    check(K, 1, LENS, [1] * len(LENS), heads, kv, D, page, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [1, 7, 16, 33, 100, 1000])
def test_single_tokens_with_a_window(K, dtype, window):
    check(K, 2, LENS, [1] * len(LENS), 8, 2, 64, 8, dtype, window=window)
    check(K, 3, [300, 40, 9], [1] * 3, 4, 1, 128, 64, dtype, window=window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,D,page", [(4, 2, 64, 16), (4, 1, 128, 16), (3, 1, 128, 4), (8, 8, 64, 64), (2, 1, 128, 12), (2, 1, 32, 8),
                                             (4, 2, 96, 16), (2, 1, 256, 16), (10, 2, 64, 128)])
def test_prompts(K, dtype, heads, kv, D, page):
    lens = [1, 2, 17, 127, 128, 130, 260]
    check(K, 4, lens, lens, heads, kv, D, page, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,page", [(64, 8), (128, 16), (128, 24)])
def test_portions_and_single_tokens_together(K, dtype, D, page):
    check(K, 5, [300, 41, 9, 513, 129, 64], [3, 1, 9, 130, 128, 1], 6, 2, D, page, dtype, wide=64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [1, 5, 64, 128, 200])
def test_prompts_with_a_window(K, dtype, window):
    check(K, 6, [300, 41, 513], [290, 41, 130], 4, 2, 64, 16, dtype, window=window)
    check(K, 7, [257, 500], [257, 2], 4, 1, 128, 8, dtype, window=window)


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_contexts(K, dtype):
    check(K, 8, [3000, 2600, 70], [1, 1, 1], 4, 1, 128, 16, dtype)
    check(K, 9, [3300], [40], 4, 1, 64, 16, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores_and_a_scale_of_its_own(K, dtype):
    q, cache, table, meta = case(10, [200, 140], [1, 40], 4, 2, 64, 16, dtype)
    q *= 30.0                                          # one key takes nearly all of the weight
    want, tol = P.attend(q, cache, table, [200, 140], [1, 40], 4, 2, 16, 64, 0, 0.3, P.U16 if dtype == torch.bfloat16 else P.U32)
    out = torch.empty(41, 256, dtype=dtype, device="cuda")
    K.attention_kv4(q.cuda(), cache.cuda(), meta, out, 4, 2, 64, scale=0.3)
    K.check_health()
    # (the bound says little where scores are in the hundreds: whatever it allows, the result lies among the values)
    assert bool(((out.cpu().double() - want).abs() <= tol).all()) and out.abs().max() < 6


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 200])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("keys,late_keys,values,late_values", [(2.0 ** -60, 1, 2.0 ** -25, 1), (2.0 ** 70, 1, 2.0 ** 50, 1),
                                                               (1, 2.0 ** -16, 2.0 ** -16, 2.0 ** 16), (2.0 ** -16, 2.0 ** 16, 1, 2.0 ** -16),
                                                               (1, 1, 0.0, 1), (0.0, 1, 1, 0.0), (1, 1, 2.0 ** 20, 0.0)])
def test_small_and_large_numbers(K, dtype, new, D, keys, late_keys, values, late_values):
    """Keys and values times powers of two, those from token 150 on times others yet; queries that bring the scores back to where
    they were.  (1600 keys: the kernels' splits too.)"""
    lens, news, page = [200, 1600], [new, new], 16
    q, cache, table, meta = case(12, lens, news, 4, 2, D, page, dtype, spoil=False)
    for b, n in enumerate(lens):
        p = torch.arange(n)
        late = (p >= 150)[:, None, None]
        k, v = rnd(n, 2, D, seed=1200 + b), rnd(n, 2, D, seed=1250 + b)
        k, v = k * torch.where(late, late_keys, 1.0) * keys, v * torch.where(late, late_values, 1.0) * (values or 1.0)
        if not values:
            v[:150] = 0.0
        P.store(cache, table[b].long()[p // page] * page + p % page, k.to(dtype), v.to(dtype), page)
    q = q / (max(keys, keys * late_keys) or 1.0)
    want, tol = P.attend(q, cache, table, lens, news, 4, 2, page, D, unit=P.U16 if dtype == torch.bfloat16 else P.U32)
    out = torch.full((q.shape[0], 4 * D), 7.0, dtype=dtype, device="cuda")
    K.attention_kv4(q.cuda(), cache.cuda(), meta, out, 4, 2, D)
    K.check_health()
    got = out.cpu().double()
    assert bool(got.isfinite().all()) and bool(((got - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("news", [[1, 1], [290, 150]])
def test_queries_of_zeros_and_of_the_smallest_numbers(K, dtype, window, news):
    """Scores of 0: the mean of the values that the window shows."""
    q, cache, table, meta = case(13, [290, 150], news, 4, 2, 64, 16, dtype)
    q[::2] = 0.0
    q[1::4] *= 1e-38
    want, tol = P.attend(q, cache, table, [290, 150], news, 4, 2, 16, 64, window, 0.0, P.U16 if dtype == torch.bfloat16 else P.U32)
    out = torch.full((q.shape[0], 256), 7.0, dtype=dtype, device="cuda")
    K.attention_kv4(q.cuda(), cache.cuda(), meta, out, 4, 2, 64, window=window)
    K.check_health()
    assert bool(((out.cpu().double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 130])
def test_a_token_that_is_not_finite_reaches_only_those_who_see_it(K, dtype, new):
    """A key of NaN at position 150 of 200: queries before it give what they give without it, queries behind it NaN."""
    heads, kv, D, page = 4, 2, 64, 16
    for lens, window in (([200], 0), ([200], 30)):
        q, cache, table, meta = case(11, lens, [new], heads, kv, D, page, dtype)
        bad = cache.clone()
        x = torch.full((1, kv, D), math.nan)
        slot = table[0].long()[150 // page] * page + 150 % page
        P.store(bad, slot.view(1), x, x, page)
        clean, got = (torch.empty(new, heads * D, dtype=dtype, device="cuda") for _ in range(2))
        K.attention_kv4(q.cuda(), cache.cuda(), meta, clean, heads, kv, D, window=window)
        K.attention_kv4(q.cuda(), bad.cuda(), meta, got, heads, kv, D, window=window)
        pos = torch.arange(200 - new, 200)
        sees = (pos >= 150) & ((pos - 150 < window) if window else torch.ones(new, dtype=torch.bool))
        assert torch.equal(got.cpu()[~sees], clean.cpu()[~sees])
        assert bool(got.cpu()[sees].isnan().all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 130])
def test_a_query_head_that_is_not_finite_spoils_no_other(K, dtype, new):
    heads, kv, D, page = 8, 2, 128, 16
    q, cache, table, meta = case(13, [500], [new], heads, kv, D, page, dtype)
    want, tol = P.attend(q, cache, table, [500], [new], heads, kv, page, D, unit=P.U16 if dtype == torch.bfloat16 else P.U32)
    clean, got = (torch.empty(new, heads * D, dtype=dtype, device="cuda") for _ in range(2))
    K.attention_kv4(q.cuda(), cache.cuda(), meta, clean, heads, kv, D)
    q[0, 2 * D + 5], q[0, 4 * D + 6] = math.nan, math.inf
    K.attention_kv4(q.cuda(), cache.cuda(), meta, got, heads, kv, D)
    spoiled = torch.zeros(new, heads, D, dtype=torch.bool)
    spoiled[0, [2, 4]] = True
    spoiled = spoiled.flatten(1)
    assert bool(got.cpu()[spoiled].isnan().all())
    # (heads that share a warp share the decision to move the reference of their sums: the others' last bits may differ)
    for x in (got, clean):
        assert bool(((x.cpu().double() - want).abs() <= tol)[~spoiled].all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_request_gives_the_same_numbers_in_any_company(K, dtype):
    """The second time, on another stream, captured and replayed: the same bits."""
    heads, kv, D, page = 8, 2, 128, 16
    lens, news = [700, 33, 260, 1500], [1, 1, 200, 1]
    q, cache, table, meta = case(12, lens, news, heads, kv, D, page, dtype)
    q, cache = q.cuda(), cache.cuda()
    first = K.attention_kv4(q, cache, meta, torch.empty(q.shape[0], heads * D, dtype=dtype, device="cuda"), heads, kv, D).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = K.attention_kv4(q, cache, meta, torch.empty_like(first), heads, kv, D)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, other)
    out = torch.zeros_like(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.attention_kv4(q, cache, meta, out, heads, kv, D)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(first, out)


# ---- page copies ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape,dtype", [((3, 20, 2, 4, 16, 64), torch.bfloat16), ((2, 600, 1280), torch.uint8), ((1, 9, 5), torch.float32),
                                         ((4, 7, 3), torch.bfloat16), ((2, 5, 13), torch.uint8), ((1, 4, 100003), torch.float32)])
def test_copy_pages(K, shape, dtype):
    x = (torch.rand(*shape) * 200).to(dtype)
    pages = shape[1]
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).tolist()
    n = min(280, pages // 2)                           # more than one launch's pairs where the pool has them
    pairs = [(order[i], order[pages - 1 - i]) for i in range(n)]
    pairs += [(pairs[0][0], order[n])] if pages > 2 * n else []       # one page copied twice
    want = x.clone()
    for a, b in pairs:
        want[:, b] = x[:, a]
    got = x.cuda()
    assert K.copy_pages(got, pairs) is got
    assert torch.equal(got.cpu(), want)
    assert K.copy_pages(got, []) is got and torch.equal(got.cpu(), want)


def test_copy_pages_past_four_gigabytes(K):
    pool = torch.zeros(1, 5000, 1 << 20, dtype=torch.uint8, device="cuda")
    pool[0, 4321] = 7
    K.copy_pages(pool, [(4321, 4999), (4320, 3)])
    assert bool((pool[0, 4999] == 7).all()) and int(pool[0, 4998].max()) == int(pool[0, 3].max()) == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_pages_past_four_gigabytes(K, dtype):
    """Byte offsets of a long pool: stored, read and attended beyond 2^32."""
    heads, kv, D, page = 4, 1, 128, 16
    per = page_bytes(kv, page, D)
    pool = (1 << 32) // per + 200
    cache = torch.zeros(pool, per, dtype=torch.uint8, device="cuda")
    n = 40
    ids = torch.tensor([pool - 1, pool - 77, pool - 30], dtype=torch.int32)
    pos = torch.arange(n)
    slots = (ids[pos // page].long() * page + pos % page).int()
    qkv = rnd(n, (heads + 2 * kv) * D, seed=3).to(dtype)
    K.rope_store_kv4(qkv.cuda(), None, slots.cuda(), cache, heads, kv, D, 0)
    small = torch.zeros(3, per, dtype=torch.uint8)
    P.store(small, pos, qkv[:, heads * D:(heads + kv) * D].view(n, kv, D), qkv[:, (heads + kv) * D:].view(n, kv, D), page)
    assert torch.equal(cache[ids.long().cuda()].cpu()[:, :], small)
    for new in (1, n):
        q = qkv[-new:, :heads * D].contiguous()
        want, tol = P.attend(q, small, torch.arange(3).view(1, 3), [n], [new], heads, kv, page, D, unit=P.U16 if dtype == torch.bfloat16 else P.U32)
        meta = SimpleNamespace(block_table=ids.view(1, 3).cuda(), token_request=torch.zeros(new, dtype=torch.int32, device="cuda"),
                               positions=torch.arange(n - new, n, dtype=torch.int32, device="cuda"), query_lens=[new], seq_lens_host=[n])
        out = K.attention_kv4(q.cuda(), cache, meta, torch.empty(new, heads * D, dtype=dtype, device="cuda"), heads, kv, D)
        assert bool(((out.cpu().double() - want).abs() <= tol).all())


# ---- refusals --------------------------------------------------------------------------------------------------------------
def test_refusals(K):
    from iitj_llm_coopt_b200.kernels import KernelError
    z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device="cuda")      # noqa: E731
    cache, slots = z(4, page_bytes(2, 16, 64), t=torch.uint8), z(3, t=torch.int32)
    tables = (z(3, 32, t=torch.float32), z(3, 32, t=torch.float32))
    qkv = z(3, 8 * 64)
    good = dict(qkv=qkv, tables=tables, slots=slots, cache_layer=cache, heads=4, kv_heads=2, head_dim=64, rotary_dim=64)
    K.rope_store_kv4(**good)
    for bad, text in ((dict(head_dim=32), "width"), (dict(rotary_dim=60), "rotary_dim"), (dict(tables=None), "tables"),
                      (dict(tables=(tables[0][:, :16].contiguous(), tables[1])), "table shape"), (dict(slots=slots[:2]), "one per token"),
                      (dict(slots=slots.long()), "dtype"), (dict(cache_layer=z(4, 2, 2, 16, 64)), "dtype"),
                      (dict(cache_layer=z(4, 1000, t=torch.uint8)), "multiple of 4 tokens"), (dict(q_out=z(3, 128)), "wrong shape"),
                      (dict(q_out=z(3, 256, t=torch.float32)), "dtype"), (dict(qkv=qkv.cpu()), "GPU only"),
                      (dict(qkv=z(3, 16 * 64)[:, ::2]), "contiguous"), (dict(qkv=z(3, 8 * 64).double()), "dtype")):
        with pytest.raises(KernelError, match=text):
            K.rope_store_kv4(**{**good, **bad})
    with pytest.raises(KernelError, match="wrong shape"):
        K.kv4_read(cache, slots, z(3, 2, 2, 32), 2, 64)
    with pytest.raises(KernelError, match="multiple of 32"):
        K.kv4_read(cache, slots, z(3, 2, 2, 48), 2, 48)
    meta = SimpleNamespace(block_table=z(1, 4, t=torch.int32), token_request=z(3, t=torch.int32), positions=z(3, t=torch.int32),
                           query_lens=[3], seq_lens_host=[3])
    good = dict(q=z(3, 256), cache_layer=cache, meta=meta, out=z(3, 256), heads=4, kv_heads=2, head_dim=64)
    for bad, text in ((dict(heads=5), "multiple of kv_heads"), (dict(out=z(3, 128)), "out"), (dict(q=z(3, 128)), "narrow"),
                      (dict(out=z(3, 256, t=torch.float32)), "dtype"), (dict(cache_layer=cache[:, 16:]), "contiguous"),
                      (dict(q=z(2, 256), out=z(2, 256)), "one position per token"),
                      (dict(scale=-0.1), "positive"), (dict(scale=math.nan), "positive"), (dict(scale=math.inf), "positive")):
        with pytest.raises(KernelError, match=text):
            K.attention_kv4(**{**good, **bad})
    pool = z(2, 6, 32)
    for pairs, text in (([(0, 6)], "pool's 6 pages"), ([(-1, 2)], "pool's 6 pages"), ([(0, 1), (2, 1)], "two copies"),
                        ([(0, 1), (1, 2)], "source of one"), ([(3, 3)], "source of one"), ([(0, 1, 2)], "page ids are wanted"),
                        ([(0, 1.5)], "page ids are wanted"), ([(0, 1 << 40)], "page ids are wanted")):
        with pytest.raises(KernelError, match=text):
            K.copy_pages(pool, pairs)
    empty = K.attention_kv4(z(0, 256), cache, SimpleNamespace(block_table=z(1, 4, t=torch.int32), token_request=z(0, t=torch.int32),
                                                              positions=z(0, t=torch.int32), query_lens=[], seq_lens_host=[]),
                            z(0, 256), 4, 2, 64)
    assert empty.shape == (0, 256)
    assert K.rope_store_kv4(z(0, 512), None, None, None, 4, 2, 64, 0).shape == (0, 512)


def test_a_captured_step_follows_its_contexts(K):
    """One graph, replayed as the contexts grow from a few keys past several splits, each kernel behind the other: the single tokens
    of both types and the general kernel (head size 96), with an early reader of the result behind each."""
    for dtype, heads, kv, D in ((torch.bfloat16, 4, 1, 128), (torch.float32, 4, 1, 128), (torch.bfloat16, 4, 2, 96)):
        lens = [1500, 1400]
        q, cache, table, meta = case(14, lens, [1, 1], heads, kv, D, 16, dtype)
        from iitj_llm_coopt_b200.kernels import attention_plan
        meta.seq_lens_host = [1500, 1400]
        attention_plan(meta, torch.device("cuda", 0)).context_bound = 1536
        dq, dcache, out, ones = q.cuda(), cache.cuda(), torch.zeros(2, heads * D, dtype=dtype, device="cuda"), torch.ones(heads * D, device="cuda")
        normed = torch.zeros_like(out)
        K.attention_kv4(dq, dcache, meta, out, heads, kv, D)
        K.rmsnorm_rows(out, ones, 1e-5, normed)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(3):
                K.attention_kv4(dq, dcache, meta, out, heads, kv, D)
                K.rmsnorm_rows(out, ones, 1e-5, normed)
        for at in ([0, 3], [40, 1399], [700, 64], [1499, 1399]):
            meta.positions.copy_(torch.tensor(at, dtype=torch.int32))
            out.fill_(7.0)
            graph.replay()
            want, tol = P.attend(q[:, :heads * D], cache, table, [a + 1 for a in at], [1, 1], heads, kv, 16, D,
                                 unit=P.U16 if dtype == torch.bfloat16 else P.U32)
            assert bool(((out.cpu().double() - want).abs() <= tol).all()), at
            again = torch.empty_like(out)
            K.rmsnorm_rows(out, ones, 1e-5, again)
            assert torch.equal(again, normed), at
