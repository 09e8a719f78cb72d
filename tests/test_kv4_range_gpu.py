"""Attention over a packed cache in bfloat16 whose numbers lie next to the ends of their range."""
import pytest
import torch

import kv4_bounds as B
import kv4_cases as C

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from iitj_llm_coopt_b200 import kernels
    return kernels.load()


@pytest.mark.parametrize("new", [1, 200])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("keys,late_keys,values,late_values", [(1, 1, 2.0 ** 122, 1), (1, 1, 1, 2.0 ** 122), (1, 1, 2.0 ** 122, 2.0 ** -122),
                                                               (1, 1, 2.0 ** 122, 2.0 ** -2), (1, 1, 2.0 ** -120, 1), (1, 1, 1, 2.0 ** 25), (1, 1, 1, 2.0 ** 20),
                                                               (1, 2.0 ** 30, 1, 1),
                                                               (2.0 ** 118, 1, 1, 1), (2.0 ** 118, 2.0 ** -10, 2.0 ** 110, 2.0 ** 10),
                                                               (1, 2.0 ** 90, 2.0 ** -3, 2.0 ** 70), (2.0 ** 66, 2.0 ** -3, 2.0 ** 66, 2.0 ** -3)])
def test_numbers_next_to_the_ends_of_their_range(K, new, D, keys, late_keys, values, late_values):
    """Keys and values times powers of two, those from token 150 on times others yet; queries that bring the largest scores back to where
    they were."""
    lens, news, heads, kv, page = [200, 1600], [new, new], 4, 2, 16
    table, cache = C.pages(21, lens, kv, D, page)
    for b, n in enumerate(lens):
        late = (torch.arange(n) >= 150)[:, None, None]
        k = C.rnd(n, kv, D, seed=2100 + b) * torch.where(late, late_keys, 1.0) * keys
        v = C.rnd(n, kv, D, seed=2150 + b) * torch.where(late, late_values, 1.0) * values
        C.fill(cache, table, b, page, k.bfloat16(), v.bfloat16())
    q = (C.rnd(sum(news), heads * D, seed=22) / max(keys, keys * late_keys)).bfloat16()
    want, tol = B.attend(q, cache, table, lens, news, heads, kv, page, D)
    got = C.attention(K, q, cache, table, lens, news, heads, kv, D)
    assert bool(got.isfinite().all()) and B.worst(got, want, tol) <= 1.0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("what", ["key", "value"])
@pytest.mark.parametrize("size", [2.0 ** 19, 2.0 ** 26, 2.0 ** 100])
def test_a_loud_token_does_not_reach_those_who_do_not_see_it(K, D, what, size):
    """Token 300 of a prompt: queries before it, in its tile of keys, give what they give without it; and with a window those far behind."""
    heads, kv, page, n = 4, 2, 16, 700
    for window in (0, 50):
        results = []
        for loud in (False, True):
            table, cache = C.pages(23, [n], kv, D, page)
            k, v = C.rnd(n, kv, D, seed=2300), C.rnd(n, kv, D, seed=2301)
            if loud:
                (k if what == "key" else v)[300] *= size
            C.fill(cache, table, 0, page, k.bfloat16(), v.bfloat16())
            q = C.rnd(n, heads * D, seed=24).bfloat16()
            want, tol = B.attend(q, cache, table, [n], [n], heads, kv, page, D, window)
            got = C.attention(K, q, cache, table, [n], [n], heads, kv, D, window)
            results.append((got.double().view_as(want), want, tol))
        (got0, want0, tol0), (got, want, tol) = results
        blind = torch.ones(n, dtype=torch.bool)
        blind[300:350 if window else n] = False
        assert bool(((got - want0).norm(dim=-1) <= tol0)[blind].all())       # by the bound of the cache without that token
        if what == "value" or size < 2.0 ** 50:        # (a score of 2^100 is one weight of 1: nothing to compare but that)
            assert B.worst(got, want, tol) <= 1.0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("what,at", [("key", 2500), ("value", 2500), ("value", 5980)])
def test_a_loud_token_in_a_long_context(K, D, what, at):
    """Few queries over many keys, which several blocks share: one of them has the loud token (at 5980 some queries do not see it)."""
    heads, kv, page, n, new = 4, 1, 16, 6000, 40
    table, cache = C.pages(25, [n], kv, D, page)
    k, v = C.rnd(n, kv, D, seed=2500), C.rnd(n, kv, D, seed=2501)
    (k if what == "key" else v)[at] *= 2.0 ** 26
    C.fill(cache, table, 0, page, k.bfloat16(), v.bfloat16())
    q = C.rnd(new, heads * D, seed=26).bfloat16()
    assert K.prefill_key_splits([(0, new, n - new, 0)], heads, kv, 0) > 1
    want, tol = B.attend(q, cache, table, [n], [new], heads, kv, page, D)
    assert B.worst(C.attention(K, q, cache, table, [n], [new], heads, kv, D), want, tol) <= 1.0
