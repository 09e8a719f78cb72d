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
                                                               (1, 1, 2.0 ** 122, 2.0 ** -2), (1, 1, 2.0 ** -120, 1),
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
