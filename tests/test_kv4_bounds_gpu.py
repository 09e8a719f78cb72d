"""Attention over a packed cache in bfloat16, every row and head within what its kernels' roundings amount to (tests/kv4_bounds.py)."""
import pytest
import torch

import kv4_bounds as B
import kv4_cases as C

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from iitj_llm_coopt_b200 import kernels
    return kernels.load()


@pytest.mark.parametrize("name", list(C.CASES))
def test_rows_and_heads(K, name):
    seed, lens, news, heads, kv, D, page, window = C.CASES[name]
    q, cache, table = C.inputs(seed, lens, news, heads, kv, D, page, torch.bfloat16)
    want, tol = B.attend(q, cache, table, lens, news, heads, kv, page, D, window)
    assert B.worst(C.attention(K, q, cache, table, lens, news, heads, kv, D, window), want, tol) <= 1.0


@pytest.mark.parametrize("heads,kv", [(2, 2), (4, 1)])        # one and two heads of a group at a time
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window", [0, 450])
def test_a_loud_key_in_the_second_half_of_a_tile(K, heads, kv, D, window):
    """Keys 200, 330 and 500 (places 72, 74 and 116 of tiles of 128 keys that every query sees whole) have scores far above all before
    them, for some rows and not for their neighbours: what was done with the tile's first half has to be scaled down for those alone."""
    lens, news, page = [900, 700], [340, 60], 16
    table, cache = C.pages(31, lens, kv, D, page)
    direction = C.rnd(D, seed=33)
    direction /= direction.norm()
    for b, n in enumerate(lens):
        k, v = C.rnd(n, kv, D, seed=3100 + b), C.rnd(n, kv, D, seed=3150 + b)
        for at, size in ((200, 10.0), (330, 20.0), (500, 30.0)):
            k[at] += size * direction
        C.fill(cache, table, b, page, k.bfloat16(), v.bfloat16())
    T = sum(news)
    # a score of size * along / sqrt(D): 10 to 100 log2 units at key 500 for the rows that are for it, below 0 for those against
    along = (torch.arange(T) % 5 - 1.0) * D ** 0.5 * 0.6
    q = (C.rnd(T, heads, D, seed=34) + along[:, None, None] * direction).flatten(1).bfloat16()
    want, tol = B.attend(q, cache, table, lens, news, heads, kv, page, D, window)
    assert B.worst(C.attention(K, q, cache, table, lens, news, heads, kv, D, window), want, tol) <= 1.0
