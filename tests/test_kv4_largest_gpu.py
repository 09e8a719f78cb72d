"""The packed cache of a float32 engine: numbers next to the largest float32."""
import pytest
import torch

import kv4_cases as C

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from iitj_llm_coopt_b200 import kernels
    return kernels.load()


LARGEST = 3.4028234663852886e38


@pytest.mark.parametrize("which", ["key", "value"])
def test_a_step_rounded_up_past_the_largest_number(K, which):
    """0 and the largest float32 in a group: a step of 137 2^117, of which fifteen are more than float32 holds.  The token counts as one
    that is not finite."""
    kv, D, page, T = 2, 64, 4, 12
    x = C.rnd(T, 3 * kv, D, seed=41)
    at = kv + (0 if which == "key" else kv)
    x[5, at, :32] = 0.0
    x[5, at, 7] = LARGEST
    x[6, at, :32] = LARGEST / 2                        # (this one's top code is below)
    x[6, at, 0] = 0.0
    x[7, at, :32] = -LARGEST * 0.99
    x[7, at, 3] = 0.0
    qkv = x.flatten(1)
    cache = torch.zeros(3, kv * page * (D // 32) * 40, dtype=torch.uint8, device="cuda")
    slots = torch.arange(T, dtype=torch.int32, device="cuda")
    K.rope_store_kv4(qkv.cuda(), None, slots, cache, kv, kv, D, 0)
    kept = K.kv4_read(cache, slots, torch.empty(T, 2, kv, D, device="cuda"), kv, D).cpu()
    assert bool(kept[5, 0, 0].isnan().all()) and bool((kept[5, 1, 0] == 0).all())
    kept[5, :, 0] = 0
    assert bool(kept.isfinite().all())
    assert abs(kept[6, 0 if which == "key" else 1, 0, 1].item() / (LARGEST / 2) - 1) < 1 / 15
    # queries that do not see the token, in one tile with some that do
    q = torch.ones(T, kv * D)
    table = torch.arange(3, dtype=torch.int32).view(1, 3)
    got = C.attention(K, q, cache.cpu(), table, [T], [T], kv, kv, D).view(T, kv, D)
    assert bool(got[:5].isfinite().all()) and bool(got[5:, 0].isnan().all())
