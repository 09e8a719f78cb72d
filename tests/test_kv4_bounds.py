"""What the bounds of tests/kv4_bounds.py refuse: results of attention over a packed cache with one mistake in them."""
import pytest
import torch

import kv4_bounds as B
import kv4_cases as C

WRONG = ["scale", "first", "step", "window", "tile", "zeros"]


@pytest.mark.parametrize("wrong", WRONG)
@pytest.mark.parametrize("name", list(C.CASES))
def test_a_mistake_is_refused(name, wrong):
    seed, lens, news, heads, kv, D, page, window = C.CASES[name]
    q, cache, table = C.inputs(seed, lens, news, heads, kv, D, page, torch.bfloat16)
    if (wrong == "window" and not any(window and t > window for t in lens)) or (wrong in ("first", "tile") and window and window < 300):
        pytest.skip("the mistake changes nothing here")
    if wrong == "tile" and max(lens) < 400:
        pytest.skip("the mistake changes nothing here")
    want, tol = B.attend(q, cache, table, lens, news, heads, kv, page, D, window)
    if wrong == "zeros":
        got = torch.zeros_like(want)
    else:
        got, _ = B.attend(q, cache, table, lens, news, heads, kv, page, D, window, wrong=wrong)
    assert B.worst(want.bfloat16(), want, tol) <= 1.0                # the result rounded once is fine
    assert B.worst(got.bfloat16(), want, tol) > 1.0
    if wrong != "window":                                            # and not for one row alone
        assert ((got - want).norm(dim=-1) > tol).float().mean() > (0.9 if wrong == "zeros" else 0.02)
