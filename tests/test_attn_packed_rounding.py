"""tests/packed_rounding.py tells the two roundings of the bf16 backward apart (CPU)."""
import pytest

from packed_rounding import case, error, gradients


@pytest.mark.parametrize("name,keys,values", [("dq", 1.0, 0.0), ("dk", 0.0, 1.0)])
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("D,hq,hkv", [(64, 4, 2), (128, 4, 1)])
def test_the_coarser_form_is_seen(D, hq, hkv, causal, name, keys, values):
    lens = [500, 131]
    exact, fine, coarse = gradients(*case(lens, hq, hkv, D, 52, keys, values), lens, causal)[name]
    assert error(coarse, exact) > 1.1 * error(fine, exact)
