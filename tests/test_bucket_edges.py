"""hostside.bucket_edges over many sizes: every border is a distance that is there."""
import numpy as np
import pytest

from nrse_amd import hostside as HS


@pytest.mark.parametrize("causal", [False, True], ids=["two-sided", "causal"])
def test_every_border_is_found(causal):
    rng = np.random.default_rng(0)
    for _ in range(400):
        n = int(rng.integers(2, 200))
        buckets = n if causal else 2 * n
        distance = int(n // 2 + 1 + np.exp(rng.uniform(0, 9)))
        e = HS.bucket_edges(buckets, distance, causal)
        assert e[0] == 0 and len(e) == n and (np.diff(e) >= 0).all() and e[-1] <= distance, (buckets, distance)
