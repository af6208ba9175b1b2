"""The bucketed bias table at borders that no formula of ours makes but the interface allows: past every length, repeated,
the type's largest value."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
MAX = np.iinfo(np.int32).max
U = 2.0 ** -24


@pytest.mark.parametrize("causal", [False, True], ids=["two-sided", "causal"])
@pytest.mark.parametrize("T", [1, 40, 700])
@pytest.mark.parametrize("edges", [[0, 3, 9, MAX], [0, 5, MAX - 255, MAX - 254, MAX - 1, MAX, MAX], [0, MAX], [0, 0, 2, 2, 40, 700, 701],
                                   [0], [0, 1, 2, 1 << 29, 1 << 30]],
                         ids=lambda e: f"{len(e)}-borders-to-{e[-1]}")
def test_borders_past_every_length(nrse_device, edges, T, causal):
    from nrse_amd import kernels as K
    H, n = 3, len(edges)
    buckets = n if causal else 2 * n
    e = np.asarray(edges, dtype=np.int32)
    dev = torch.from_numpy(e).to(nrse_device)
    d = np.arange(-(T - 1), T)
    dist = np.maximum(-d, 0) if causal else np.abs(d)
    b = np.searchsorted(e.astype(np.int64), dist, side="right") - 1
    if not causal:
        b = b + (d > 0) * n
    b = torch.from_numpy(b).to(nrse_device)
    g = torch.Generator(device=nrse_device).manual_seed(T + n)
    E = torch.randn(buckets, H, generator=g, device=nrse_device)
    vec = torch.full((H, 2 * T - 1), float("nan"), device=nrse_device)
    K.rel_bias_expand(E, dev, vec, causal=causal)
    assert torch.equal(vec, E[b].t())
    dvec = torch.randn(H, 2 * T - 1, generator=g, device=nrse_device)
    dE = torch.full((buckets, H), float("nan"), device=nrse_device)
    K.rel_bias_collect(dvec, dev, dE, causal=causal)
    want = torch.zeros(buckets, H, dtype=torch.float64, device=nrse_device).index_add_(0, b, dvec.t().double())
    mag = torch.zeros(buckets, H, dtype=torch.float64, device=nrse_device).index_add_(0, b, dvec.t().double().abs())
    # (an empty bucket: exactly zero)
    assert ((dE - want).abs() <= 2 * T * U * mag).all()
