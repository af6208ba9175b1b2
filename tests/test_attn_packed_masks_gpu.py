"""Packed attention under masks written as finite biases, against 64 bits (tests/packed_bounds.py): first tiles masked,
windows, rows of nothing but masks, rows without a score above -2^6, NaN."""
import math

import pytest
import torch

from packed_bounds import reference
from packed_reference import worst
from test_attn_packed_gpu import check, cu_of, data, run

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
LOWEST = torch.finfo(F32).min
NAN = float("nan")


def masked(lens, hq, hkv, D, dtype, dev, seed, mask, kind):
    """Gates from 0.1 to 2; `kind`: the keys far behind the query, a window around it, or every key but that window."""
    q, k, v, do, _, _ = data(lens, hq, hkv, D, dtype, None, dev, seed)
    g = torch.Generator(device=dev).manual_seed(seed)
    T = max(lens)
    gate = 0.1 + 1.9 * torch.rand(hq, sum(lens), generator=g, device=dev)
    vec = torch.randn(hq, 2 * T - 1, generator=g, device=dev)
    d = torch.arange(-(T - 1), T, device=dev)
    vec[:, {"behind": d < -200, "outside": d.abs() > 40, "inside": d.abs() < 90}[kind]] = mask
    return q, k, v, do, gate, vec


@pytest.mark.parametrize("mask", [-1e3, -1e4, -1e6, -1e9, -1e30, LOWEST, -math.inf])
@pytest.mark.parametrize("kind", ["behind", "outside"])
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("dtype,D", [(BF16, 64), (BF16, 128), (F32, 64), (F32, 128)])
def test_finite_masks_few_rows(nrse_device, dtype, D, causal, kind, mask):
    """Two streams over the keys."""
    from nrse_amd import kernels as K
    lens = [512, 3, 290]
    q, k, v, do, gate, vec = masked(lens, 2, 1, D, dtype, nrse_device, 41, mask, kind)
    cu = cu_of(lens, nrse_device)
    got = run(K, q, k, v, cu, do, causal=causal, gate=gate, vec=vec)
    check(got, reference(q, k, v, cu, causal=causal, gate=gate, vec=vec, dout=do))


@pytest.mark.parametrize("mask", [-1e3, -1e6, -1e30])
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("dtype,D", [(BF16, 64), (BF16, 128), (F32, 64), (F32, 128)])
def test_finite_masks_one_stream(nrse_device, dtype, D, causal, mask):
    from nrse_amd import kernels as K
    lens = [512] * 9
    q, k, v, do, gate, vec = masked(lens, 16, 4, D, dtype, nrse_device, 42, mask, "behind")
    cu = cu_of(lens, nrse_device)
    got = run(K, q, k, v, cu, do, causal=causal, gate=gate, vec=vec)
    check(got, reference(q, k, v, cu, causal=causal, gate=gate, vec=vec, dout=do))


@pytest.mark.parametrize("mask", [-300.0, -5e3, -1e6, -1e9, -1e30, LOWEST, -math.inf])
@pytest.mark.parametrize("dtype,D", [(BF16, 64), (F32, 64)])
@pytest.mark.parametrize("hq", [2, 48], ids=["two-streams", "one-stream"])
def test_rows_of_nothing_but_masks(nrse_device, hq, dtype, D, mask):
    """Causal, the 90 nearest keys masked: the first 90 rows of a sequence have none left. Down to -2^14 they are the
    softmax of what the mask hides; below they are left nothing: zeros, lse -inf, no gradient."""
    from nrse_amd import kernels as K
    lens = [1] + [140] * 9
    q, k, v, do, gate, vec = masked(lens, hq, 1, D, dtype, nrse_device, 43, mask, "inside")
    cu = cu_of(lens, nrse_device)
    got = run(K, q, k, v, cu, do, causal=True, gate=gate, vec=vec)
    ref = reference(q, k, v, cu, causal=True, gate=gate, vec=vec, dout=do)
    check(got, ref)
    none = torch.isinf(ref["lse"][0])
    assert bool(none.any()) == (mask <= -1e6)
    assert (got["lse"][none] == -math.inf).all()
    for name in ("out", "dq"):
        assert (got[name].transpose(0, 1)[none] == 0).all(), name
    assert (got["dgate"][none] == 0).all()


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (BF16, 128), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("hq,lens", [(2, [300, 5]), (16, [300, 70] * 12)], ids=["two-streams", "one-stream"])
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
def test_rows_whose_scores_are_all_low(nrse_device, causal, hq, lens, dtype, D):
    """No score of some rows reaches -2^6, by the products alone: they are swept again relative to their largest."""
    from nrse_amd import kernels as K
    q, k, v, do, _, _ = data(lens, hq, 1, D, dtype, None, nrse_device, 44)
    k = (k.float() * 0.2 + 1).to(dtype)
    low = torch.arange(q.shape[0], device=nrse_device) % 3 == 1
    q[low] = (q[low].float() * 0.2 - 12 - 20 * (torch.arange(int(low.sum()), device=nrse_device) % 4)[:, None, None]).to(dtype)
    cu = cu_of(lens, nrse_device)
    ref = reference(q, k, v, cu, causal=causal, dout=do)
    assert (ref["lse"][0] < -70).any() and (ref["lse"][0] > -20).any()
    check(run(K, q, k, v, cu, do, causal=causal), ref)


@pytest.mark.parametrize("hq", [2, 48], ids=["two-streams", "one-stream"])
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_distance_slopes(nrse_device, dtype, hq):
    """A bias that falls with the distance, to thousands: most tiles of a row lie below -2^6."""
    from nrse_amd import kernels as K
    lens = [600, 33] if hq == 2 else [200] * 9
    T = max(lens)
    q, k, v, do, _, _ = data(lens, hq, hq // 2, 64, dtype, None, nrse_device, 45)
    d = torch.arange(-(T - 1), T, device=nrse_device, dtype=F32)
    vec = (-d.abs() * torch.linspace(0.1, 9, hq, device=nrse_device)[:, None]).contiguous()
    cu = cu_of(lens, nrse_device)
    for causal in (False, True):
        got = run(K, q, k, v, cu, do, causal=causal, vec=vec)
        check(got, reference(q, k, v, cu, causal=causal, vec=vec, dout=do))


@pytest.mark.parametrize("bias", [None, "gated"])
@pytest.mark.parametrize("dtype,D", [(BF16, 64), (BF16, 128), (F32, 64)])
@pytest.mark.parametrize("hq", [2, 48], ids=["two-streams", "one-stream"])
def test_a_row_of_nan_is_nan_and_no_other(nrse_device, hq, dtype, D, bias):
    from nrse_amd import kernels as K
    lens = [140] * 9
    q, k, v, _, gate, vec = data(lens, hq, 1, D, dtype, bias, nrse_device, 46)
    cu = cu_of(lens, nrse_device)
    want = run(K, q, k, v, cu, causal=True, gate=gate, vec=vec)
    q[77, 1] = NAN
    got = run(K, q, k, v, cu, causal=True, gate=gate, vec=vec)
    hit = torch.zeros(q.shape[:2], dtype=torch.bool, device=nrse_device)
    hit[77, 1] = True
    assert torch.isnan(got["out"][hit]).all() and torch.isnan(got["lse"][hit.t()]).all()
    assert torch.equal(got["out"][~hit], want["out"][~hit]) and torch.equal(got["lse"][~hit.t()], want["lse"][~hit.t()])


def test_a_row_left_nothing_is_zeros_beside_infinite_values(nrse_device):
    """A masked key's value does not reach a row that is left nothing."""
    from nrse_amd import kernels as K
    q, k, v, _, _, _ = data([100], 2, 1, 64, F32, None, nrse_device, 47)
    vec = torch.full((2, 199), -1e9, device=nrse_device)
    v[50] = float("inf")
    got = run(K, q, k, v, cu_of([100], nrse_device), vec=vec)
    assert (got["out"] == 0).all() and (got["lse"] == -math.inf).all()
    assert worst(got["out"], (torch.zeros_like(got["out"], dtype=torch.float64),) * 2) == 0
