"""The bound that holds the packed forward under large finite masks, on the CPU: a restatement of its row in f32, step by
step, keeps it; one that takes a row's first tile for its reference whatever it holds does not."""
import math

import numpy as np
import pytest
import torch

from packed_bounds import reference

f = np.float32
LOG2E = f(1.4426950408889634)


def fma(a, b, c):
    return (np.asarray(a, np.float64) * np.asarray(b, np.float64) + np.asarray(c, np.float64)).astype(np.float32)


def forward_row(s, bias, gate, V, floor, tile=64):
    """One row of the forward in f32: s q.k in f32, `floor` the score from which a row takes a reference."""
    c1, gl = f(0.125) * LOG2E, f(gate) * LOG2E
    o, l, mref, thr = np.zeros(V.shape[1], np.float32), f(0), f(0), -math.inf

    def sweep():
        nonlocal o, l, mref, thr
        o, l = np.zeros(V.shape[1], np.float32), f(0)
        for k in range(0, len(s), tile):
            v = fma(s[k:k + tile], c1, fma(gl, bias[k:k + tile], -mref))
            mx = v.max()
            if mx > thr:
                first = thr < 0
                low = first and not mx > floor
                sh = f(0) if low else mx if first else max(mx, f(0))
                al = f(np.exp2(np.float64(-sh))) if np.any(o) or l else f(1)
                thr = max(thr, mx) if low else 8.0
                mref, l, o, v = f(mref + sh), f(l * al), o * al, (v - sh).astype(np.float32)
            p = np.exp2(v.astype(np.float64)).astype(np.float32)
            l, o = f(l + p.sum(dtype=np.float64)), (o + p.astype(np.float64) @ V[k:k + tile]).astype(np.float32)

    sweep()
    if thr < 0 and thr > -16384 * LOG2E:
        mref, thr = f(thr), 8.0
        sweep()
    if thr < 0:
        return np.zeros(V.shape[1]), -math.inf
    return o.astype(np.float64) / float(l), (float(mref) + math.log2(l)) * math.log(2)


@pytest.mark.parametrize("gate", [0.1, 0.6, 1.0, 2.0])
@pytest.mark.parametrize("mask", [-1e3, -1e4, -1e6, -1e9, -1e30, float(np.finfo(np.float32).min), -math.inf])
def test_the_bound_tells_the_forms_apart(mask, gate):
    rng = np.random.default_rng(1)
    n, D = 512, 64
    K, V, Q = (torch.from_numpy(rng.standard_normal((n, 1, D)).astype(np.float32)) for _ in range(3))
    vec = torch.from_numpy(rng.standard_normal((1, 2 * n - 1)).astype(np.float32))
    i = 511
    vec[0, n - 1 - i:n - 1 - i + 266] = mask          # row i: the first 266 keys
    g = torch.full((1, n), gate)
    ref = reference(Q, K, V, torch.tensor([0, n]), causal=False, gate=g, vec=vec)
    s = (Q[i, 0].numpy().astype(np.float64) @ K[:, 0].numpy().T.astype(np.float64)).astype(np.float32)
    bias = vec[0, n - 1 - i:2 * n - 1 - i].numpy()

    def worst(floor):
        with np.errstate(over="ignore", invalid="ignore"):
            o, lse = forward_row(s, bias, gate, V[:, 0].numpy().astype(np.float64), floor)
        eo = np.abs(o - ref["out"][0][i, 0].numpy()) / ref["out"][1][i, 0].numpy()
        return max(eo.max(), abs(lse - float(ref["lse"][0][0, i])) / float(ref["lse"][1][0, i]))
    assert worst(-64.0) <= 1
    # the reference of the first tile, whatever it holds: a visible score is off by up to half a step of mask * gate * log2 e,
    # from 2^-6 on at 2^18, against 2 e_s of about 2^-10
    if mask > -1e38 and mask * gate < -2.0 ** 18:
        assert not worst(-math.inf) <= 1


@pytest.mark.parametrize("mask,left", [(-500.0, True), (-5000.0, True), (-1e9, False), (-1e30, False), (-math.inf, False)])
def test_rows_of_nothing_but_masks(mask, left):
    """Such a row is the softmax of what the mask hides, as long as its lse can tell, and nothing below -2^14."""
    rng = np.random.default_rng(2)
    n, D = 130, 64
    K, V, Q = (torch.from_numpy(rng.standard_normal((n, 1, D)).astype(np.float32)) for _ in range(3))
    vec = torch.full((1, 2 * n - 1), mask)
    ref = reference(Q, K, V, torch.tensor([0, n]), causal=False, vec=vec)
    assert bool(torch.isinf(ref["lse"][0]).all()) is not left
    s = (Q[5, 0].numpy().astype(np.float64) @ K[:, 0].numpy().T.astype(np.float64)).astype(np.float32)
    with np.errstate(invalid="ignore"):
        o, lse = forward_row(s, np.full(n, mask, np.float32), 1.0, V[:, 0].numpy().astype(np.float64), -64.0)
    if left:
        assert (np.abs(o - ref["out"][0][5, 0].numpy()) <= ref["out"][1][5, 0].numpy()).all()
        assert abs(lse - float(ref["lse"][0][0, 5])) <= float(ref["lse"][1][0, 5])
    else:
        assert (o == 0).all() and lse == -math.inf
