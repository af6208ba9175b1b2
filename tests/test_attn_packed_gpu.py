"""Packed attention with its bucketed bias, and the many-tensor gradient norm, on the GPU against 64-bit references
(tests/packed_reference.py: the value and the error that the formulas allow, element by element)."""
import itertools

import numpy as np
import pytest
import torch

from packed_reference import F64, U, reference, worst

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
NAN = float("nan")


def cu_of(lens, dev):
    return torch.tensor([0, *itertools.accumulate(lens)], dtype=torch.int32, device=dev)


def run(K, q, k, v, cu, dout=None, *, causal=False, scale=None, used=None, gate=None, vec=None, fill=NAN, kv_out=None):
    """Forward and, with dout, backward into buffers filled with `fill`."""
    kw = dict(causal=causal, scale=scale, seq_lens=used, gate=gate, bias_vec=vec)
    r = {"out": torch.full_like(q, fill), "lse": torch.full((q.shape[1], q.shape[0]), fill, device=q.device)}
    K.attn_packed_fwd(q, k, v, cu, r["out"], r["lse"], **kw)
    if dout is not None:
        r["dq"] = torch.full(q.shape, fill, dtype=q.dtype, device=q.device)
        r["dk"], r["dv"] = (torch.full(k.shape, fill, dtype=q.dtype, device=q.device) for _ in range(2))
        if vec is not None:
            r["dvec"] = torch.full_like(vec, fill)
            if gate is not None:
                r["dgate"] = torch.full_like(gate, fill)
        K.attn_packed_bwd(q, k, v, cu, r["out"], dout, r["lse"], r["dq"], r["dk"], r["dv"], dgate=r.get("dgate"),
                          dbias_vec=r.get("dvec"), **kw)
    return r


def check(got, ref, what=""):
    for name in ref:
        w = worst(got[name], ref[name])
        assert w <= 1.0, (what, name, w)


def data(lens, hq, hkv, D, dtype, bias, dev, seed, extra=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    N, T = sum(lens) + extra, max(max(lens), 1) + seed % 3
    rnd = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    q, k, v, do = (rnd(N, h, D).to(dtype) for h in (hq, hkv, hkv, hq))
    gate = 0.5 + torch.rand(hq, N, generator=g, device=dev) if bias == "gated" else None
    vec = rnd(hq, 2 * T - 1) if bias else None
    return q, k, v, do, gate, vec


@pytest.mark.parametrize("lens", [[1], [2, 1], [31, 33, 0, 64], [127, 128, 129], [300, 5, 0, 0, 191, 65]],
                         ids=lambda x: "-".join(map(str, x)))
@pytest.mark.parametrize("heads", [(1, 1), (4, 2), (6, 1), (8, 8)], ids=str)
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("bias", [None, "plain", "gated"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_against_64_bits(nrse_device, dtype, D, bias, causal, heads, lens):
    from nrse_amd import kernels as K
    hq, hkv = heads
    q, k, v, do, gate, vec = data(lens, hq, hkv, D, dtype, bias, nrse_device, sum(lens) + hq)
    cu = cu_of(lens, nrse_device)
    got = run(K, q, k, v, cu, do, causal=causal, gate=gate, vec=vec)
    check(got, reference(q, k, v, cu, causal=causal, gate=gate, vec=vec, dout=do))


@pytest.mark.parametrize("D,causal", [(64, False), (128, True)])
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_long_sequence(nrse_device, dtype, D, causal):
    """Many tiles, scores that grow along the keys (the running maximum moves at every tile)."""
    from nrse_amd import kernels as K
    q, k, v, do, gate, vec = data([1777, 3], 2, 1, D, dtype, "gated", nrse_device, 5)
    k = (k.float() * torch.linspace(0.1, 6.0, k.shape[0], device=nrse_device)[:, None, None]).to(dtype)
    cu = cu_of([1777, 3], nrse_device)
    got = run(K, q, k, v, cu, do, causal=causal, gate=gate, vec=vec)
    check(got, reference(q, k, v, cu, causal=causal, gate=gate, vec=vec, dout=do))


@pytest.mark.parametrize("heads", [(1, 1), (8, 1)], ids=str)
@pytest.mark.parametrize("bias", [None, "gated"])
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("dtype,D", [(BF16, 64), (BF16, 128), (F32, 64), (F32, 128)])
def test_few_blocks(nrse_device, dtype, D, causal, bias, heads):
    """One or two long sequences of few key heads: key blocks in slices and parts, streams over the keys."""
    from nrse_amd import kernels as K
    lens = [1400, 1] if D == 64 else [900]
    q, k, v, do, gate, vec = data(lens, *heads, D, dtype, bias, nrse_device, 8)
    cu = cu_of(lens, nrse_device)
    got = run(K, q, k, v, cu, do, causal=causal, gate=gate, vec=vec)
    check(got, reference(q, k, v, cu, causal=causal, gate=gate, vec=vec, dout=do))


@pytest.mark.parametrize("lens", [[2048] * 3 + [333], [128] * 40 + [1]], ids=["long", "many"])
@pytest.mark.parametrize("bias", [None, "gated"])
@pytest.mark.parametrize("dtype,D", [(BF16, 64), (BF16, 128), (F32, 64)])
def test_many_blocks(nrse_device, dtype, D, bias, lens):
    """Enough blocks for one stream and one slice (the other form of each kernel)."""
    from nrse_amd import kernels as K
    hq = 16
    q, k, v, do, gate, vec = data(lens, hq, hq, D, dtype, bias, nrse_device, 10)
    cu = cu_of(lens, nrse_device)
    got = run(K, q, k, v, cu, do, causal=True, gate=gate, vec=vec)
    check(got, reference(q, k, v, cu, causal=True, gate=gate, vec=vec, dout=do))


@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("bias", [None, "gated"])
@pytest.mark.parametrize("dtype,D", [(BF16, 64), (BF16, 128), (F32, 64), (F32, 128)])
def test_one_stream(nrse_device, dtype, D, bias, causal):
    """Short sequences of many heads in no order of their lengths: one stream over the keys, for every type and mask."""
    from nrse_amd import kernels as K
    lens = [60, 150, 0, 129, 64] * 7 + [333, 1]
    q, k, v, do, gate, vec = data(lens, 16, 4, D, dtype, bias, nrse_device, 24)
    cu = cu_of(lens, nrse_device)
    got = run(K, q, k, v, cu, do, causal=causal, gate=gate, vec=vec)
    check(got, reference(q, k, v, cu, causal=causal, gate=gate, vec=vec, dout=do))


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_scales(nrse_device, scale):
    from nrse_amd import kernels as K
    q, k, v, do, _, _ = data([90, 150], 2, 2, 64, F32, None, nrse_device, 6)
    cu = cu_of([90, 150], nrse_device)
    got = run(K, q, k, v, cu, do, causal=True, scale=scale)
    check(got, reference(q, k, v, cu, causal=True, scale=scale, dout=do))


@pytest.mark.parametrize("layout", ["fused", "heads-first", "odd-stride"])
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_strides(nrse_device, dtype, layout):
    from nrse_amd import kernels as K
    lens, hq, hkv, D = [70, 201], 4, 2, 64
    N = sum(lens)
    q, k, v, do, gate, vec = data(lens, hq, hkv, D, dtype, "gated", nrse_device, 7)
    cu = cu_of(lens, nrse_device)

    def like(x):
        n, h, d = x.shape
        if layout == "heads-first":
            y = torch.full((h, n, d), NAN, dtype=dtype, device=nrse_device).transpose(0, 1)
        elif layout == "odd-stride":     # rows of 3 heads more, starting behind one
            y = torch.full((n, h + 3, d + 8), NAN, dtype=dtype, device=nrse_device)[:, 1:h + 1, :d]
        else:
            y = torch.full((n, 8, d), NAN, dtype=dtype, device=nrse_device)[:, 2:2 + h]
        y.copy_(x)
        return y

    def none(x):
        return like(torch.full_like(x, NAN))
    if layout == "fused":
        qkv = torch.cat([q, k, v], 1)
        qs, ks, vs = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        g = torch.full_like(qkv, NAN)
        dq, dk, dv = g[:, :hq], g[:, hq:hq + hkv], g[:, hq + hkv:]
    else:
        qs, ks, vs = like(q), like(k), like(v)
        dq, dk, dv = none(q), none(k), none(v)
    out, dos = none(q), like(do)
    lse = torch.empty(hq, N, device=nrse_device)
    dgate, dvec = torch.empty_like(gate), torch.empty_like(vec)
    K.attn_packed_fwd(qs, ks, vs, cu, out, lse, gate=gate, bias_vec=vec)
    K.attn_packed_bwd(qs, ks, vs, cu, out, dos, lse, dq, dk, dv, gate=gate, bias_vec=vec, dgate=dgate, dbias_vec=dvec)
    plain = run(K, q, k, v, cu, do, gate=gate, vec=vec)
    for name, x in dict(out=out, lse=lse, dq=dq, dk=dk, dv=dv, dgate=dgate, dvec=dvec).items():
        assert torch.equal(x, plain[name]), name


@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("bias", [None, "gated"])
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_padded_batch_and_rows_of_no_sequence(nrse_device, dtype, bias, causal):
    """Used lengths inside padded stretches, rows before the first and behind the last sequence: what they hold (NaN,
    infinities) reaches nothing, and what is in the outputs there stays, bit for bit."""
    from nrse_amd import kernels as K
    lens, hq, hkv, D = [150, 150, 150, 40], 4, 2, 64
    used = torch.tensor([150, 37, 0, 40], dtype=torch.int32, device=nrse_device)
    q, k, v, do, gate, vec = data(lens, hq, hkv, D, dtype, bias, nrse_device, 9, extra=70 + 3)
    cu = cu_of(lens, nrse_device) + 3
    N = q.shape[0]
    real = torch.zeros(N, dtype=torch.bool, device=nrse_device)
    for i, n in enumerate(used.tolist()):
        real[3 + 150 * i:3 + 150 * i + n] = True
    ref = reference(q, k, v, cu, causal=causal, used=used, gate=gate, vec=vec, dout=do)
    for x in (q, k, v, do):
        x[~real] = torch.tensor([NAN, float("inf"), -float("inf")], device=nrse_device, dtype=dtype).repeat(D)[:D]
    if gate is not None:
        gate[:, ~real] = NAN
    got = run(K, q, k, v, cu, do, causal=causal, used=used, gate=gate, vec=vec, fill=7.0)
    check(got, ref)
    for name in ("out", "dq", "dk", "dv"):
        assert (got[name][~real] == 7.0).all(), name
    for name in ("lse", "dgate"):
        if name in got:
            assert (got[name][:, ~real] == 7.0).all(), name


@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_bias_that_masks(nrse_device, dtype, causal):
    """-inf in the bias: a window (whole tiles of a row left out, the first ones too), and rows that are left nothing
    (zeros, lse -inf, no gradient)."""
    from nrse_amd import kernels as K
    lens, T = [500, 3], 500
    q, k, v, do, gate, _ = data(lens, 2, 1, 64, dtype, "gated", nrse_device, 11)
    cu = cu_of(lens, nrse_device)
    d = torch.arange(-(T - 1), T, device=nrse_device)
    vec = torch.randn(2, 2 * T - 1, device=nrse_device)
    vec[0, (d.abs() > 40)] = -float("inf")
    vec[1, d.abs() < 90] = -float("inf")     # under a causal mask the first 90 rows have no key left
    vec[1, d.abs() > 200] = -float("inf")
    got = run(K, q, k, v, cu, do, causal=causal, gate=gate, vec=vec)
    ref = reference(q, k, v, cu, causal=causal, gate=gate, vec=vec, dout=do)
    check(got, ref)
    empty = torch.isinf(ref["lse"][0])
    assert empty.any() and (got["lse"][empty] == -float("inf")).all()
    assert (got["out"].transpose(0, 1)[empty] == 0).all() and (got["dq"].transpose(0, 1)[empty] == 0).all()
    # the type's lowest value masks as -inf does
    low = torch.where(torch.isinf(vec), torch.full_like(vec, torch.finfo(F32).min), vec)[:1].repeat(2, 1)
    a = run(K, q, k, v, cu, do, causal=causal, gate=gate + 1, vec=low)
    b = run(K, q, k, v, cu, do, causal=causal, gate=gate + 1, vec=vec[:1].repeat(2, 1))
    for name in a:
        assert torch.equal(a[name], b[name]), name


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_extreme_scores(nrse_device, dtype):
    """One score far above the others, and rows whose scores all lie near the type's end."""
    from nrse_amd import kernels as K
    q, k, v, do, _, _ = data([200], 2, 2, 64, dtype, None, nrse_device, 12)
    q[7], k[33] = 60.0, 60.0
    q[11] = 1e4
    cu = cu_of([200], nrse_device)
    got = run(K, q, k, v, cu, do)
    check(got, reference(q, k, v, cu, causal=False, dout=do))


def test_offsets_past_32_bits(nrse_device):
    """Rows 16 MB apart: 300 of them reach 4.7 GB."""
    from nrse_amd import kernels as K
    lens, D = [290, 10], 64
    N = sum(lens)
    big = torch.empty(N, 1 << 23, dtype=BF16, device=nrse_device)
    q, k, v, do, _, _ = data(lens, 1, 1, D, BF16, None, nrse_device, 13)
    cu = cu_of(lens, nrse_device)
    want = run(K, q, k, v, cu, do, causal=True)
    view = [big[:, 64 * i:64 * i + 64].unsqueeze(1) for i in range(8)]
    for x, y in zip(view, (q, k, v, do)):
        x.copy_(y)
    lse = torch.empty(1, N, device=nrse_device)
    K.attn_packed_fwd(view[0], view[1], view[2], cu, view[4], lse, causal=True)
    K.attn_packed_bwd(view[0], view[1], view[2], cu, view[4], view[3], lse, view[5], view[6], view[7], causal=True)
    for x, name in zip(view[4:], ("out", "dq", "dk", "dv")):
        assert torch.equal(x, want[name]), name


def test_cu_seqlens_are_clamped(nrse_device):
    """Bounds past the rows, falling or negative: the sequences are what is left of them inside the tensors."""
    from nrse_amd import kernels as K
    q, k, v, do, _, _ = data([100, 100], 2, 1, 64, F32, None, nrse_device, 14)
    # (held to the reference, not to another call's bits: the number of sequences is part of what the order
    # of the sums goes by)
    ref = reference(q, k, v, cu_of([100, 100], nrse_device), causal=False, dout=do)
    for cu in ([-5, 100, 10 ** 9], [0, 100, 2 ** 31 - 1, 150, 150]):
        c = torch.tensor(cu, dtype=torch.int32, device=nrse_device)
        got = run(K, q, k, v, c, do)
        for name in ref:
            part = (slice(None), slice(0, 100)) if name == "lse" else slice(0, 100)
            assert worst(got[name][part], tuple(x[part] for x in ref[name])) <= 1.0, name


def test_many_sequences(nrse_device):
    """More sequences than a wave has lanes."""
    from nrse_amd import kernels as K
    lens = [(7 * i) % 23 for i in range(333)]
    q, k, v, do, gate, vec = data(lens, 2, 1, 64, F32, "gated", nrse_device, 15)
    cu = cu_of(lens, nrse_device)
    got = run(K, q, k, v, cu, do, causal=True, gate=gate, vec=vec)
    check(got, reference(q, k, v, cu, causal=True, gate=gate, vec=vec, dout=do))


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (BF16, 128), (F32, 64)])
def test_same_bits_and_two_streams(nrse_device, dtype, D):
    from nrse_amd import kernels as K
    lens = [700, 131, 64]
    q, k, v, do, gate, vec = data(lens, 8, 2, D, dtype, "gated", nrse_device, 16)
    cu = cu_of(lens, nrse_device)
    want = run(K, q, k, v, cu, do, causal=True, gate=gate, vec=vec)
    q2, do2 = (q.float() * 0.5).to(dtype), (do.float() * 2).to(dtype)
    want2 = run(K, q2, k, v, cu, do2, causal=True, gate=gate, vec=vec)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):   # two calls at once, each on a stream of its own
        with torch.cuda.stream(s1):
            a = run(K, q, k, v, cu, do, causal=True, gate=gate, vec=vec)
        with torch.cuda.stream(s2):
            b = run(K, q2, k, v, cu, do2, causal=True, gate=gate, vec=vec)
        torch.cuda.synchronize()
        for name in want:
            assert torch.equal(a[name], want[name]) and torch.equal(b[name], want2[name]), name


def test_accumulate_bias_gradient(nrse_device):
    """One bias shared by two layers: the second layer's gradient is added."""
    from nrse_amd import kernels as K
    lens = [130, 41]
    cu = cu_of(lens, nrse_device)
    q, k, v, do, gate, vec = data(lens, 4, 4, 64, F32, "gated", nrse_device, 17)
    one = run(K, q, k, v, cu, do, gate=gate, vec=vec)
    dvec = one["dvec"].clone()
    K.attn_packed_bwd(q, k, v, cu, one["out"], do, one["lse"], one["dq"], one["dk"], one["dv"], gate=gate, bias_vec=vec,
                      dbias_vec=dvec, accumulate=True)
    assert torch.equal(dvec, one["dvec"] + one["dvec"])
    # no rows: overwritten with zeros, or left
    none = torch.zeros(1, dtype=torch.int32, device=nrse_device)
    K.attn_packed_bwd(q, k, v, none, one["out"], do, one["lse"], one["dq"], one["dk"], one["dv"], gate=gate,
                      bias_vec=vec, dbias_vec=dvec, accumulate=True)
    assert torch.equal(dvec, one["dvec"] + one["dvec"])
    K.attn_packed_bwd(q, k, v, none, one["out"], do, one["lse"], one["dq"], one["dk"], one["dv"], gate=gate,
                      bias_vec=vec, dbias_vec=dvec)
    assert (dvec == 0).all()


def test_gradients_against_differences(nrse_device):
    """f32, central differences of sum(out * dout) along random directions."""
    from nrse_amd import kernels as K
    lens = [45, 20]
    cu = cu_of(lens, nrse_device)
    q, k, v, do, gate, vec = data(lens, 4, 2, 64, F32, "gated", nrse_device, 18)
    g = run(K, q, k, v, cu, do, causal=True, gate=gate, vec=vec)
    x = dict(dq=q, dk=k, dv=v, dgate=gate, dvec=vec)

    def loss(y):
        out = torch.empty_like(q)
        K.attn_packed_fwd(y["dq"], y["dk"], y["dv"], cu, out, causal=True, gate=y["dgate"], bias_vec=y["dvec"])
        return float((out.to(F64) * do.to(F64)).sum())
    gen = torch.Generator(device=nrse_device).manual_seed(1)
    for name in x:
        e = torch.randn(x[name].shape, generator=gen, device=nrse_device)
        e = e * (2.0 ** -7 / e.abs().max())
        hi, lo = ({**x, name: x[name] + s * e} for s in (1, -1))
        step = (hi[name].to(F64) - lo[name].to(F64))
        want, got = float((g[name].to(F64) * step).sum()), loss(hi) - loss(lo)
        # the loss: f32 outputs, ~1e3 of them rounded (2^-24 |out dout| each, and the products' sums 100 times
        # that); the differences: third order, (2^-7)^2 of the first
        noise = 100 * U * float((do.abs().to(F64)).sum()) / do.numel() ** 0.5
        size = float((g[name].to(F64).abs() * step.abs()).sum())
        assert abs(want - got) <= noise + 2.0 ** -12 * size, (name, want, got, noise, size)


def test_capture_and_replay(nrse_device):
    """Forward, backward, table and clip recorded once and replayed with new inputs, eager work between."""
    from nrse_amd import hostside as HS
    from nrse_amd import kernels as K
    lens = [120, 61, 200]
    cu = cu_of(lens, nrse_device)
    q, k, v, do, gate, _ = data(lens, 4, 2, 64, BF16, "gated", nrse_device, 19)
    edges = torch.from_numpy(HS.bucket_edges(32, 128)).to(nrse_device)
    E = torch.randn(32, 4, device=nrse_device)

    def step(o):
        K.rel_bias_expand(E, edges, o["vec"])
        K.attn_packed_fwd(q, k, v, cu, o["out"], o["lse"], gate=gate, bias_vec=o["vec"])
        K.attn_packed_bwd(q, k, v, cu, o["out"], do, o["lse"], o["dq"], o["dk"], o["dv"], gate=gate, bias_vec=o["vec"],
                          dgate=o["dgate"], dbias_vec=o["dvec"])
        K.rel_bias_collect(o["dvec"], edges, o["dE"])
        K.clip_grad_norm([o["dq"], o["dk"], o["dv"], o["dE"]], 0.1, o["norm"])

    def buffers():
        f = lambda *s: torch.empty(*s, device=nrse_device)  # noqa: E731
        return dict(vec=f(4, 399), out=torch.empty_like(q), lse=f(4, q.shape[0]), dq=torch.empty_like(q),
                    dk=torch.empty_like(k), dv=torch.empty_like(v), dgate=f(*gate.shape), dvec=f(4, 399), dE=f(32, 4),
                    norm=f(1))
    o = buffers()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(o)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(o)
    gen = torch.Generator(device=nrse_device).manual_seed(3)
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=gen, device=nrse_device))
        E.copy_(torch.randn(E.shape, generator=gen, device=nrse_device))
        w = buffers()
        step(w)
        torch.cuda.synchronize()
        graph.replay()
        w2 = buffers()
        step(w2)
        torch.cuda.synchronize()
        for name in o:
            assert torch.equal(o[name], w[name]) and torch.equal(w2[name], w[name]), (i, name)


@pytest.mark.parametrize("dtype,d,hq,hkv,causal", [(BF16, 64, 4, 2, False), (BF16, 128, 8, 2, True),
                                                   (torch.float32, 64, 4, 4, True)])
def test_a_graph_replays_with_other_lengths(nrse_device, dtype, d, hq, hkv, causal):
    """The lengths are read on the device: a recorded call serves every batch of as many sequences and rows."""
    from nrse_amd import kernels as K
    lens = [120, 61, 200, 9]
    cu = cu_of(lens, nrse_device)
    q, k, v, do, gate, vec = data(lens, hq, hkv, d, dtype, "gated", nrse_device, 23)
    rows, wide = q.shape[0], torch.randn(hq, 2 * 390 - 1, device=nrse_device)

    def step(o):
        kw = dict(causal=causal, gate=gate, bias_vec=wide)
        K.attn_packed_fwd(q, k, v, cu, o["out"], o["lse"], **kw)
        K.attn_packed_bwd(q, k, v, cu, o["out"], do, o["lse"], o["dq"], o["dk"], o["dv"], dgate=o["dgate"],
                          dbias_vec=o["dvec"], **kw)

    def buffers():
        return dict(out=torch.empty_like(q), lse=torch.empty(hq, rows, device=nrse_device), dq=torch.empty_like(q),
                    dk=torch.empty_like(k), dv=torch.empty_like(v), dgate=torch.empty_like(gate),
                    dvec=torch.empty_like(wide))
    o = buffers()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(o)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(o)
    for other in ([390, 0, 0, 0], [1, 129, 128, 132], [0, 0, 195, 195], lens, [97, 98, 97, 98]):
        assert sum(other) == rows
        cu.copy_(cu_of(other, nrse_device))
        graph.replay()
        w = buffers()
        step(w)
        torch.cuda.synchronize()
        for name in o:
            assert torch.equal(o[name], w[name]), (other, name)


def test_wrapper_refusals(nrse_device):
    from nrse_amd import _lib, kernels as K
    q, k, v, do, gate, vec = data([20], 4, 2, 64, BF16, "gated", nrse_device, 20)
    cu, out = cu_of([20], nrse_device), torch.empty_like(q)

    def refused(match, *a, **kw):
        with pytest.raises(_lib.NrseError, match=match):
            K.attn_packed_fwd(*a, **kw)
    refused("shape", q, k[:10], v, cu, out)
    refused("shape", q, k, v[:, :1], cu, out)
    refused("heads", q, k[:, :1].expand(-1, 3, -1), v, cu, out)
    refused("dtype", q.half(), k.half(), v.half(), cu, out.half())
    refused("expected torch.bfloat16", q, k.float(), v, cu, out)
    refused("contiguous", q, k.transpose(0, 2).contiguous().transpose(0, 2), v, cu, out)
    refused("int32", q, k, v, cu.long(), out)
    refused("seq_lens", q, k, v, cu, out, seq_lens=cu)
    refused("head_dim", q[..., :32], k[..., :32], v[..., :32], cu, out[..., :32])
    refused("gate needs", q, k, v, cu, out, gate=gate)
    refused("gate", q, k, v, cu, out, gate=gate[:, :5], bias_vec=vec)
    refused("bias_vec", q, k, v, cu, out, bias_vec=vec[:, :-1])
    refused("lse", q, k, v, cu, out, torch.empty(20, 4, device=nrse_device))
    refused("16-byte", q[:, :, 4:], k[:, :, 4:], v[:, :, 4:], cu, out[:, :, 4:]) if q.shape[2] == 68 else None
    lse = torch.empty(4, 20, device=nrse_device)
    with pytest.raises(_lib.NrseError, match="not there"):
        K.attn_packed_bwd(q, k, v, cu, out, do, lse, q.clone(), k.clone(), v.clone(), dbias_vec=vec)
    edges = torch.arange(8, dtype=torch.int32, device=nrse_device)
    with pytest.raises(_lib.NrseError, match="table"):
        K.rel_bias_expand(torch.randn(15, 4, device=nrse_device), edges, vec)
    with pytest.raises(_lib.NrseError, match="edges"):
        K.rel_bias_expand(torch.randn(16, 4, device=nrse_device), edges.long(), vec)


# ------------------------------------------------------------------------------------------------ the table
@pytest.mark.parametrize("T", [1, 2, 65, 1500])
@pytest.mark.parametrize("buckets,distance", [(320, 800), (32, 128)])
@pytest.mark.parametrize("causal", [False, True], ids=["two-sided", "causal"])
def test_bias_table(nrse_device, causal, buckets, distance, T):
    from nrse_amd import hostside as HS
    from nrse_amd import kernels as K
    H = 5
    e = HS.bucket_edges(buckets, distance, causal)
    edges = torch.from_numpy(e).to(nrse_device)
    E = torch.randn(buckets, H, device=nrse_device)
    vec = torch.full((H, 2 * T - 1), NAN, device=nrse_device)
    K.rel_bias_expand(E, edges, vec, causal=causal)
    d = np.arange(-(T - 1), T)
    if causal:
        b = np.searchsorted(e.astype(np.int64), np.maximum(-d, 0), side="right") - 1
    else:
        b = HS.bucket_vector(T, buckets, distance)
    b = torch.from_numpy(np.asarray(b)).long().to(nrse_device)
    assert torch.equal(vec, E[b].t())
    dvec = torch.randn(H, 2 * T - 1, device=nrse_device)
    dE = torch.full((buckets, H), NAN, device=nrse_device)
    K.rel_bias_collect(dvec, edges, dE, causal=causal)
    want = torch.zeros(buckets, H, dtype=F64, device=nrse_device).index_add_(0, b, dvec.t().to(F64))
    mag = torch.zeros(buckets, H, dtype=F64, device=nrse_device).index_add_(0, b, dvec.t().abs().to(F64))
    assert ((dE - want).abs() <= (2 * T) * U * mag).all()
    again = dE.clone()
    K.rel_bias_collect(dvec, edges, again, causal=causal, accumulate=True)
    assert torch.equal(again, dE + dE)


# ------------------------------------------------------------------------------------------------ gradients' norm
def grads(sizes, dtypes, dev, seed, shift=0):
    """Views of one buffer per type, each `shift` elements off an aligned place."""
    g = torch.Generator(device=dev).manual_seed(seed)
    return [torch.randn(n + shift, generator=g, device=dev).to(dtypes[i % len(dtypes)])[shift:] for i, n in enumerate(sizes)]


@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("dtypes", [(F32,), (BF16,), (F32, BF16)], ids=["f32", "bf16", "both"])
@pytest.mark.parametrize("sizes", [[1], [0, 5, 0], [4095, 4096, 4097], [7 + 13 * (i % 60) for i in range(400)], [3000001, 2, 70000]],
                         ids=["one", "empty", "chunk", "many", "large"])
def test_clip(nrse_device, sizes, dtypes, shift):
    from nrse_amd import kernels as K
    xs = grads(sizes, dtypes, nrse_device, len(sizes), shift)
    was = [x.clone() for x in xs]
    want = float(sum(x.to(F64).square().sum() for x in xs)) ** 0.5
    norm = torch.full((1,), NAN, device=nrse_device)
    K.grad_norm(xs, norm)
    # f64 sums of exact squares, one rounding to f32
    assert abs(float(norm) - want) <= (U + 1e-12) * want
    for limit in (2 * want, float("inf")):     # nothing to clip: the same bits
        n2 = torch.full((1,), NAN, device=nrse_device)
        K.clip_grad_norm(xs, limit, n2)
        assert torch.equal(n2, norm) and all(torch.equal(a, b) for a, b in zip(xs, was))
    K.clip_grad_norm(xs, 0.25 * want, norm)
    c = 0.25 * want / (want + 1e-6)
    for x, w in zip(xs, was):
        # the factor and the product each rounded to f32, the value to its type
        h = 2.0 ** -8 if x.dtype == BF16 else U
        err = (x.to(F64) - w.to(F64) * c).abs()
        assert (err <= (h + 3 * U) * c * w.to(F64).abs()).all()
    K.clip_grad_norm(xs, 0.0, norm)
    assert all((x == 0).all() for x in xs)


def test_clip_ends(nrse_device):
    """Values whose squares leave f32, infinities, NaN; an empty list; the norm's bits from call to call."""
    from nrse_amd import _lib, kernels as K
    norm = torch.full((1,), NAN, device=nrse_device)
    K.grad_norm([], norm)
    assert float(norm) == 0.0
    K.clip_grad_norm([], 1.0, norm)
    assert float(norm) == 0.0
    for v in (1e30, 1e-30):
        x = torch.full((1000,), v, device=nrse_device)
        K.grad_norm([x], norm)
        assert abs(float(norm) / (v * 1000 ** 0.5) - 1) < 1e-6
    x = torch.ones(5000, device=nrse_device)
    x[4500] = float("inf")
    K.clip_grad_norm([x], 1.0, norm)           # as torch: 1 / inf = 0, and 0 * inf is NaN
    assert float(norm) == float("inf") and (x[:4500] == 0).all() and bool(torch.isnan(x[4500]))
    x[4500] = NAN
    K.clip_grad_norm([x], 1.0, norm)
    assert bool(torch.isnan(norm)) and bool(torch.isnan(x).all())
    xs = grads([100000, 3, 777777], (F32, BF16), nrse_device, 2)
    seen = set()
    for _ in range(5):
        K.grad_norm(xs, norm)
        seen.add(float(norm))
    assert len(seen) == 1
    y = torch.ones(64, device=nrse_device)
    for bad in ([y, y], [y[:40], y[39:]]):
        with pytest.raises(_lib.NrseError, match="overlap"):
            K.clip_grad_norm(bad, 1.0, norm)
    for bad in (y.half(), y.view(8, 8).t(), y.cpu()):
        with pytest.raises(_lib.NrseError):
            K.clip_grad_norm([bad], 1.0, norm)
    with pytest.raises(_lib.NrseError, match="max_norm"):
        K.clip_grad_norm([y], -1.0, norm)


# ------------------------------------------------------------------------------------------------ together
def test_a_training_step_of_them(nrse_device):
    """A ragged batch under a learned bucketed bias: table -> bias -> attention -> loss, back to the table, and the clip
    of all gradients, against autograd in 64 bits."""
    from nrse_amd import hostside as HS
    from nrse_amd import kernels as K
    lens, hq, hkv, D = [150, 64, 201], 4, 2, 64
    cu, T = cu_of(lens, nrse_device), 201
    q, k, v, do, gate, _ = data(lens, hq, hkv, D, F32, "gated", nrse_device, 21)
    e = HS.bucket_edges(64, 128)
    edges = torch.from_numpy(e).to(nrse_device)
    E = torch.randn(64, hq, device=nrse_device)
    vec = torch.empty(hq, 2 * T - 1, device=nrse_device)
    K.rel_bias_expand(E, edges, vec)
    g = run(K, q, k, v, cu, do, gate=gate, vec=vec)
    dE = torch.empty_like(E)
    K.rel_bias_collect(g["dvec"], edges, dE)
    leaves = [x.to(F64).requires_grad_() for x in (q, k, v, gate, E)]
    a, b, c, gt, tab = leaves
    bucket = torch.from_numpy(HS.bucket_vector(T, 64, 128)).long().to(nrse_device)
    loss = 0.0
    for lo, hi in zip(cu[:-1].tolist(), cu[1:].tolist()):
        n = hi - lo
        off = torch.arange(n, device=nrse_device)[None] - torch.arange(n, device=nrse_device)[:, None] + T - 1
        for h in range(hq):
            s = a[lo:hi, h] @ b[lo:hi, h // 2].T / 8 + gt[h, lo:hi, None] * tab[bucket[off], h]
            loss = loss + (torch.softmax(s, 1) @ c[lo:hi, h // 2] * do[lo:hi, h].to(F64)).sum()
    loss.backward()
    got = [g["dq"], g["dk"], g["dv"], g["dgate"], dE]
    for x, y in zip(got, leaves):
        # f32 throughout: sums of up to 201 (table: 2e4) terms around zero
        assert float((x - y.grad).norm() / y.grad.norm()) < 2e-5
    norm = torch.empty(1, device=nrse_device)
    K.clip_grad_norm(got, 0.5, norm)
    want = float(sum(y.grad.square().sum() for y in leaves)) ** 0.5
    assert abs(float(norm) / want - 1) < 2e-5
    for x, y in zip(got, leaves):
        ref = y.grad * 0.5 / (want + 1e-6)
        assert float((x - ref).norm() / ref.norm()) < 4e-5
