"""Packed attention, bucketed bias and many-tensor gradient norm, host side (CPU): the C entry points refuse what the
kernels do not take before anything is launched, and the bucket borders are the buckets."""
import ctypes
import os

import numpy as np
import pytest
import torch

from nrse_amd import _lib
from nrse_amd import hostside as HS
from nrse_amd import kernels as K

pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")
A = 1 << 20   # an aligned address that is never read: every call below is refused on the host


def fwd_params(**kw):
    p = _lib.AttnPackedFwdParams()
    d = dict(dtype=_lib.BF16, q=A, k=A, v=A, out=A, lse=A, cu_seqlens=A, nseq=2, rows=256, hq=8, hkv=2, head_dim=64,
             scale=0.125, bias_len=0)
    for s, heads in (("q", 8), ("k", 2), ("v", 2), ("out", 8)):
        d[s + "_row"], d[s + "_head"] = heads * 64, 64
    d.update(kw)
    for k, v in d.items():
        setattr(p, k, v)
    return p


def bwd_params(**kw):
    p = _lib.AttnPackedBwdParams()
    d = dict(dtype=_lib.BF16, q=A, k=A, v=A, out=A, dout=A, dq=A, dk=A, dv=A, lse=A, delta=A, cu_seqlens=A, nseq=2,
             rows=256, hq=8, hkv=2, head_dim=64, scale=0.125, bias_len=0)
    for s, heads in (("q", 8), ("k", 2), ("v", 2), ("out", 8), ("dout", 8), ("dq", 8), ("dk", 2), ("dv", 2)):
        d[s + "_row"], d[s + "_head"] = heads * 64, 64
    d.update(kw)
    for k, v in d.items():
        setattr(p, k, v)
    return p


COMMON = [(dict(dtype=_lib.FP8), "dtype"), (dict(dtype=_lib.BF16X3), "dtype"), (dict(head_dim=80), "head_dim"),
          (dict(head_dim=256), "head_dim"), (dict(hq=6, hkv=4), "heads"), (dict(hkv=0), "heads"), (dict(hq=0), "heads"),
          (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"), (dict(nseq=-1), "rows"),
          (dict(cu_seqlens=None), "cu_seqlens"), (dict(gate=A), "bias"), (dict(bias_vec=A, bias_len=0), "bias_len"),
          (dict(q=None), "q is null"), (dict(k=A + 8), "k: base"), (dict(v_row=132), "v: base"),
          (dict(q_head=60), "q: base"), (dict(k_row=56), "row stride"), (dict(q_row=1 << 24), "row stride"),
          (dict(k_head=0), "head stride"), (dict(out=None), "out is null"), (dict(out_row=0), "row stride")]


@pytest.mark.parametrize("kw,word", COMMON)
def test_refusals(kw, word):
    L = _lib.lib()
    for p, fn in ((fwd_params(**kw), L.nrse_attn_packed_fwd), (bwd_params(**kw), L.nrse_attn_packed_bwd)):
        assert fn(ctypes.byref(p), None) < 0
        assert word in L.nrse_last_error().decode(), L.nrse_last_error()


@pytest.mark.parametrize("kw,word", [
    (dict(dout=None), "dout is null"), (dict(dq=A + 2), "dq: base"), (dict(dk_row=60), "dk: base"),
    (dict(dv=None), "dv is null"), (dict(lse=None), "lse"), (dict(delta=None), "delta"),
    (dict(dbias_vec=A), "not there"), (dict(dgate=A), "not there"),
    (dict(bias_vec=A, bias_len=300, dgate=A), "without a gate"),
    (dict(bias_vec=A, bias_len=300, dbias_vec=A), "workspace"), (dict(rows=4096, nseq=1), "workspace")])
def test_backward_refusals(kw, word):
    L = _lib.lib()
    assert L.nrse_attn_packed_bwd(ctypes.byref(bwd_params(**kw)), None) < 0
    assert word in L.nrse_last_error().decode(), L.nrse_last_error()


def apart(make, **kw):
    """Every operand at an address of its own."""
    names = [n for n, _ in make()._fields_ if f"{n}_row" in dict(make()._fields_)]
    return make(**{**{n: A + (i << 32) for i, n in enumerate(names)}, **kw})


@pytest.mark.parametrize("make,kw", [
    (fwd_params, dict(out="q")), (fwd_params, dict(out="v")), (bwd_params, dict(dq="q")), (bwd_params, dict(dk="k")),
    (bwd_params, dict(dv="dout")), (bwd_params, dict(dq="out")), (bwd_params, dict(dv="dk"))])
def test_outputs_at_another_operands_address_are_refused(make, kw):
    L = _lib.lib()
    p = apart(make, rows=100000, nseq=10)
    for name, of in kw.items():
        setattr(p, name, getattr(p, of))
    fn = L.nrse_attn_packed_fwd if make is fwd_params else L.nrse_attn_packed_bwd
    assert fn(ctypes.byref(p), None) < 0 and "address" in L.nrse_last_error().decode(), L.nrse_last_error()


@pytest.mark.parametrize("make,name", [(fwd_params, "out"), (bwd_params, "dq"), (bwd_params, "dk"), (bwd_params, "dv")])
def test_outputs_whose_rows_and_heads_overlap_are_refused(make, name):
    L = _lib.lib()
    p = apart(make, rows=100000, nseq=10, **{f"{name}_row": 64, f"{name}_head": 64})
    fn = L.nrse_attn_packed_fwd if make is fwd_params else L.nrse_attn_packed_bwd
    assert fn(ctypes.byref(p), None) < 0 and "overlap" in L.nrse_last_error().decode(), L.nrse_last_error()


@pytest.mark.parametrize("make", [fwd_params, bwd_params])
def test_grids_past_the_launch_limit_are_refused(make):
    L = _lib.lib()
    p = apart(make, rows=1 << 28, nseq=1)   # 2^21 blocks of 8 heads
    fn = L.nrse_attn_packed_fwd if make is fwd_params else L.nrse_attn_packed_bwd
    assert fn(ctypes.byref(p), None) < 0 and "workgroups" in L.nrse_last_error().decode(), L.nrse_last_error()


@pytest.mark.parametrize("make", [fwd_params, bwd_params])
@pytest.mark.parametrize("delta", [-8, 8])
def test_struct_size_is_checked(make, delta):
    L = _lib.lib()
    p = make()
    p.struct_size += delta
    fn = L.nrse_attn_packed_fwd if make is fwd_params else L.nrse_attn_packed_bwd
    assert fn(ctypes.byref(p), None) == -1 and "struct_size" in L.nrse_last_error().decode()
    if make is bwd_params:
        assert L.nrse_attn_packed_bwd_workspace(ctypes.byref(p)) == -1


def test_nothing_to_do_is_no_error():
    """No rows or no sequences: nothing is launched and no pointer is needed."""
    L = _lib.lib()
    for kw in (dict(rows=0, q=None, k=None, v=None, out=None), dict(nseq=0, cu_seqlens=None)):
        assert L.nrse_attn_packed_fwd(ctypes.byref(fwd_params(**kw)), None) == 0
        assert L.nrse_attn_packed_bwd(ctypes.byref(bwd_params(**kw)), None) == 0


def test_workspace():
    """The bias gradient's slab, and the sums of sliced key blocks where a batch has too few of them for the chip; a
    batch with enough blocks needs neither."""
    L = _lib.lib()

    def floats(**kw):
        return L.nrse_attn_packed_bwd_workspace(ctypes.byref(bwd_params(**kw)))
    assert floats(rows=100000, hkv=8, nseq=10) == 0
    assert floats(rows=100000, hkv=8, nseq=10, bias_vec=A, bias_len=256) == 0
    assert floats(rows=100000, hkv=8, nseq=10, bias_vec=A, bias_len=256, dbias_vec=A) > 0
    few = floats(rows=4096, hkv=1, nseq=1)
    assert few > 0 and few % (2 * 4096 * 64) == 0
    assert floats(rows=0) == 0 and floats(nseq=0) == 0


def test_wrappers_take_device_tensors_only():
    q, k = torch.zeros(4, 2, 64), torch.zeros(4, 2, 64)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(_lib.NrseError, match="device tensors"):
        K.attn_packed_fwd(q, k, k, cu, torch.empty_like(q))
    for shape in ((5,), (2, 4), (1, 2, 3)):   # (not [heads, 2 T - 1])
        with pytest.raises(_lib.NrseError, match="heads, 2 T - 1"):
            K.rel_bias_expand(q, cu, torch.zeros(shape))
    with pytest.raises(_lib.NrseError, match="on the device"):
        K.grad_norm([q], torch.zeros(1))
    with pytest.raises(_lib.NrseError, match="on the device"):
        K.clip_grad_norm([q], 1.0, torch.zeros(1))


@pytest.mark.parametrize("buckets,distance", [(320, 800), (32, 128), (64, 256), (4, 3), (16, 1000000)])
def test_bucket_edges_are_bucket_vector(buckets, distance):
    T = 3000
    edges = HS.bucket_edges(buckets, distance).astype(np.int64)
    assert edges[0] == 0 and (np.diff(edges) >= 0).all() and len(edges) == buckets // 2
    d = np.arange(-(T - 1), T)
    b = np.searchsorted(edges, np.abs(d), side="right") - 1 + (d > 0) * (buckets // 2)
    assert np.array_equal(b, HS.bucket_vector(T, buckets, distance))


def test_bucket_edges_causal_and_refusals():
    edges = HS.bucket_edges(32, 128, causal=True)
    assert len(edges) == 32 and edges[16] == 16 and edges[31] <= 128 and (np.diff(edges) > 0).all()
    for bad in ((2, 128), (32, 8), (0, 10)):
        with pytest.raises(ValueError):
            HS.bucket_edges(*bad)


def lists(*sizes, dtype=_lib.F32, at=None):
    n = len(sizes)
    where, ptrs = A, []
    for s in sizes:
        ptrs.append(where)
        where += s * 4 + 4
    ptrs = ptrs if at is None else at
    return ((ctypes.c_void_p * n)(*ptrs), (ctypes.c_longlong * n)(*sizes), (ctypes.c_int * n)(*[dtype] * n), n)


def test_gradient_lists_are_checked():
    L = _lib.lib()
    ws = L.nrse_grad_norm_workspace(*lists(5, 0, 100000))
    assert ws >= 3
    assert L.nrse_grad_norm_workspace(*lists(5, dtype=_lib.FP8)) < 0 and "dtype" in L.nrse_last_error().decode()
    assert L.nrse_grad_norm_workspace(*lists(5, -1)) < 0
    assert L.nrse_grad_norm_workspace(*lists(5, at=[None])) < 0
    assert L.nrse_grad_norm_workspace(*lists(5, at=[A + 2])) < 0 and "address" in L.nrse_last_error().decode()
    assert L.nrse_clip_grad_norm(*lists(5), 1.0, None, A, None) < 0 and "null" in L.nrse_last_error().decode()
    assert L.nrse_clip_grad_norm(*lists(5), -1.0, A, A, None) < 0 and "max_norm" in L.nrse_last_error().decode()
    assert L.nrse_clip_grad_norm(*lists(5), float("nan"), A, A, None) < 0
    for at in ([A, A], [A, A + 16], [A + 16, A]):   # the same tensor twice, two that overlap
        assert L.nrse_clip_grad_norm(*lists(5, 5, at=at), 1.0, A, A, None) < 0
        assert "overlap" in L.nrse_last_error().decode()


@pytest.mark.parametrize("bad", [dict(n=0), dict(H=0), dict(T=0), dict(edges=None), dict(E=None), dict(vec=None)])
def test_bias_table_refusals(bad):
    L = _lib.lib()
    a = dict(E=A, edges=A, n=16, vec=A, H=4, T=100)
    a.update(bad)
    assert L.nrse_rel_bias_expand(a["E"], a["edges"], a["n"], a["vec"], a["H"], a["T"], 0, None) < 0
    assert L.nrse_rel_bias_collect(a["vec"], a["edges"], a["n"], a["E"], a["H"], a["T"], 0, 0, None) < 0
