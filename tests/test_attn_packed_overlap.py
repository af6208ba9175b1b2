"""What packed attention and the gradient norm refuse on the host, before anything is launched (CPU): outputs that share
memory with another operand, wholly or in part, and launches past their grid."""
import ctypes
import os

import pytest

from nrse_amd import _lib
from test_attn_packed import A, bwd_params, fwd_params

pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")
ROWS, T = 100000, 300
FAR = 1 << 34


def spread(make):
    """Every operand, a gated bias among them, at an address of its own."""
    names = ["q", "k", "v", "out", "lse", "cu_seqlens", "seq_lens", "bias_vec", "gate"]
    if make is bwd_params:
        names += ["dout", "dq", "dk", "dv", "delta", "dgate", "dbias_vec", "part"]
    return make(rows=ROWS, nseq=10, bias_len=T, **{n: A + i * FAR for i, n in enumerate(names)})


def refusal(make, p):
    L = _lib.lib()
    fn = L.nrse_attn_packed_fwd if make is fwd_params else L.nrse_attn_packed_bwd
    assert fn(ctypes.byref(p), None) < 0
    return L.nrse_last_error().decode()


HQ, HKV = 8 * 128 * ROWS, 2 * 128 * ROWS     # bytes of the operands of test_attn_packed's shapes
VEC, PER_ROW = 8 * (2 * T - 1) * 4, 8 * ROWS * 4


@pytest.mark.parametrize("out,of,by", [
    ("out", "q", HQ - 128), ("out", "k", HKV - 16), ("out", "v", -HQ + 16), ("out", "gate", 0), ("out", "bias_vec", VEC - 16),
    ("out", "cu_seqlens", 32), ("out", "seq_lens", -HQ + 16), ("lse", "q", 1024), ("lse", "out", HQ - 4), ("lse", "cu_seqlens", 40),
    ("lse", "gate", PER_ROW - 4), ("lse", "bias_vec", 0)])
def test_forward(out, of, by):
    p = spread(fwd_params)
    setattr(p, out, getattr(p, of) + by)
    e = refusal(fwd_params, p)
    assert "share" in e and out in e and of in e, e


@pytest.mark.parametrize("out,of,by", [
    ("dq", "q", 128), ("dq", "out", HQ - 16), ("dq", "lse", 0), ("dk", "dv", HKV - 16), ("dk", "k", -HKV + 16), ("dv", "dout", 160),
    ("dv", "dq", HQ - 16), ("delta", "lse", 0), ("delta", "gate", 4), ("delta", "dgate", PER_ROW - 4), ("delta", "q", 0),
    ("dgate", "gate", 0), ("dgate", "lse", -PER_ROW + 4), ("dbias_vec", "bias_vec", VEC - 4), ("dbias_vec", "dk", 0),
    ("dbias_vec", "delta", 0), ("part", "q", HQ - 16), ("part", "lse", 0), ("part", "dq", 16), ("part", "bias_vec", 0),
    ("part", "seq_lens", 32), ("part", "delta", 0)])
def test_backward(out, of, by):
    p = spread(bwd_params)
    setattr(p, out, getattr(p, of) + by)
    e = refusal(bwd_params, p)
    assert "share" in e and out in e and of in e, e


def test_the_end_of_the_workspace_counts():
    p = spread(bwd_params)
    n = _lib.lib().nrse_attn_packed_bwd_workspace(ctypes.byref(p))
    assert n > 0
    p.q = p.part + 4 * (n - n % 4) - 16
    assert "share" in refusal(bwd_params, p)


def test_an_unaligned_workspace_is_refused():
    p = spread(bwd_params)
    p.part += 4
    assert "aligned" in refusal(bwd_params, p)


def test_bias_tables():
    L = _lib.lib()
    E, edges, vec, n, H = A, A + FAR, A + 2 * FAR, 16, 4
    for bad in (dict(vec=E + 4), dict(vec=E - 4 * H * (2 * T - 1) + 4), dict(vec=edges + 60)):
        a = dict(E=E, edges=edges, vec=vec)
        a.update(bad)
        assert L.nrse_rel_bias_expand(a["E"], a["edges"], n, a["vec"], H, T, 0, None) < 0
        assert "share" in L.nrse_last_error().decode()
    for bad in (dict(E=vec + 4), dict(E=vec - 2 * n * H * 4 + 4), dict(E=edges)):
        a = dict(E=E, edges=edges, vec=vec)
        a.update(bad)
        assert L.nrse_rel_bias_collect(a["vec"], a["edges"], n, a["E"], H, T, 0, 0, None) < 0
        assert "share" in L.nrse_last_error().decode()


@pytest.mark.parametrize("fn", ["nrse_grad_norm", "nrse_clip_grad_norm"])
@pytest.mark.parametrize("norm,part", [(A + 16, A + FAR), (A + FAR, A - 8), (A + FAR, A + 4 * 100000 - 8), (A + FAR, A + FAR - 8)],
                         ids=["norm-in-a-tensor", "part-before", "part-behind", "norm-in-part"])
def test_gradient_norm_scratch_in_a_tensor(fn, norm, part):
    L = _lib.lib()
    a = ((ctypes.c_void_p * 2)(A + 2 * FAR, A), (ctypes.c_longlong * 2)(5, 100000), (ctypes.c_int * 2)(_lib.F32, _lib.F32), 2)
    limit = () if fn == "nrse_grad_norm" else (1.0,)
    assert getattr(L, fn)(*a, *limit, norm, part, None) < 0 and "overlap" in L.nrse_last_error().decode()


def test_launches_past_their_grid_are_refused_before_the_first():
    """The bias gradient's launch has a head per grid row and a workgroup per 64 entries: refused where it could not
    start, not after the other kernels have run."""
    p = spread(bwd_params)
    p.hq = p.hkv = 1 << 16
    p.rows, p.nseq = 100, 1
    for x in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        setattr(p, x + "_row", 64 << 16)
    assert "65535" in refusal(bwd_params, p)
    p = spread(bwd_params)
    p.bias_len = 1 << 29
    assert "bias_len" in refusal(bwd_params, p)
