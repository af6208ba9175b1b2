"""How close the packed backward comes, against bounds as close (tests/packed_bounds.py) and against its own roundings
(tests/packed_rounding.py); and the refusal of operands off their 16 bytes."""
import pytest
import torch

from packed_bounds import reference
from packed_rounding import case, error, gradients
from test_attn_packed_gpu import check, cu_of, data, run

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("lens", [[31, 33, 0, 64], [300, 5, 0, 0, 191, 65], [1400, 1]], ids=lambda x: "-".join(map(str, x)))
@pytest.mark.parametrize("heads", [(4, 2), (6, 1)], ids=str)
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("bias", [None, "plain", "gated"])
@pytest.mark.parametrize("dtype,D", [(BF16, 64), (BF16, 128), (F32, 64), (F32, 128)])
def test_close_bounds(nrse_device, dtype, D, bias, causal, heads, lens):
    from nrse_amd import kernels as K
    q, k, v, do, gate, vec = data(lens, *heads, D, dtype, bias, nrse_device, 51)
    cu = cu_of(lens, nrse_device)
    got = run(K, q, k, v, cu, do, causal=causal, gate=gate, vec=vec)
    check(got, reference(q, k, v, cu, causal=causal, gate=gate, vec=vec, dout=do))


@pytest.mark.parametrize("name,keys,values", [("dq", 1.0, 0.0), ("dk", 0.0, 1.0)])
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("D,hq,hkv", [(64, 4, 2), (128, 4, 1), (64, 16, 16)])
def test_rounded_once_less(nrse_device, D, hq, hkv, causal, name, keys, values):
    """dQ takes dS in two bf16 parts, and dK delta from f32 sums: the error over the norm is nearer to that form's than
    to the coarser one's, which is at least a tenth larger (over 1e5 elements either stays within 1 %)."""
    from nrse_amd import kernels as K
    lens = [500, 131]
    q, k, v, do = case(lens, hq, hkv, D, 52, keys, values, nrse_device)
    exact, fine, coarse = gradients(q, k, v, do, lens, causal)[name]
    fine, coarse = error(fine, exact), error(coarse, exact)
    assert coarse > 1.1 * fine
    got = run(K, q, k, v, cu_of(lens, nrse_device), do, causal=causal)
    assert error(got[name], exact) < (fine * coarse) ** 0.5, (error(got[name], exact), fine, coarse)


@pytest.mark.parametrize("dtype,off", [(BF16, 4), (BF16, 1), (F32, 2)])
def test_operands_off_their_16_bytes_are_refused(nrse_device, dtype, off):
    from nrse_amd import _lib, kernels as K
    wide = torch.zeros(4, 20, 4, 72, dtype=dtype, device=nrse_device)
    cu = cu_of([20], nrse_device)
    good = [wide[i, ..., :64] for i in range(4)]
    for i in range(4):
        x = list(good)
        x[i] = wide[i, ..., off:64 + off]
        with pytest.raises(_lib.NrseError, match="16-byte"):
            K.attn_packed_fwd(*x[:3], cu, x[3])
    odd = torch.zeros(20, 4, 64 + off, dtype=dtype, device=nrse_device)[..., :64]
    with pytest.raises(_lib.NrseError, match="16-byte"):
        K.attn_packed_fwd(odd, good[1], good[2], cu, good[3])
    K.attn_packed_fwd(*good[:3], cu, good[3])
