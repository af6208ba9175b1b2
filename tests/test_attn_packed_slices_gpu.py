"""Packed attention's backward where a short sequence stands beside long ones: its key blocks have fewer (head, query
tile) pairs than the batch has slices, and some slices have none."""
import pytest

import torch

from packed_reference import reference
from test_attn_packed_gpu import check, cu_of, data, run

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("bias", [None, "gated"])
@pytest.mark.parametrize("heads", [(1, 1), (2, 1)], ids=str)
@pytest.mark.parametrize("dtype,D", [(BF16, 128), (BF16, 64), (F32, 64)])
def test_slices_without_a_pair(nrse_device, dtype, D, heads, bias, causal):
    from nrse_amd import kernels as K
    lens = [1400, 1, 1400, 40]
    q, k, v, do, gate, vec = data(lens, *heads, D, dtype, bias, nrse_device, 31)
    cu = cu_of(lens, nrse_device)
    got = run(K, q, k, v, cu, do, causal=causal, gate=gate, vec=vec)
    check(got, reference(q, k, v, cu, causal=causal, gate=gate, vec=vec, dout=do))
