"""clip_grad_norm_ beside autograd: an in-place change that it can see."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_graph_that_saved_a_gradient_sees_the_clip(nrse_device):
    from nrse_amd.train import clip_grad_norm_
    p = torch.nn.Parameter(torch.ones(8, 6, device=nrse_device))
    p.grad = torch.full((8, 6), 3.0, device=nrse_device)
    q = torch.nn.Parameter(torch.ones(4, 5, device=nrse_device))
    q.grad = torch.ones(5, 4, device=nrse_device).t()      # dense in another order
    w = torch.ones(8, 6, device=nrse_device, requires_grad=True)
    y = (p.grad * w).sum()
    z = (q.grad * w[:4, :5]).sum()
    versions = p.grad._version, q.grad._version
    clip_grad_norm_([p, q], 1.0)
    assert (p.grad._version, q.grad._version) == (versions[0] + 1, versions[1] + 1)
    for x in (y, z):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            x.backward()
    with torch.inference_mode():
        q.grad = torch.ones(4, 5, device=nrse_device)
    clip_grad_norm_([p, q], 1e-3)                          # (an inference tensor has no version)
    assert float(q.grad.norm()) < 1e-3
