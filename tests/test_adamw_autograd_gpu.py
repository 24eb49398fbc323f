"""AdamW's in-place writes as autograd sees them: of the parameters that a step updates, and of no other."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_parameter_without_a_gradient_is_not_written(gpu_device):
    from dnanet_amd.optim import HipAdamW
    p, q = (torch.randn(50, device="cuda", requires_grad=True) for _ in range(2))
    opt = HipAdamW([p, q], lr=1e-2)
    p.grad = torch.ones_like(p)
    first, second, versions = (p * p).sum(), (q * q).sum(), (p._version, q._version)
    for _ in range(2):
        opt.step()
    assert p._version > versions[0] and q._version == versions[1]
    second.backward()
    assert torch.equal(q.grad, 2 * q.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        first.backward()
    opt.step()
    assert q._version > versions[1]
