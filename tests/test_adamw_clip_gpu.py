"""AdamW's ``max_grad_norm`` set, changed and taken back after construction: every step as by an optimizer that was made with it."""
import pytest
import torch

from test_adamw_gpu import tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_clipping_follows_the_attribute(gpu_device, bits):
    from dnanet_amd.optim import HipAdamW
    for values in ((None, 0.01, 0.5, None, 0.02), (0.01, None, 0.01)):
        a, b = tensors(seed=3), tensors(seed=3)
        opt = HipAdamW(a, lr=1e-2, state_bits=bits, seed=4, max_grad_norm=values[0])
        state = None
        for value in values:
            opt.max_grad_norm = value
            opt.step()
            other = HipAdamW(b, lr=1e-2, state_bits=bits, seed=4, max_grad_norm=value)
            if state is not None:
                other.load_state_dict(state)
            other.step()
            state = other.state_dict()
            assert all(torch.equal(p, q) for p, q in zip(a, b)), value
            assert torch.equal(opt.exp_avg_sq.view(torch.uint8), other.exp_avg_sq.view(torch.uint8)), value
            assert (opt.grad_norm is None) == (value is None) and (value is None or torch.equal(opt.grad_norm, other.grad_norm))
        for bad in (0.0, -1.0, float("nan")):
            with pytest.raises(ValueError, match="above zero"):
                opt.max_grad_norm = bad
        assert opt.max_grad_norm == values[-1]


def test_a_captured_step_no_longer_matches(gpu_device):
    """A graph holds the norm it was captured with: another one asks for a new capture."""
    from dnanet_amd.optim import HipAdamW
    from dnanet_amd.unet import GraphedTrainStep
    from test_group_norm_net_gpu import make
    m, x, t = make(2, 16, 5, 128, 2, 4, "relu", "fp32")
    opt = HipAdamW(m, lr=1e-3)
    step = GraphedTrainStep(m, opt, x.cuda(), t.cuda())
    assert step.matches(x)
    opt.max_grad_norm = 1e-3
    assert not step.matches(x)
    step = GraphedTrainStep(m, opt, x.cuda(), t.cuda())
    step(x.cuda(), t.cuda())
    torch.cuda.synchronize()
    assert float(opt.grad_norm) > 0 and step.matches(x)
