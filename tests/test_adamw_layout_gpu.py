"""AdamW steps on tensors that keep their address and become others: refused, or taken for what they are now."""
import pytest
import torch

from test_adamw_gpu import U, reference

pytestmark = pytest.mark.gpu


def optimizer(own, shape=(40, 40), bits=32):
    """A parameter after one step, its gradient and the optimizer; ``own``: the gradient in the group's own list."""
    from dnanet_amd.optim import HipAdamW
    torch.manual_seed(0)
    p, g = torch.randn(shape, device="cuda"), torch.randn(shape, device="cuda")
    if own:
        opt = HipAdamW([{"params": [p], "grads": [g]}], lr=1e-2, state_bits=bits)
    else:
        p.grad = g
        opt = HipAdamW([p], lr=1e-2, state_bits=bits)
    opt.step()
    return p, g, opt


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("own", [False, True])
def test_a_shorter_parameter_at_the_same_address_is_refused(gpu_device, own, bits):
    for change in (lambda t: setattr(t, "data", t.data[:7]), lambda t: t.resize_(7, 40), lambda t: t.set_(t.untyped_storage(), 0, (7, 40), (40, 1))):
        p, g, opt = optimizer(own, bits=bits)
        whole, address = p.data, p.data_ptr()
        change(p)
        assert p.data_ptr() == address
        keep, moments = torch.as_strided(whole, (1600,), (1,)).clone(), opt.exp_avg.clone()
        with pytest.raises(ValueError, match="new optimizer"):
            opt.step()
        assert torch.equal(torch.as_strided(whole, (1600,), (1,)), keep) and torch.equal(opt.exp_avg.view(torch.uint8), moments.view(torch.uint8))
        assert opt.step_count == 1


@pytest.mark.parametrize("own", [False, True])
def test_a_strided_parameter_or_gradient_is_refused(gpu_device, own):
    p, g, opt = optimizer(own)
    p.data = p.data.t()
    with pytest.raises(ValueError, match="contiguous"):
        opt.step()
    p, g, opt = optimizer(own)
    g.data = g.data.t()
    with pytest.raises(ValueError, match="contiguous"):
        opt.step()


def test_a_shorter_gradient_is_refused(gpu_device):
    p, g, opt = optimizer(True)
    g.data = g.data[:7]
    with pytest.raises(ValueError, match="of the parameter's shape"):
        opt.step()


def test_a_gradient_of_another_type_is_read_as_what_it_is(gpu_device):
    p, g, opt = optimizer(True)
    m, v = opt.exp_avg[:1600].double().cpu(), opt.exp_avg_sq[:1600].double().cpu()
    address = g.data_ptr()
    g.data = torch.as_strided(g.data.view(torch.bfloat16), (40, 40), (40, 1))
    g.copy_(torch.linspace(-1, 1, 1600).view(40, 40))
    assert g.data_ptr() == address and g.dtype == torch.bfloat16 and g.is_contiguous()
    before = p.double().cpu().flatten()
    opt.step()
    want, _, _, step = reference(before, g.double().cpu().flatten(), m, v, 2, decay=1e-2)
    assert bool(((p.double().cpu().flatten() - want).abs() <= 4 * U * (before.abs() + want.abs()) + 64 * U * step.abs()).all())


def test_gradients_that_change_places(gpu_device):
    """One memory as the gradient of first one parameter, then the other: the one without a gradient stays as it is."""
    from dnanet_amd.optim import HipAdamW
    p, q, g = torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda"), torch.ones(300, device="cuda")
    opt = HipAdamW([p, q], lr=1e-2, weight_decay=0.0)
    p.grad = g
    opt.step()
    assert bool(p.any()) and not q.any()
    p.grad, q.grad, keep = None, g, p.clone()
    opt.step()
    assert torch.equal(p, keep) and bool(q.any())
