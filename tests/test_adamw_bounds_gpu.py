"""AdamW with fp32 moments over several steps, clipped and not, within bounds that scale with the values (derived, and shown to find
mistakes, in ``test_adamw_bounds_cpu.py``)."""
import pytest
import torch

from test_adamw_bounds_cpu import BETAS, DECAY, EPS, LR, U, Bounds, gradients, parameters

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("clip", [None, 0.5])
def test_moments_and_parameters(gpu_device, shift, clip):
    from dnanet_amd.optim import HipAdamW
    host = parameters()
    params = []
    for p in host:                                   # `shift` elements into their storage
        q = torch.zeros(p.numel() + shift, device="cuda")[shift:]
        q.copy_(p)
        q.grad = torch.zeros(p.numel() + shift, device="cuda")[shift:]
        params.append(q)
    opt, bounds = HipAdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, max_grad_norm=clip), Bounds(host)
    for t in range(1, 7):
        grads, coef, norm = gradients(t, clip)
        for p, g in zip(params, grads):
            p.grad.copy_(g)
        bounds.step(grads, coef)
        opt.step()
        if clip:
            assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
        parts = [[x[at:at + p.numel()].cpu() for p, at in zip(params, opt.offsets)] for x in (opt.exp_avg, opt.exp_avg_sq)]
        assert bounds.outside([p.cpu() for p in params], *parts) == set(), t
