"""The random bits that round 8-bit moments: 16 each of a hash of (tensor's number, element in the tensor, step, seed).

``number`` counts the optimizer's parameters through its groups, tensors without elements or gradients included.  Codes and scales are
compared bit by bit with the formulas in 64 bits (their own tolerance: none)."""
import pytest
import torch

from test_adamw_gpu import SIZES, U, step8, tensors

pytestmark = pytest.mark.gpu
NUMBER = 0xC2B2AE35          # the key moves on by this from one tensor to the next


def check(opt, params, grads_of, steps, seed, rates, left_out=()):
    """``steps`` steps of ``opt``; codes, scales and parameters of every tensor against the formula."""
    zero = lambda n: (torch.zeros(n, dtype=torch.float64), torch.zeros((n + 255) // 256, dtype=torch.float64))  # noqa: E731
    state = [(zero(p.numel()), zero(p.numel())) for p in params]
    ref = [p.double().cpu() for p in params]
    size = [torch.zeros(p.numel(), dtype=torch.float64) for p in params]
    for t in range(1, steps + 1):
        grads_of(t)
        opt.step()
        for k, p in enumerate(params):
            if k not in left_out:
                ref[k], state[k], step = step8(ref[k], p.grad.double().cpu(), state[k], t, k * NUMBER, seed, lr=rates[k])
                size[k] = size[k] + step.abs()
    for k, p in enumerate(params):
        n, at = p.numel(), opt.offsets[k]
        for (q, s), codes, scales in zip(state[k], (opt.exp_avg, opt.exp_avg_sq), (opt.exp_avg_scale, opt.exp_avg_sq_scale)):
            assert torch.equal(scales[at // 256:at // 256 + s.numel()].double().cpu(), s), k
            assert torch.equal(codes[at:at + n].float().double().cpu(), q), k
        tol = steps * 4 * U * (ref[k].abs() + 0.5) + 64 * U * size[k]
        assert bool(((p.double().cpu() - ref[k]).abs() <= tol).all()), k


def wide_gradients(params, gen):
    """Magnitudes over 2^30: the smallest second moments round to the lowest code; a tenth are zero."""
    for p in params:
        if p.grad is not None:
            p.grad.copy_(torch.randn(p.shape, generator=gen) * 10 ** (-4.5 * torch.rand(p.shape, generator=gen))
                         * (torch.rand(p.shape, generator=gen) > 0.1))


@pytest.mark.parametrize("shift", [0, 3])
def test_bits_of_every_tensor(gpu_device, shift):
    from dnanet_amd.optim import HipAdamW
    params, gen = tensors(SIZES, shift=shift, seed=4), torch.Generator().manual_seed(3)
    opt = HipAdamW(params, lr=1e-2, weight_decay=0.1, state_bits=8, seed=77)
    check(opt, params, lambda t: wide_gradients(params, gen), 5, 77, [1e-2] * len(params))


def test_bits_across_groups_launches_and_missing_gradients(gpu_device):
    """230 tensors: three launches; groups of their own rates: a call each; tensors without a gradient keep their number."""
    from dnanet_amd.optim import HipAdamW
    gen = torch.Generator().manual_seed(0)
    params = tensors([int(torch.randint(1, 900, (1,), generator=gen)) for _ in range(230)], seed=1)
    out = (0, 57, 130, 229)
    for k in out:
        params[k].grad = None
    opt = HipAdamW([{"params": params[:100], "lr": 1e-2}, {"params": params[100:], "lr": 3e-3}], weight_decay=0.1, state_bits=8, seed=(1 << 32) - 5)
    check(opt, params, lambda t: wide_gradients(params, gen), 3, (1 << 32) - 5, [1e-2] * 100 + [3e-3] * 130, out)


def test_bits_do_not_depend_on_the_sizes_before(gpu_device):
    """The second tensor's codes are the same behind a first one of any size."""
    from dnanet_amd.optim import HipAdamW
    codes = []
    for before in (1, 300, 70000):
        first, second = tensors([before, 5000], seed=2)
        torch.manual_seed(5)
        second.grad = torch.randn(5000, device="cuda")
        opt = HipAdamW([first, second], state_bits=8, seed=9)
        opt.step()
        at = opt.offsets[1]
        codes.append(torch.stack([x.view(torch.uint8)[at:at + 5000] for x in (opt.exp_avg, opt.exp_avg_sq)]).cpu())
    assert torch.equal(codes[0], codes[1]) and torch.equal(codes[0], codes[2])
