"""The bf16 group-norm net against the 64-bit form: logits within the bar of the BatchNorm net (2e-2 of the largest), gradients
within what rounding every stored tensor to bf16 makes of them.

The yardstick for a gradient is arithmetic of its own: the 64-bit net with every tensor that is stored between kernels (convolution
outputs, activations, their gradients, the weights' images) rounded to bf16 at random, up with the probability of the
remainder.  Such a rounding is off by at most twice as much as one to nearest and its mean square, u^2 r (1 - r) against
min(r, 1 - r)^2, is at least as large at every remainder r, so the root of its mean squared error bounds what nearest
rounding is expected to leave.  The 2-norm of a tensor's error is a sum over many independent roundings and stays near that root:
twice it is allowed, and six times for tensors of fewer than 64 elements, whose norm is a few draws (six sigma)."""
import pytest
import torch
import torch.nn.functional as F

from test_group_norm_net_gpu import ACT, dice, make, plain_forward

pytestmark = pytest.mark.gpu


def to_bf16(x, gen):
    """fp64 -> bf16 values in fp64, rounded up or down in proportion (8 bits of precision, relative steps of 2^-7 of the power of two)."""
    mantissa, exponent = torch.frexp(x)                       # |mantissa| in [0.5, 1): 256 steps to 1
    return torch.ldexp(torch.floor(mantissa * 256 + torch.rand(x.shape, generator=gen, dtype=x.dtype)) / 256, exponent)


class Stored(torch.autograd.Function):
    """A tensor that lies in memory as bf16, and its gradient."""

    @staticmethod
    def forward(ctx, x, gen, value):
        ctx.gen = gen
        return to_bf16(x, gen) if value else x.clone()

    @staticmethod
    def backward(ctx, g):
        return to_bf16(g, ctx.gen), None, None


class Weight(torch.autograd.Function):
    """A weight's image in bf16; its gradient is fp32."""

    @staticmethod
    def forward(ctx, w):
        return w.float().bfloat16().to(w.dtype)

    @staticmethod
    def backward(ctx, g):
        return g


def rounded_forward(sd, x, depth, groups, act, gen):
    def stored(v, value=True):
        return Stored.apply(v, gen, value)

    def double(prefix, x):
        for conv, norm in ((0, 1), (3, 4)):
            k = f"{prefix}.double_conv."
            y = stored(F.conv2d(x, Weight.apply(sd[f"{k}{conv}.weight"]), sd[f"{k}{conv}.bias"], padding=(1, 2)))
            x = stored(ACT[act](F.group_norm(y, groups, sd[f"{k}{norm}.weight"], sd[f"{k}{norm}.bias"], 1e-5)))
        return x

    skips = []
    for l in range(depth):
        x = double(f"encoders.{l}.conv", x)
        skips.append(x)
        x = stored(F.max_pool2d(x, (1, 2)), False)
    x = double("bottleneck", x)
    for i in range(depth):
        up = stored(F.conv_transpose2d(x, Weight.apply(sd[f"decoders.{i}.up.weight"]), sd[f"decoders.{i}.up.bias"], stride=(1, 2)))
        x = double(f"decoders.{i}.conv", stored(torch.cat([up, skips[depth - 1 - i]], 1), False))
    return F.conv2d(x, sd["outputs.weight"], sd["outputs.bias"])


@pytest.mark.parametrize("act", ["relu", "silu"])
def test_logits_and_gradients(gpu_device, act):
    depth, groups = 2, 8
    m, x, t = make(depth, 32, 5, 256, 4, groups, act, "bf16")
    sd = {k: v.detach().double().cpu().requires_grad_(True) for k, v in m.state_dict().items()}
    logits = plain_forward(sd, x.double(), depth, groups, act, (3, 5))
    dice(logits, t).backward()
    want = {k: v.grad.clone() for k, v in sd.items()}
    samples, squares = 8, {k: 0.0 for k in sd}
    for s in range(samples):
        gen = torch.Generator().manual_seed(s)
        for v in sd.values():
            v.grad = None
        dice(rounded_forward(sd, to_bf16(x.double(), gen), depth, groups, act, gen), t).backward()
        for k, v in sd.items():
            squares[k] += float((v.grad - want[k]).square().sum()) / samples
    m.train()
    got = m(x.cuda()).detach()
    print("\nlogits, of the largest:", float((got.double().cpu() - logits.detach()).abs().max()) / float(logits.detach().abs().max()))
    assert float((got.double().cpu() - logits.detach()).abs().max()) < 2e-2 * float(logits.detach().abs().max())
    m.dice_forward(got, t.cuda())
    m.backward()
    report = {}
    for k, w in want.items():
        err, bound = float((m.grad(k).double().cpu() - w).norm()), (2 if w.numel() >= 64 else 6) * squares[k] ** 0.5
        report[k] = (round(err / bound, 3), round(err / float(w.norm()), 4), round(bound / float(w.norm()), 4))
    print("\nerror / bound, error / gradient, bound / gradient:", report)
    assert all(r[0] <= 1 for r in report.values()), {k: r for k, r in report.items() if r[0] > 1}
    # what the bounds are worth: a part of the gradients of the convolutions' weights (ReLU: masks of values next to 0 change sides)
    assert all(r[2] < {"relu": 0.4, "silu": 0.1}[act] for k, r in report.items() if want[k].dim() == 4), report
