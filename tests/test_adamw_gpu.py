"""AdamW over many tensors, fp32 and 8-bit moments, gradient clipping: against the formulas in 64 bits.

Tolerances count roundings, u = 2^-24: a moment is one product and one fma away from its inputs, a step adds that error again;
the quotient of a step is within 16 u of itself (sqrt, division, three products).  8-bit codes are compared bit by bit: the kernel
forms new moments in fp64, so that a code differs only where two fp64 results round to different fp32 values (2^-29)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SIZES = [1, 3, 4, 255, 256, 257, 1000, 4095, 4096, 4097, 20000, 7, 0, 64]


def tensors(sizes=SIZES, dtype=torch.float32, gdtype=None, seed=0, shift=0):
    """Parameters with gradients; ``shift``: start this many elements into their storage (unaligned)."""
    gen = torch.Generator().manual_seed(seed)
    out = []
    for n in sizes:
        p, g = 0.1 * torch.randn(n + shift, generator=gen), torch.randn(n + shift, generator=gen) * 10 ** (4 * torch.rand(1, generator=gen) - 5)
        p, g = p.to(dtype).cuda()[shift:], g.to(gdtype or dtype).cuda()[shift:]
        if g.dtype == p.dtype:
            p.grad = g
        out.append(p if g.dtype == p.dtype else (p, g))
    return out


def reference(p, g, m, v, t, lr=1e-2, betas=(0.9, 0.999), eps=1e-8, decay=0.1, coef=1.0):
    g = g * coef
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    step = lr * (m / (1 - betas[0] ** t)) / ((v / (1 - betas[1] ** t)).sqrt() + eps)
    return p * (1 - lr * decay) - step, m, v, step


def moments(opt, k):
    n, at = opt._params[k].numel(), opt.offsets[k]
    out = []
    for x, s in ((opt.exp_avg, opt.exp_avg_scale), (opt.exp_avg_sq, opt.exp_avg_sq_scale)):
        x = x[at:at + n].float().cpu().double()
        if s is not None:
            x = x * s[at // 256:at // 256 + (n + 255) // 256].cpu().double().repeat_interleave(256)[:n]
        out.append(x)
    return out


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("clip", [None, 0.5])
def test_fp32_states(gpu_device, shift, clip):
    from dnanet_amd.optim import HipAdamW
    params = tensors(shift=shift)
    opt = HipAdamW(params, lr=1e-2, weight_decay=0.1, max_grad_norm=clip)
    ref = [(p.double().cpu(), torch.zeros(p.numel(), dtype=torch.float64), torch.zeros(p.numel(), dtype=torch.float64)) for p in params]
    steps = 6
    gen = torch.Generator().manual_seed(9)
    for t in range(1, steps + 1):
        for p in params:
            p.grad.copy_(torch.randn(p.shape, generator=gen) * 0.3)
        grads = [p.grad.double().cpu() for p in params]
        coef = 1.0
        if clip:
            norm = math.sqrt(sum(float((g * g).sum()) for g in grads))
            coef = min(1.0, clip / (norm + 1e-6))
        opt.step()
        if clip:
            assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
        ref = [reference(p, g, m, v, t, coef=coef)[:3] for (p, m, v), g in zip(ref, grads)]
    for k, (p, (rp, rm, rv)) in enumerate(zip(params, ref)):
        m, v = moments(opt, k)
        big = 2.0
        assert bool(((m - rm).abs() <= steps * 4 * U * big).all()) and bool(((v - rv).abs() <= steps * 4 * U * big ** 2).all())
        # a step is at most lr * (1 - beta1) / sqrt(1 - beta2) times a few; its relative error: 16 u and what its moments carry
        tol = steps * (4 * U * rp.abs() + 1e-2 * 4 * (64 * U + steps * 8 * U * big / (rv.sqrt() + 1e-8)))
        assert bool(((p.double().cpu() - rp).abs() <= tol).all())


@pytest.mark.parametrize("pdtype,gdtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("bits", [32, 8])
def test_types(gpu_device, pdtype, gdtype, bits):
    """One step: a bf16 parameter is rounded once, to nearest."""
    from dnanet_amd.optim import HipAdamW
    params = tensors(dtype=pdtype, gdtype=gdtype)
    if pdtype != gdtype:                     # gradients of another type: a list of their own
        params, grads = zip(*params)
        opt = HipAdamW([{"params": params, "grads": grads}], lr=1e-2, weight_decay=0.1, state_bits=bits)
    else:
        grads = [p.grad for p in params]
        opt = HipAdamW(params, lr=1e-2, weight_decay=0.1, state_bits=bits)
    before = [p.double().cpu() for p in params]
    opt.step()
    for p, g, b in zip(params, grads, before):
        want, _, _, step = reference(b, g.double().cpu(), 0.0, 0.0, 1)
        tol = (2.0 ** -8 if pdtype == torch.bfloat16 else 0.0) * want.abs() + 4 * U * (b.abs() + want.abs()) + 64 * U * step.abs()
        assert bool(((p.double().cpu() - want).abs() <= tol).all())


def hash32(x):
    x = x & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def quantise(x, bits, floor):
    """(values over the scale, scales) of a tensor's moments ``x`` (fp64): e4m3 steps, rounded up where the 16 bits reach."""
    n = x.numel()
    y = torch.nn.functional.pad(x.float().abs(), (0, -n % 256)).view(-1, 256)
    top = torch.where(y.isfinite(), y, torch.zeros_like(y)).amax(1).double()
    k = torch.ceil(torch.log2(top.clamp(min=1e-300) / 448)).clamp(min=-126)
    scale = torch.where(top > 0, 2.0 ** k, torch.zeros_like(top))
    r = (y.double() * 2.0 ** -k[:, None]).flatten()[:n]
    r = torch.where(r < 2.0 ** -6, (r.float() + 2.0 ** -6).double() - 2.0 ** -6, r)          # the kernel's fp32 sum below 2^-6
    e = torch.floor(torch.log2(r.clamp(min=2.0 ** -6)))
    unit = 2.0 ** (e - 3)
    q = (torch.floor(r / unit + bits.double() / 65536) * unit).clamp(max=448)
    if floor:
        q = torch.where(x.float() > 0, q.clamp(min=2.0 ** -9), q)
    q = torch.where(x < 0, -q, q)
    return torch.where(x.float().isfinite(), q, torch.full_like(q, float("nan"))), scale


def step8(p, g, state, t, at, seed, lr=1e-2, betas=(0.9, 0.999), eps=1e-8, decay=0.1, coef=1.0):
    (qm, sm), (qv, sv) = state
    n = p.numel()
    old_m, old_v = qm * sm.repeat_interleave(256)[:n], qv * sv.repeat_interleave(256)[:n]
    new, m, v, step = reference(p, g, old_m, old_v, t, lr, betas, eps, decay, coef)
    bits = hash32(torch.arange(at, at + n) + t * 0x9E3779B9 + seed * 0x85EBCA6B)
    return new, (quantise(m, bits & 0xFFFF, False), quantise(v, bits >> 16, True)), step


@pytest.mark.parametrize("shift", [0, 3])
def test_8_bit_states(gpu_device, shift):
    """Codes and scales bit by bit over several steps, parameters against the formula on the unrounded moments."""
    from dnanet_amd.optim import HipAdamW
    params = tensors(shift=shift, seed=4)
    opt = HipAdamW(params, lr=1e-2, weight_decay=0.1, state_bits=8, seed=77)
    zero = lambda n: (torch.zeros(n, dtype=torch.float64), torch.zeros((n + 255) // 256, dtype=torch.float64))  # noqa: E731
    state = [(zero(p.numel()), zero(p.numel())) for p in params]
    ref = [p.double().cpu() for p in params]
    gen = torch.Generator().manual_seed(3)
    steps = 5
    size = [0.0] * len(params)
    for t in range(1, steps + 1):
        for p in params:
            # magnitudes over 2^30: the smallest second moments round to the lowest code
            p.grad.copy_(torch.randn(p.shape, generator=gen) * 10 ** (-4.5 * torch.rand(p.shape, generator=gen)) * (torch.rand(p.shape, generator=gen) > 0.1))
        opt.step()
        for k, p in enumerate(params):
            ref[k], state[k], step = step8(ref[k], p.grad.double().cpu(), state[k], t, opt.offsets[k], 77)
            size[k] = size[k] + step.abs()
    for k, p in enumerate(params):
        n, at = p.numel(), opt.offsets[k]
        for (q, s), codes, scales in zip(state[k], (opt.exp_avg, opt.exp_avg_sq), (opt.exp_avg_scale, opt.exp_avg_sq_scale)):
            assert torch.equal(scales[at // 256:at // 256 + s.numel()].double().cpu(), s)
            assert torch.equal(codes[at:at + n].float().double().cpu(), q)
        tol = steps * 4 * U * (ref[k].abs() + 0.5) + 64 * U * size[k]
        assert bool(((p.double().cpu() - ref[k]).abs() <= tol).all())
    tail = opt.exp_avg.view(torch.uint8)
    for k, p in enumerate(params):
        n, at = p.numel(), opt.offsets[k]
        assert not bool(tail[at + n:at + (n + 255) // 256 * 256].any()), "places past a tensor's end stay zero"


def test_8_bit_rounding_is_unbiased_and_follows(gpu_device):
    """Gradients of half of the elements drop to a tenth: their second moments follow (to nearest they would stand still).
    The mean over 4096 elements of a quantity with deviation below 0.5 is within 0.5 / 64 * 6 of its expectation."""
    from dnanet_amd.optim import HipAdamW
    n = 8192
    p = torch.zeros(n).cuda()
    p.grad = torch.ones(n).cuda()
    opt = HipAdamW([p], lr=0.0, weight_decay=0.0, state_bits=8, betas=(0.9, 0.99))
    for _ in range(500):
        opt.step()
    p.grad[::2] = 0.1
    for _ in range(500):
        opt.step()
    _, v = moments(opt, 0)
    want = 0.01 * (1 - 0.99 ** 500) + 1.0 * 0.99 ** 500 * (1 - 0.99 ** 500)
    assert abs(float(v[::2].mean()) / want - 1) < 0.05 + 0.02
    assert abs(float(v[1::2].mean()) / (1 - 0.99 ** 1000) - 1) < 0.05


def test_non_finite_gradient_keeps_to_its_element(gpu_device):
    from dnanet_amd.optim import HipAdamW
    for bits in (32, 8):
        for value in (float("nan"), float("inf")):
            out = []
            for spoil in (False, True):
                params = tensors([700, 300], seed=2)
                params[0].grad[0], params[0].grad[300] = 1.0, 0.0
                opt = HipAdamW(params, lr=1e-2, state_bits=bits)
                opt.step()
                if spoil:
                    params[0].grad[300] = value
                opt.step()
                params[0].grad[300] = 0.0
                opt.step()
                out.append((torch.cat([p.cpu() for p in params]), moments(opt, 0)))
            (clean, mc), (dirty, md) = out
            assert bool(dirty[300].isnan()), "as in fp32: a NaN / infinite moment spoils its own element"
            keep = torch.arange(1000) != 300
            assert torch.equal(clean[keep], dirty[keep])
            assert torch.equal(mc[0][keep[:700]], md[0][keep[:700]]) and torch.equal(mc[1][keep[:700]], md[1][keep[:700]])


def test_zero_gradients_move_nothing(gpu_device):
    from dnanet_amd.optim import HipAdamW
    for bits in (32, 8):
        p = torch.randn(1000).cuda()
        keep = p.clone()
        p.grad = torch.zeros_like(p)
        opt = HipAdamW([p], weight_decay=0.0, state_bits=bits, max_grad_norm=1.0)
        for _ in range(3):
            opt.step()
        assert torch.equal(p, keep) and float(opt.grad_norm) == 0.0
        assert not opt.exp_avg.view(torch.uint8).any() and not opt.exp_avg_sq.view(torch.uint8).any()


def test_clip_of_extreme_gradients(gpu_device):
    """Squares past fp32 are squares in fp64; a non-finite norm makes the step NaN, as torch's clip_grad_norm_ does."""
    from dnanet_amd.optim import HipAdamW
    p = torch.zeros(5000).cuda()
    p.grad = torch.full_like(p, 1e30)
    opt = HipAdamW([p], max_grad_norm=1.0)
    opt.step()
    want = 1e30 * math.sqrt(5000)
    assert abs(float(opt.grad_norm) - want) < 4 * U * want and bool(p.isfinite().all()) and float(p.abs().max()) > 0
    p.grad[17] = float("nan")
    opt.step()
    assert math.isnan(float(opt.grad_norm)) and bool(p.isnan().all())


def test_many_tensors_and_groups(gpu_device):
    """More tensors than a launch takes, groups of their own rates, tensors without gradients: as one optimizer per tensor."""
    from dnanet_amd.optim import HipAdamW
    gen = torch.Generator().manual_seed(0)
    sizes = [int(torch.randint(1, 3000, (1,), generator=gen)) for _ in range(230)]
    for clip in (None, 1e-3):
        together, alone = tensors(sizes), tensors(sizes)
        for k in (0, 50, 229):
            together[k].grad = None
        groups = [{"params": together[:100], "lr": 1e-2, "weight_decay": 0.0}, {"params": together[100:], "lr": 3e-3, "betas": (0.8, 0.95)}]
        opt = HipAdamW(groups, lr=5e-3, weight_decay=0.1, max_grad_norm=clip)
        opt.step()
        opt.step()
        coef = 1.0
        if clip:
            norm = math.sqrt(sum(float(p.grad.double().square().sum()) for k, p in enumerate(alone) if k not in (0, 50, 229)))
            assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
            coef = float(opt._clip[1])
        for k, (a, b) in enumerate(zip(together, alone)):
            if k not in (0, 50, 229):
                b.grad.mul_(coef)
                one = HipAdamW([b], lr=1e-2 if k < 100 else 3e-3, weight_decay=0.0 if k < 100 else 0.1, betas=(0.9, 0.999) if k < 100 else (0.8, 0.95))
                one.step()
                one.step()
            assert torch.equal(a, b), k


def test_gradients_that_come_and_go(gpu_device):
    """New gradient tensors every step (autograd's), dropped ones, a decay that changes: the table follows."""
    from dnanet_amd.optim import HipAdamW
    torch.manual_seed(0)
    w = torch.randn(64, 32, device="cuda", requires_grad=True)
    b = torch.zeros(64, device="cuda", requires_grad=True)
    opt = HipAdamW([w, b], lr=1e-2, weight_decay=0.1)
    mine = [w.detach().double().cpu().clone().requires_grad_(True), b.detach().double().cpu().clone().requires_grad_(True)]
    ref = torch.optim.AdamW(mine, lr=1e-2, weight_decay=0.1)
    x = torch.randn(16, 32, device="cuda")
    for t in range(4):
        if t == 2:
            opt.param_groups[0]["weight_decay"] = ref.param_groups[0]["weight_decay"] = 0.3
        ((x @ w.t() + b) ** 2).mean().backward()
        for p, q in zip((w, b), mine):
            q.grad = p.grad.double().cpu()
        opt.step()
        ref.step()
        opt.zero_grad()
        assert w.grad is None
    for p, q in zip((w, b), mine):
        assert bool(((p.double().cpu() - q).abs() <= 4 * (8 * U * (q.abs() + 0.1) + 4e-2 * 64 * U)).all())
    saved = (w * 2).sum()
    y = (w * w).sum()
    w.grad = torch.ones_like(w)
    opt.step()
    saved.backward()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()                              # autograd knows that the step wrote w


def test_captured_step(gpu_device):
    """A step captured with its learning rate and number on the device, replayed with eager steps in between."""
    from dnanet_amd.optim import HipAdamW
    for bits in (32, 8):
        a, b = tensors(seed=6), tensors(seed=6)
        oa, ob = (HipAdamW(x, lr=1e-2, state_bits=bits, max_grad_norm=0.1, seed=5) for x in (a, b))
        hyper, step = torch.zeros(4).cuda(), torch.zeros(1, dtype=torch.int64).cuda()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            oa.step(device_state=(hyper, step))
        oa.step_count = 0
        for t, lr in enumerate([1e-2, 1e-2, 3e-3, 1e-3]):
            for p, q in zip(a, b):
                p.grad.mul_(0.7)
                q.grad.mul_(0.7)
            hyper[0] = lr
            ob.param_groups[0]["lr"] = lr
            graph.replay()
            ob.step()
            torch.cuda.synchronize()
            for p, q in zip(a, b):
                # the device forms lr / (1 - beta^t) from the fp32 learning rate, the host from its own: 2^-24 of a step
                assert bool(((p - q).abs() <= (t + 1) * (4 * U * (q.abs() + 0.1) + 4e-2 * 16 * U)).all())
            assert torch.equal(oa.exp_avg.view(torch.uint8), ob.exp_avg.view(torch.uint8))
            assert torch.equal(oa.exp_avg_sq.view(torch.uint8), ob.exp_avg_sq.view(torch.uint8))
            assert torch.equal(oa.grad_norm, ob.grad_norm) and int(step) == t + 1
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="device_state"):
        with torch.cuda.graph(graph):
            oa.step()
    groups = HipAdamW([{"params": tensors([5]), "lr": 1.0}, {"params": tensors([5]), "lr": 2.0}])
    with pytest.raises(ValueError, match="one learning rate"):
        groups.step(device_state=(hyper, step))


def test_other_stream_and_repeatability(gpu_device):
    from dnanet_amd.optim import HipAdamW
    results = []
    for stream in (None, torch.cuda.Stream()):
        params = tensors(seed=8)
        opt = HipAdamW(params, state_bits=8, max_grad_norm=1.0, seed=1)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for _ in range(3):
                opt.step()
        torch.cuda.synchronize()
        results.append([p.cpu() for p in params] + [opt.exp_avg_sq.view(torch.uint8).cpu(), opt.grad_norm.cpu()])
    assert all(torch.equal(x, y) for x, y in zip(*results))


def test_state_dict(gpu_device):
    from dnanet_amd.optim import HipAdamW
    for bits in (32, 8):
        a = tensors(seed=3)
        oa = HipAdamW(a, lr=1e-2, state_bits=bits, seed=9)
        oa.step()
        b = [p.clone() for p in a]
        for p, q in zip(a, b):
            q.grad = p.grad
        ob = HipAdamW(b, lr=5.0, state_bits=bits)
        ob.load_state_dict(oa.state_dict())
        oa.step()
        ob.step()
        assert all(torch.equal(p, q) for p, q in zip(a, b)) and torch.equal(oa.exp_avg.view(torch.uint8), ob.exp_avg.view(torch.uint8))
    with pytest.raises(ValueError, match="state_bits"):
        HipAdamW(b).load_state_dict(oa.state_dict())


def test_elements_past_32_bits(gpu_device):
    """2^31 + 777 elements: the last ones are updated as they are alone, with the rounding bits of their place."""
    from dnanet_amd.optim import HipAdamW
    n = (1 << 31) + 777
    p = torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda")
    p.grad = torch.full((n,), 0.25, dtype=torch.bfloat16, device="cuda")
    p.grad[-777:] = torch.linspace(-1, 1, 777)
    opt = HipAdamW([p], lr=1e-2, weight_decay=0.1, state_bits=8, seed=3)
    opt.step()
    new, ((qm, sm), (qv, sv)), _ = step8(torch.full((777,), 0.5, dtype=torch.float64), p.grad[-777:].double().cpu(),
                                         ((torch.zeros(777).double(), torch.zeros(4).double()),) * 2, 1, 1 << 31, 3)
    assert torch.equal(opt.exp_avg[1 << 31:][:777].float().double().cpu(), qm) and torch.equal(opt.exp_avg_sq_scale[-4:].double().cpu(), sv)
    assert torch.equal(opt.exp_avg_sq[1 << 31:][:777].float().double().cpu(), qv)
    assert bool(((p[-777:].double().cpu() - new).abs() <= 2.0 ** -8 * new.abs() + 1e-8).all())


def test_refusals(gpu_device):
    from dnanet_amd.optim import HipAdamW
    p = torch.zeros(8, 8).cuda()
    for bad in ([p.t()[1:]], [p.double()], [p.cpu()], [p, p], [p, p[2:4]], [], ["x"]):
        with pytest.raises(ValueError):
            HipAdamW(bad)
    for kw in ({"state_bits": 16}, {"max_grad_norm": 0.0}, {"max_grad_norm": float("nan")}, {"betas": (1.0, 0.9)}, {"eps": -1.0}, {"lr": -1.0},
               {"weight_decay": -0.1}, {"seed": -1}, {"seed": 1 << 32}):
        with pytest.raises(ValueError):
            HipAdamW([p], **kw)
    with pytest.raises(ValueError, match="gradients for"):
        HipAdamW([{"params": [p], "grads": []}])
    with pytest.raises(ValueError, match="unknown"):
        HipAdamW([{"params": [p], "amsgrad": True}])
    opt = HipAdamW([p])
    p.grad = torch.zeros(8, 8).cuda().t()
    with pytest.raises(ValueError, match="contiguous"):
        opt.step()
    p.grad = torch.zeros(1, 8).cuda().expand(8, 8)
    with pytest.raises(ValueError, match="contiguous"):
        opt.step()
    assert opt.step_count == 0


def test_8_bit_signed_zeros_and_denormals(gpu_device):
    """Gradients of both zeros, fp32 denormals and magnitudes whose moments round to zero: codes and scales bit by bit, no code of
    a negative zero from a zero."""
    from dnanet_amd.optim import HipAdamW
    gen = torch.Generator().manual_seed(12)
    n = 2048 + 100
    p = torch.randn(n, generator=gen).cuda()
    opt = HipAdamW([p], state_bits=8, seed=3)
    p.grad = torch.empty(n).cuda()
    state = [(torch.zeros(n, dtype=torch.float64), torch.zeros((n + 255) // 256, dtype=torch.float64)) for _ in range(2)]
    size = torch.tensor([0.0, -0.0, 1e-42, -1e-42, 1e-30, -1e-30, 1.0, -1.0, 1e-3, -1e-4])
    for t in range(1, 4):
        g = size[torch.randint(len(size), (n,), generator=gen)]
        g[:256], g[256:512], g[512:768] = g[:256].sign() * 1e-40, -0.0, g[512:768].sign() * 1e-36
        p.grad.copy_(g)
        opt.step()
        _, state, _ = step8(torch.zeros(n, dtype=torch.float64), p.grad.double().cpu(), state, t, 0, 3)
        for (q, s), codes, scales in zip(state, (opt.exp_avg, opt.exp_avg_sq), (opt.exp_avg_scale, opt.exp_avg_sq_scale)):
            assert torch.equal(scales.double().cpu(), s) and torch.equal(codes[:n].float().double().cpu(), q)
    assert not opt.exp_avg.view(torch.uint8)[256:512].any() and not opt.exp_avg_sq.view(torch.uint8)[256:512].any()


@pytest.mark.parametrize("bits", [32, 8])
def test_denormal_second_moments_without_eps(gpu_device, bits):
    """eps = 0 and gradients of 1e-18: the second moment, 1e-39 and up, is an fp32 denormal.  The first step is lr * sign(g), off by
    half of v's error, two roundings to 2^-150 of at least 1e-39, and 16 roundings of the quotient."""
    from dnanet_amd.optim import HipAdamW
    gen = torch.Generator().manual_seed(5)
    p = torch.zeros(3000).cuda()
    sign = torch.where(torch.rand(3000, generator=gen) < 0.5, 1.0, -1.0)
    p.grad = (sign * (1e-18 * (1 + torch.rand(3000, generator=gen)))).cuda()
    opt = HipAdamW([p], lr=1e-2, eps=0.0, weight_decay=0.0, state_bits=bits)
    opt.step()
    want = -float(torch.tensor(1e-2)) * sign.double()
    assert bool(((p.double().cpu() - want).abs() <= 1e-2 * (2.0 ** -150 / 1e-39 + 16 * U)).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_unaligned_bf16_with_clipping(gpu_device, bits):
    """bf16 parameters and gradients that start at an odd element: as the same values in tensors of their own."""
    from dnanet_amd.optim import HipAdamW
    out = []
    for shift in (0, 1):
        gen = torch.Generator().manual_seed(8)
        params = []
        for n in (1, 5, 300, 5000):
            p = torch.zeros(n + shift, dtype=torch.bfloat16).cuda()[shift:]
            g = torch.zeros(n + shift, dtype=torch.bfloat16).cuda()[shift:]
            p.copy_(torch.randn(n, generator=gen))
            g.copy_(torch.randn(n, generator=gen))
            p.grad = g
            params.append(p)
        opt = HipAdamW(params, lr=1e-2, state_bits=bits, max_grad_norm=0.5)
        for _ in range(3):
            opt.step()
        # the norm's partial sums are the same numbers added in another order: fp64, then one rounding to fp32 of norm and coefficient
        out.append((float(opt.grad_norm), torch.cat(params).float().cpu()))
    assert abs(out[0][0] - out[1][0]) <= 2 * U * out[0][0]
    # three steps of 1e-2 from gradients that differ by 2^-23: a parameter rounds to the same bf16 value or to its neighbour
    assert bool(((out[0][1] - out[1][1]).abs() <= 3 * 2.0 ** -8 * out[0][1].abs() + 3e-2 * 2.0 ** -8).all())


def test_a_parameter_that_changes_its_size_is_refused(gpu_device):
    from dnanet_amd.optim import HipAdamW
    p = torch.randn(300).cuda()
    p.grad = torch.randn(300).cuda()
    opt = HipAdamW([p])
    opt.step()
    p.grad = None
    p.data = torch.randn(70000).cuda()
    p.grad = torch.randn(70000).cuda()
    with pytest.raises(ValueError, match="new optimizer"):
        opt.step()
