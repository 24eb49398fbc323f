"""Group norm + activation on plane-record tensors against the definition in 64 bits.

Tolerances count roundings, u = 2^-24 (fp32) and 2^-8 (half a step of bf16).  A sum passes through at most 17 fp32 additions per
summand before it is joined in fp64, each value through a few more operations: 64 u on the sum of the magnitudes that enter."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {"fp32": 0.0, "bf16": 2.0 ** -8}
EPS = 1e-5

# n, c, groups, h, w: one group per channel / one in all, groups inside records, across pieces, over whole planes, padded last
# planes, one pixel, odd widths, planes of several segments, groups over several planes of several segments, a last set of planes
# shorter than the others, more segments than one cluster of blocks takes
SHAPES = [(1, 8, 1, 1, 1), (2, 8, 8, 1, 1), (1, 8, 2, 1, 3), (3, 24, 8, 5, 37), (2, 40, 5, 3, 64), (2, 48, 16, 6, 33), (1, 32, 8, 5, 1024),
          (2, 32, 32, 2, 129), (1, 64, 1, 5, 520), (2, 72, 9, 1, 250), (1, 512, 8, 5, 16), (17, 16, 4, 6, 96), (1, 20, 4, 2, 4099),
          (3, 96, 3, 5, 700), (1, 60, 5, 4, 1500), (2, 60, 5, 1, 40), (1, 16, 2, 7, 20001), (2, 1024, 1, 5, 32), (3, 512, 2, 6, 256)]
ACTS = {"none": lambda z: z, "relu": torch.relu, "silu": F.silu}


def make(shape, dtype, seed=0, offset=0.5, dev="cuda"):
    from dnanet_amd.hip import BF16, F32, PlaneBuffer
    n, c, groups, h, w = shape
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, c, h, w, generator=g) * torch.exp(torch.randn(c, 1, 1, generator=g)) + offset * torch.randn(c, 1, 1, generator=g)
    x += 20 * (torch.rand(n, 1, h, w, generator=g) < 0.02)
    if dtype == "bf16":
        x = x.bfloat16().float()
    gamma, beta = 1 + 0.3 * torch.randn(c, generator=g), 0.3 * torch.randn(c, generator=g)
    buf = PlaneBuffer.from_nchw(x.to(dev), BF16 if dtype == "bf16" else F32)
    return buf, x.double(), gamma, beta


def definition(x, gamma, beta, groups, act, eps=EPS):
    n, c = x.shape[:2]
    xg = x.reshape(n, groups, -1)
    mean, var = xg.mean(-1), xg.var(-1, unbiased=False)
    rstd = (var + eps) ** -0.5
    scale = gamma.double() * rstd.repeat_interleave(c // groups, 1)
    shift = beta.double() - mean.repeat_interleave(c // groups, 1) * scale
    z = x * scale[..., None, None] + shift[..., None, None]
    return ACTS[act](z), mean, rstd, scale, shift


def close(got, want, tol, what):
    err = (got.double().cpu() - want).abs()
    bad = err > tol
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(err.max()):.3e}"


@pytest.mark.parametrize("act", ["relu", "silu", "none"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(gpu_device, shape, dtype, act):
    from dnanet_amd import hip
    from dnanet_amd.group_norm import group_norm_act
    buf, x, gamma, beta = make(shape, dtype)
    n, c, groups, h, w = shape
    out, stats = group_norm_act(buf.ref(c), gamma.cuda(), beta.cuda(), groups, EPS, act)
    a, mean, rstd, scale, shift = definition(x, gamma, beta, groups, act)
    xmax = float(x.abs().max())
    close(stats.mean, mean, 32 * U * xmax, "mean")
    # the variance around a mean that is off by d is off by d^2
    close(stats.rstd, rstd, rstd * (64 * U + (32 * U * xmax * rstd) ** 2), "rstd")
    tol = 64 * U * (float((gamma.abs() * 1.0).max()) * rstd.max() * xmax + beta.abs().max())
    close(stats.scale[:, :c], scale, tol, "scale")
    close(stats.shift[:, :c], shift, tol, "shift")
    assert not stats.scale[:, c:].any() and not stats.shift[:, c:].any()
    close(out.to_nchw(c), a, tol * 1.1 + HALF[dtype] * a.abs(), "output")
    full = out.to_nchw(hip.planes(c, buf.dtype) * hip.epr(buf.dtype))
    assert not full[:, c:].any(), "record slots past the channels are zero"


def backward_definition(g, x, gamma, mean, rstd, scale, shift, groups, act):
    n, c, h, w = x.shape
    per = c // groups
    z = x * scale[..., None, None] + shift[..., None, None]
    s = torch.sigmoid(z)
    slope = {"none": torch.ones_like(z), "relu": (z > 0).double(), "silu": s * (1 + z * (1 - s))}[act]
    dz = g * slope
    rs = rstd.repeat_interleave(per, 1)[..., None, None]
    xh = (x - mean.repeat_interleave(per, 1)[..., None, None]) * rs
    t = dz * gamma.double().view(1, c, 1, 1)

    def mean_g(v):
        return v.reshape(n, groups, -1).mean(-1).repeat_interleave(per, 1)[..., None, None]

    dx = rs * (t - mean_g(t) - xh * mean_g(t * xh))
    size = rs * (t.abs() + mean_g(t.abs()) + xh.abs() * mean_g((t * xh).abs()))
    return dx, (dz * xh).sum((0, 2, 3)), dz.sum((0, 2, 3)), size, (dz * xh).abs().sum((0, 2, 3)), dz.abs().sum((0, 2, 3))


@pytest.mark.parametrize("act", ["relu", "silu", "none"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(gpu_device, shape, dtype, act):
    from dnanet_amd.group_norm import group_norm_act, group_norm_act_backward
    from dnanet_amd.hip import PlaneBuffer
    buf, x, gamma, beta = make(shape, dtype, seed=1)
    n, c, groups, h, w = shape
    _, stats = group_norm_act(buf.ref(c), gamma.cuda(), beta.cuda(), groups, EPS, act)
    g = torch.randn(n, c, h, w, generator=torch.Generator().manual_seed(2))
    g = g.bfloat16().float() if dtype == "bf16" else g
    gbuf = PlaneBuffer.from_nchw(g.cuda(), buf.dtype)
    keep = gbuf.data.clone()
    dx, dgamma, dbeta = group_norm_act_backward(gbuf.ref(c), buf.ref(c), gamma.cuda(), stats)
    assert torch.equal(gbuf.data, keep)
    saved = [t.double().cpu() for t in (stats.mean, stats.rstd, stats.scale[:, :c], stats.shift[:, :c])]
    want = backward_definition(g.double(), x, gamma, *saved, groups, act)
    close(dx.to_nchw(c), want[0], 64 * U * want[3] + HALF[dtype] * want[0].abs(), "dx")
    close(dgamma, want[1], 64 * U * want[4] + 1e-30, "dgamma")
    close(dbeta, want[2], 64 * U * want[5] + 1e-30, "dbeta")
    # in place: the same bits
    group_norm_act_backward(gbuf.ref(c), buf.ref(c), gamma.cuda(), stats, out=gbuf.ref(c))
    assert torch.equal(gbuf.data, dx.data)


# groups (or planes) of 96, 120 and 192 blocks, and of 384, which take the form of three launches
LARGE = [(2, 128, 1, 6, 4096), (1, 40, 4, 6, 40000), (1, 16, 2, 6, 65536), (1, 512, 1, 6, 4096)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", LARGE)
def test_large_groups(gpu_device, shape, dtype):
    test_forward(gpu_device, shape, dtype, "silu")
    test_backward(gpu_device, shape, dtype, "relu")


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(600, 24, 3, 1, 9), (140, 64, 8, 2, 300), (129, 64, 4, 1, 65), (127, 64, 4, 1, 65)])
def test_many_images(gpu_device, shape, dtype):
    """Around and past the number of blocks up to which a launch sums the parameter gradients itself."""
    test_forward(gpu_device, shape, dtype, "relu")
    test_backward(gpu_device, shape, dtype, "silu")


def test_backward_agrees_with_differences(gpu_device):
    """L = sum(w * a): <dx, d> + <dgamma, dg> + <dbeta, db> of the kernels against the change of the definition's L along that
    direction, in 64 bits: the quotient's own error is step^2 / 6 of a third derivative (below 4 sum|w|), the kernels' 64 u of
    the magnitudes that enter each gradient."""
    from dnanet_amd.group_norm import group_norm_act, group_norm_act_backward
    from dnanet_amd.hip import F32, PlaneBuffer
    shape = (2, 16, 4, 3, 21)
    n, c, groups, h, w = shape
    gen = torch.Generator().manual_seed(5)
    x, d, wgt = (torch.randn(n, c, h, w, generator=gen) for _ in range(3))
    gamma, beta, dg, db = 1 + 0.2 * torch.randn(c, generator=gen), 0.2 * torch.randn(c, generator=gen), torch.randn(c, generator=gen), torch.randn(c, generator=gen)

    def loss(step):
        moved = [v.double() + step * e.double() for v, e in ((x, d), (gamma, dg), (beta, db))]
        return float((definition(*moved, groups, "silu")[0] * wgt.double()).sum())

    buf = PlaneBuffer.from_nchw(x.cuda(), F32)
    _, stats = group_norm_act(buf.ref(c), gamma.cuda(), beta.cuda(), groups, EPS, "silu")
    dx, dgamma, dbeta = group_norm_act_backward(PlaneBuffer.from_nchw(wgt.cuda(), F32).ref(c), buf.ref(c), gamma.cuda(), stats)
    slope = float((dx.to_nchw(c).double().cpu() * d).sum() + (dgamma.double().cpu() * dg).sum() + (dbeta.double().cpu() * db).sum())
    step = 2.0 ** -14
    quotient = (loss(step) - loss(-step)) / (2 * step)
    saved = [t.double().cpu() for t in (stats.mean, stats.rstd, stats.scale[:, :c], stats.shift[:, :c])]
    _, _, _, size, size_g, size_b = backward_definition(wgt.double(), x.double(), gamma, *saved, groups, "silu")
    off = 64 * U * float((size * d.abs()).sum() + (size_g * dg.abs()).sum() + (size_b * db.abs()).sum()) + 4 * step ** 2 * float(wgt.abs().sum())
    assert off < 0.05 * abs(slope), "the direction says something"
    assert abs(quotient - slope) <= off, (quotient, slope, off)


def test_mean_far_from_zero_does_not_cancel(gpu_device):
    """mean 1000, deviation 1: E[x^2] - mean^2 in fp32 would keep one digit."""
    from dnanet_amd.group_norm import group_norm_act
    from dnanet_amd.hip import F32, PlaneBuffer
    x = 1000 + torch.randn(2, 16, 5, 999, generator=torch.Generator().manual_seed(0))
    _, stats = group_norm_act(PlaneBuffer.from_nchw(x.cuda(), F32).ref(16), torch.ones(16).cuda(), torch.zeros(16).cuda(), 4, EPS, "none")
    rstd = (x.double().reshape(2, 4, -1).var(-1, unbiased=False) + EPS) ** -0.5
    close(stats.rstd, rstd, rstd * (64 * U + (32 * U * 1005) ** 2), "rstd")


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("act", ["relu", "silu"])
def test_non_finite_values_stay_in_their_group(gpu_device, value, act):
    from dnanet_amd.group_norm import group_norm_act
    from dnanet_amd.hip import F32, PlaneBuffer
    x = torch.randn(2, 32, 5, 70, generator=torch.Generator().manual_seed(0))
    gamma, beta = torch.ones(32).cuda(), torch.zeros(32).cuda()
    clean, _ = group_norm_act(PlaneBuffer.from_nchw(x.cuda(), F32).ref(32), gamma, beta, 8, EPS, act)
    x[1, 13, 2, 40] = value                                    # channel 13: group 3
    out, _ = group_norm_act(PlaneBuffer.from_nchw(x.cuda(), F32).ref(32), gamma, beta, 8, EPS, act)
    got, want = out.to_nchw(32), clean.to_nchw(32)
    assert bool(got[1, 12:16].isnan().all()), "a group with a NaN / infinity has no statistics"
    got[1, 12:16] = want[1, 12:16]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(2, 12, 3, 5, 300), (3, 20, 5, 2, 4096), (2, 36, 9, 6, 40), (1, 515, 1, 2, 4096)])
def test_slots_past_the_channels_may_hold_anything(gpu_device, shape, dtype):
    """NaN and infinities in a partial plane's unused slots: the results of zeros there, zeros in those slots of the outputs."""
    from dnanet_amd import hip
    from dnanet_amd.group_norm import group_norm_act, group_norm_act_backward
    from dnanet_amd.hip import PlaneBuffer
    n, c, groups, h, w = shape
    clean, _, gamma, beta = make(shape, dtype, seed=4)
    gamma, beta, epr = gamma.cuda(), beta.cuda(), hip.epr(clean.dtype)
    grad = PlaneBuffer.wrap(clean.data.flip(-2).contiguous())
    dirty = [PlaneBuffer.wrap(b.data.clone()) for b in (clean, grad)]
    used = c % epr
    assert used
    for b, value in zip(dirty, (float("nan"), float("inf"))):
        b.data[:, -1, :, :, used:] = value
        b.data[:, -1, ::2, :, used:] = -value
    results = []
    for x, g in ((clean, grad), dirty):
        a, stats = group_norm_act(x.ref(c), gamma, beta, groups, EPS, "silu")
        dx, dgamma, dbeta = group_norm_act_backward(g.ref(c), x.ref(c), gamma, stats)
        results.append((a.data, dx.data, stats.mean, stats.rstd, stats.scale, stats.shift, dgamma, dbeta))
    for want, got in zip(*results):
        assert torch.equal(got, want)
    assert not results[1][0][:, -1, :, :, used:].any() and not results[1][1][:, -1, :, :, used:].any()


def test_constant_group(gpu_device):
    """Variance 0: rstd = eps^-1/2 = 316, z = beta up to one rounding of the shift (3 * 316), and the gradient is finite."""
    from dnanet_amd.group_norm import group_norm_act, group_norm_act_backward
    from dnanet_amd.hip import F32, PlaneBuffer
    x = torch.full((1, 8, 2, 50), 3.0)
    beta = torch.linspace(-1, 1, 8)
    buf = PlaneBuffer.from_nchw(x.cuda(), F32)
    out, stats = group_norm_act(buf.ref(8), torch.ones(8).cuda(), beta.cuda(), 2, EPS, "none")
    close(out.to_nchw(8), beta.double().view(1, 8, 1, 1).expand(1, 8, 2, 50), 2 * U * 3 * 317, "output")
    dx, _, _ = group_norm_act_backward(PlaneBuffer.from_nchw(torch.randn_like(x).cuda(), F32).ref(8), buf.ref(8), torch.ones(8).cuda(), stats)
    assert bool(dx.data.isfinite().all())


def test_part_of_a_wider_buffer(gpu_device):
    """x, output and gradients in the planes [2, 4) / [1, 3) of wider buffers; the other planes stay as they were."""
    from dnanet_amd.group_norm import group_norm_act, group_norm_act_backward
    from dnanet_amd.hip import BF16, PlaneBuffer
    small, x, gamma, beta = make((3, 24, 3, 5, 77), "bf16")
    n, c, groups, h, w = 3, 24, 3, 5, 77
    want, wstats = group_norm_act(small.ref(c), gamma.cuda(), beta.cuda(), groups, EPS, "relu")
    wide, res = PlaneBuffer(n, 5, h, w, BF16, "cuda"), PlaneBuffer(n, 4, h, w, BF16, "cuda")
    wide.data.fill_(7.0)
    res.data.fill_(9.0)
    wide.data[:, 2:4] = small.data
    _, stats = group_norm_act(wide.ref(c, 2), gamma.cuda(), beta.cuda(), groups, EPS, "relu", out=res.ref(c, 1))
    assert torch.equal(res.data[:, 1:3], want.data) and torch.equal(stats.shift, wstats.shift)
    assert bool((res.data[:, 0] == 9).all()) and bool((res.data[:, 3] == 9).all()) and bool((wide.data[:, :2] == 7).all())
    g = torch.randn(n, c, h, w).cuda()
    gs = PlaneBuffer.from_nchw(g, BF16)
    dx0, dg0, db0 = group_norm_act_backward(gs.ref(c), small.ref(c), gamma.cuda(), wstats)
    res.data[:, 1:3] = gs.data
    _, dg1, db1 = group_norm_act_backward(res.ref(c, 1), wide.ref(c, 2), gamma.cuda(), stats, out=res.ref(c, 1))
    assert torch.equal(res.data[:, 1:3], dx0.data) and torch.equal(dg0, dg1) and torch.equal(db0, db1)
    assert bool((res.data[:, 0] == 9).all()) and bool((res.data[:, 3] == 9).all())


def test_in_place_and_repeatable(gpu_device):
    from dnanet_amd.group_norm import group_norm_act
    buf, _, gamma, beta = make((5, 64, 8, 5, 640), "bf16")
    args = (gamma.cuda(), beta.cuda(), 8, EPS, "silu")
    first, s1 = group_norm_act(buf.ref(64), *args)
    second, s2 = group_norm_act(buf.ref(64), *args)
    assert torch.equal(first.data, second.data) and torch.equal(s1.mean, s2.mean)
    group_norm_act(buf.ref(64), *args, out=buf.ref(64))
    assert torch.equal(buf.data, first.data)


def test_empty_batch(gpu_device):
    from dnanet_amd.group_norm import group_norm_act
    from dnanet_amd.hip import F32, PlaneBuffer
    out, stats = group_norm_act(PlaneBuffer(0, 4, 5, 32, F32, "cuda").ref(32), torch.ones(32).cuda(), torch.zeros(32).cuda(), 8)
    assert out.data.shape[0] == 0 and stats.mean.shape == (0, 8)


def test_graphs_and_streams(gpu_device):
    """Two graphs captured one after the other and replayed on two streams at once, eager calls in between, another stream."""
    from dnanet_amd.group_norm import group_norm_act, group_norm_act_backward
    shape = (6, 64, 8, 5, 512)
    n, c, groups, h, w = shape
    made = [make(shape, "bf16", seed=s) for s in (1, 2)]
    vec = [(m[2].cuda(), m[3].cuda()) for m in made]

    def both(k):
        a, stats = group_norm_act(made[k][0].ref(c), *vec[k], groups, EPS, "silu")
        return a, group_norm_act_backward(a.ref(c), made[k][0].ref(c), vec[k][0], stats)

    want = [both(k) for k in range(2)]
    torch.cuda.synchronize()
    graphs, got = [], []
    for k in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got.append(both(k))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        for k in range(2):
            for t in (got[k][0].data, got[k][1][0].data, got[k][1][1], got[k][1][2]):
                t.zero_()
        torch.cuda.synchronize()
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
        eager = both(0)
        torch.cuda.synchronize()
        for k in range(2):
            for a, b in ((got[k], want[k]), (eager, want[0])):
                assert torch.equal(a[0].data, b[0].data) and torch.equal(a[1][0].data, b[1][0].data)
                assert torch.equal(a[1][1], b[1][1]) and torch.equal(a[1][2], b[1][2])
    with torch.cuda.stream(streams[0]):
        other = both(1)
    streams[0].synchronize()
    assert torch.equal(other[0].data, want[1][0].data) and torch.equal(other[1][0].data, want[1][1][0].data)


def test_one_workspace_for_many_sizes(gpu_device):
    """A caller's workspace serves calls of any sizes, one after the other, forward and backward."""
    from dnanet_amd import hip
    from dnanet_amd.group_norm import group_norm_act, group_norm_act_backward
    ws = torch.zeros(8 << 20, dtype=torch.uint8, device="cuda")
    for seed in range(2):
        for shape in SHAPES:
            buf, _, gamma, beta = make(shape, "bf16", seed)
            args = (gamma.cuda(), beta.cuda(), shape[2], EPS, "relu")
            a, s1 = group_norm_act(buf.ref(shape[1]), *args, workspace=ws)
            b, s2 = group_norm_act(buf.ref(shape[1]), *args)
            assert torch.equal(a.data, b.data) and torch.equal(s1.rstd, s2.rstd)
            ga = group_norm_act_backward(a.ref(shape[1]), buf.ref(shape[1]), args[0], s1, workspace=ws)
            gb = group_norm_act_backward(b.ref(shape[1]), buf.ref(shape[1]), args[0], s2)
            assert torch.equal(ga[0].data, gb[0].data) and torch.equal(ga[1], gb[1])
    assert hip.lib.dn_group_norm_workspace_bytes(1, 8, 1, 1, 1, 0) > 0


def test_offsets_past_32_bits(gpu_device):
    """A 4.4-GB tensor: its last images come out as they do alone."""
    from dnanet_amd.group_norm import group_norm_act, group_norm_act_backward
    from dnanet_amd.hip import F32, PlaneBuffer
    n, c, h, w = 1420, 32, 6, 4096
    big = PlaneBuffer(n, 4, h, w, F32, "cuda")
    assert big.data.numel() * 4 > 1 << 32
    torch.manual_seed(0)
    big.data.normal_()
    gamma, beta = torch.rand(c).cuda() + 0.5, torch.rand(c).cuda()
    out, stats = group_norm_act(big.ref(c), gamma, beta, 8, EPS, "relu")
    tail = PlaneBuffer.wrap(big.data[-2:].clone())
    want, wstats = group_norm_act(tail.ref(c), gamma, beta, 8, EPS, "relu")
    assert torch.equal(out.data[-2:], want.data) and torch.equal(stats.scale[-2:], wstats.scale)
    group_norm_act_backward(out.ref(c), big.ref(c), gamma, stats, out=out.ref(c))
    dx, _, _ = group_norm_act_backward(want.ref(c), tail.ref(c), gamma, wstats)
    assert torch.equal(out.data[-2:], dx.data)


def test_refusals(gpu_device):
    from dnanet_amd.group_norm import group_norm_act, group_norm_act_backward
    from dnanet_amd.hip import BF16, F32, HipError, PlaneBuffer
    x = PlaneBuffer(2, 4, 5, 32, F32, "cuda", zero=True)
    one, zero = torch.ones(32).cuda(), torch.zeros(32).cuda()
    with pytest.raises(ValueError, match="divide"):
        group_norm_act(x.ref(32), one, zero, 5)
    with pytest.raises(ValueError, match="divide"):
        group_norm_act(x.ref(32), one, zero, 0)
    with pytest.raises(ValueError, match="activation"):
        group_norm_act(x.ref(32), one, zero, 8, activation="gelu")
    with pytest.raises(ValueError, match="gamma"):
        group_norm_act(x.ref(32), one[:16], zero, 8)
    with pytest.raises(ValueError, match="gamma"):
        group_norm_act(x.ref(32), one.double(), zero, 8)
    with pytest.raises(ValueError, match="beta"):
        group_norm_act(x.ref(32), one, zero.cpu(), 8)
    with pytest.raises(HipError, match="eps"):
        group_norm_act(x.ref(32), one, zero, 8, eps=0.0)
    with pytest.raises(ValueError, match="out is"):
        group_norm_act(x.ref(32), one, zero, 8, out=PlaneBuffer(2, 4, 5, 31, F32, "cuda").ref(32))
    with pytest.raises(ValueError, match="out is"):
        group_norm_act(x.ref(32), one, zero, 8, out=PlaneBuffer(2, 2, 5, 32, BF16, "cuda").ref(32))
    with pytest.raises(HipError, match="channels"):
        group_norm_act(x.ref(32), one, zero, 8, out=PlaneBuffer(2, 4, 5, 32, F32, "cuda").ref(24))
    with pytest.raises(HipError, match="workspace"):
        group_norm_act(x.ref(32), one, zero, 8, workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError, match="record"):
        PlaneBuffer.wrap(torch.zeros(2, 4, 5, 32, 16, device="cuda"))
    with pytest.raises(ValueError, match="record"):
        PlaneBuffer.wrap(torch.zeros(2, 4, 32, 5, 8, device="cuda").transpose(2, 3))
    a, stats = group_norm_act(x.ref(32), one, zero, 8)
    with pytest.raises(ValueError, match="overlap"):
        group_norm_act_backward(a.ref(32), x.ref(32), one, stats, out=x.ref(32))
    with pytest.raises(ValueError, match="stats.mean"):
        stats.groups = 4
        group_norm_act_backward(a.ref(32), x.ref(32), one, stats)


def test_refused_workspaces_and_outputs(gpu_device):
    from dnanet_amd.group_norm import group_norm_act, group_norm_act_backward
    from dnanet_amd.hip import F32, HipError, PlaneBuffer
    x = PlaneBuffer(2, 8, 5, 32, F32, "cuda", zero=True)
    one, zero = torch.ones(32).cuda(), torch.zeros(32).cuda()
    for ws in (torch.zeros(1 << 24), torch.zeros(1 << 24, dtype=torch.uint8), torch.zeros(1 << 24).cuda(),
               torch.zeros(1 << 24, dtype=torch.uint8, device="cuda")[::2]):
        with pytest.raises(ValueError, match="workspace"):
            group_norm_act(x.ref(32), one, zero, 8, workspace=ws)
    for plane0 in (1, 3):
        with pytest.raises(HipError, match="overlaps"):
            group_norm_act(x.ref(32), one, zero, 8, out=x.ref(32, plane0))
    a, stats = group_norm_act(x.ref(32), one, zero, 8, out=x.ref(32, 4))
    g = PlaneBuffer(2, 8, 5, 32, F32, "cuda", zero=True)
    with pytest.raises(HipError, match="overlaps"):
        group_norm_act_backward(g.ref(32, 4), x.ref(32, 0), one, stats, out=g.ref(32, 3))
    with pytest.raises(HipError, match="dgamma and dbeta"):
        group_norm_act_backward(a.ref(32, 4), x.ref(32, 0), one, stats, dgamma=one, dbeta=one)


GIVE_UP = """
import hashlib, sys, torch
sys.path[:0] = [{root!r}, {tests!r}]
from test_group_norm_gpu import digests
print("DIGESTS", digests())
"""
EXCHANGE_SHAPES = [(2, 40, 5, 3, 2000), (3, 64, 2, 5, 1500), (2, 60, 5, 4, 1500), (16, 32, 8, 6, 4096), (30, 128, 8, 5, 1024), (130, 512, 8, 6, 256)]


def digests():
    """Hashes of forward and (in place) backward results at shapes whose groups are spread over several blocks."""
    import hashlib
    from dnanet_amd import hip
    from dnanet_amd.group_norm import group_norm_act, group_norm_act_backward
    from dnanet_amd.hip import PlaneBuffer
    out = []
    for dtype in (hip.BF16, hip.F32):
        for n, c, groups, h, w in EXCHANGE_SHAPES:
            gen = torch.Generator(device="cuda").manual_seed(n + c)
            x, g = (PlaneBuffer(n, hip.planes(c, dtype), h, w, dtype, "cuda") for _ in range(2))
            for b in (x, g):
                b.data.copy_(torch.randn(b.data.shape, generator=gen, device="cuda"))
                if c % hip.epr(dtype):
                    b.data[:, -1, :, :, c % hip.epr(dtype):] = 0
            gamma, beta = torch.rand(c, generator=gen, device="cuda") + 0.5, torch.rand(c, generator=gen, device="cuda")
            for act in ("relu", "silu"):
                a, stats = group_norm_act(x.ref(c), gamma, beta, groups, EPS, act)
                mine = PlaneBuffer.wrap(g.data.clone())
                _, dgamma, dbeta = group_norm_act_backward(mine.ref(c), x.ref(c), gamma, stats, out=mine.ref(c))
                md5 = hashlib.md5()
                for t in (a.data, mine.data, dgamma, dbeta, stats.mean, stats.rstd, stats.scale, stats.shift):
                    md5.update(t.contiguous().view(torch.uint8).cpu().numpy().tobytes())
                out.append(md5.hexdigest()[:12])
    return out


def test_blocks_that_give_up_waiting(gpu_device):
    """A block that does not find the sums it waits for leaves its segment to the launch's last block: with no patience at all
    (one look) the results are the same bits."""
    import os
    import subprocess
    import sys
    tests = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, DN_TUNE_GN_POLLS="1")
    run = subprocess.run([sys.executable, "-c", GIVE_UP.format(root=os.path.dirname(tests), tests=tests)], env=env, capture_output=True,
                         text=True, timeout=100)
    assert run.returncode == 0, run.stderr[-2000:]
    impatient = run.stdout.split("DIGESTS ", 1)[1].strip()
    assert impatient == str(digests())
