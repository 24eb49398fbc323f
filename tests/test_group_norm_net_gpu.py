"""The U-Net with group norm, AdamW and clipping as ``fit`` runs them: forward, gradients and updates against plain torch in 64
bits (held to the bars of the BatchNorm net: logits 2e-5 of the largest, gradients 2e-3 of a tensor's largest), graph replay
against launch by launch, checkpoints, and the reference API's keywords."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
ACT = {"relu": torch.relu, "silu": F.silu, "none": lambda z: z}


def plain_forward(sd, x, depth, groups, act, kernel, convs=None):
    """``convs``: filled with (weight key, input, output) of every convolution, outputs keeping their gradients."""
    pad = (kernel[0] // 2, kernel[1] // 2)

    def double(prefix, x):
        for conv, norm in ((0, 1), (3, 4)):
            k = f"{prefix}.double_conv."
            y = F.conv2d(x, sd[f"{k}{conv}.weight"], sd[f"{k}{conv}.bias"], padding=pad)
            if convs is not None:
                y.retain_grad()
                convs[f"{k}{conv}.weight"] = (x, y)
            x = y
            x = ACT[act](F.group_norm(x, groups, sd[f"{k}{norm}.weight"], sd[f"{k}{norm}.bias"], 1e-5))
        return x

    skips = []
    for l in range(depth):
        x = double(f"encoders.{l}.conv", x)
        skips.append(x)
        x = F.max_pool2d(x, (1, 2))
    x = double("bottleneck", x)
    for i in range(depth):
        up = F.conv_transpose2d(x, sd[f"decoders.{i}.up.weight"], sd[f"decoders.{i}.up.bias"], stride=(1, 2))
        x = double(f"decoders.{i}.conv", torch.cat([up, skips[depth - 1 - i]], 1))
    return F.conv2d(x, sd["outputs.weight"], sd["outputs.bias"])


def dice(logits, t):
    p = torch.sigmoid(logits).flatten()
    t = t.flatten().to(p.dtype)
    return 1 - (2 * (p * t).sum() + 1) / (p.sum() + t.sum() + 1)


def make(depth, filters, h, w, n, groups, act, dtype, kernel=(3, 5), seed=0):
    from dnanet_amd.unet import HipUNet
    m = HipUNet(depth, kernel, filters, "cuda", dtype=dtype, norm="group", num_groups=groups, activation=act)
    m.reset_parameters(torch.Generator().manual_seed(seed))
    gen = torch.Generator().manual_seed(seed + 1)
    for u in m.conv_units:
        m.tensor(u.bn + ".weight").data.copy_(1 + 0.2 * torch.randn(u.cout, generator=gen))
        m.tensor(u.bn + ".bias").data.copy_(0.2 * torch.randn(u.cout, generator=gen))
    m._param_epoch += 1
    x = (torch.rand(n, 1, h, w, generator=gen) ** 4 * 8000).round()
    t = (torch.rand(n, 1, h, w, generator=gen) < 0.05).to(torch.int8)
    return m, x, t


@pytest.mark.parametrize("depth,filters,h,w,n,groups,act,kernel", [
    (2, 32, 5, 256, 2, 8, "relu", (3, 5)), (2, 16, 6, 96, 3, 4, "silu", (3, 5)), (1, 24, 5, 50, 1, 8, "silu", (3, 5)),
    (3, 8, 5, 128, 2, 1, "relu", (1, 3)), (2, 8, 3, 32, 2, 8, "silu", (1, 1))])
def test_net_forward_and_gradients(gpu_device, depth, filters, h, w, n, groups, act, kernel):
    m, x, t = make(depth, filters, h, w, n, groups, act, "fp32", kernel)
    sd = {k: v.detach().double().cpu().requires_grad_(True) for k, v in m.state_dict().items()}
    assert not any("running" in k or "num_batches" in k for k in sd)
    convs = {}
    logits = plain_forward(sd, x.double(), depth, groups, act, kernel, convs)
    loss = dice(logits, t)
    loss.backward()
    m.eval()
    got = m(x.cuda()).double().cpu()
    scale = float(logits.detach().abs().max())
    assert float((got - logits.detach()).abs().max()) < 2e-5 * scale
    m.train()
    train = m(x.cuda())
    assert float((train.double().cpu() - logits.detach()).abs().max()) < 2e-5 * scale, "training and evaluation compute the same"
    sums = m.dice_forward(train, t.cuda())
    assert abs(float(sums[4]) - float(loss.detach())) < 2e-5
    m.backward()
    for k, v in sd.items():
        err = float((m.grad(k).double().cpu() - v.grad).abs().max())
        rounding = 1e-9
        if k in convs:
            # a weight gradient is a sum of products dy * x; where it cancels (a 1x1 kernel on one channel in front of one-channel
            # groups: scaling y changes nothing, the gradient is 0) the roundings of the products stay: 256 u of their sum.  A
            # bias likewise: sum dy is 0 in front of one-channel groups
            a, y = convs[k]
            rounding += 256 * 2.0 ** -24 * float(torch.nn.grad.conv2d_weight(a.detach().abs(), v.shape, y.grad.abs(),
                                                                              padding=(kernel[0] // 2, kernel[1] // 2)).max())
        elif k.endswith(".bias") and k[:-4] + "weight" in convs:
            rounding += 256 * 2.0 ** -24 * float(convs[k[:-4] + "weight"][1].grad.abs().sum((0, 2, 3)).max())
        assert err < 2e-3 * float(v.grad.abs().max()) + rounding, (k, err, float(v.grad.abs().max()))


def test_net_bf16_and_batch_independence(gpu_device):
    """bf16: logits within the bar of the BatchNorm net (2e-2 of the largest); a profile's result does not depend on its batch."""
    m, x, t = make(2, 32, 5, 256, 4, 8, "silu", "bf16")
    sd = {k: v.detach().double().cpu() for k, v in m.state_dict().items()}
    want = plain_forward(sd, x.double(), 2, 8, "silu", (3, 5))
    m.eval()
    got = m(x.cuda())
    assert float((got.double().cpu() - want).abs().max()) < 4e-2 * float(want.abs().max())
    assert torch.equal(m(x[2:3].cuda()), got[2:3])
    m.train()
    assert torch.equal(m(x[1:2].cuda()), m(x.cuda())[1:2])


@pytest.mark.parametrize("bits,clip", [(32, None), (8, 0.05)])
def test_training_step_group_norm_adamw(gpu_device, bits, clip):
    """Forward, backward, clipped AdamW on the net's arena: the update against torch.optim.AdamW in 64 bits on the kernels' own
    gradients, weights decayed and vectors not; gradients zeroed by the step."""
    from dnanet_amd.optim import HipAdamW
    m, x, t = make(2, 16, 5, 128, 2, 4, "silu", "fp32")
    m.train()
    opt = HipAdamW(m, lr=1e-3, weight_decay=0.1, state_bits=bits, max_grad_norm=clip)
    opt.zero_grad()
    m.dice_forward(m(x.cuda()), t.cuda())
    m.backward()
    keys = [k for k, _, kind in m.spec if kind == "param"]
    mine = {k: m.tensor(k).detach().double().cpu().requires_grad_(True) for k in keys}
    for k in keys:
        mine[k].grad = m.grad(k).double().cpu()
    if clip:
        norm = torch.nn.utils.clip_grad_norm_(list(mine.values()), clip)
    ref = torch.optim.AdamW([{"params": [mine[k] for k in keys if mine[k].dim() == 4], "weight_decay": 0.1},
                             {"params": [mine[k] for k in keys if mine[k].dim() != 4], "weight_decay": 0.0}], lr=1e-3)
    ref.step()
    opt.step()
    if clip:
        assert float(norm) > clip and abs(float(opt.grad_norm) - float(norm)) < 4e-7 * float(norm)
    for k in keys:
        got, want = m.tensor(k).detach().double().cpu(), mine[k].detach()
        # first step: lr * g / (|g| + eps), off by a few roundings of the step (1e-3) and of the parameter
        assert float((got - want).abs().max()) <= 2.0 ** -24 * (4 * float(want.abs().max()) + 64e-3), k
    assert not m.flat_grads.any()


@pytest.mark.parametrize("optimizer", ["adamw", "adamw8bit"])
def test_fit_graph_equals_launch_by_launch(gpu_device, optimizer):
    from dnanet_amd.model import DNANet_UNet
    from dnanet_amd.data import SyntheticDataset
    images = list(SyntheticDataset(10, rows=5, width=256, seed=3))
    out = []
    for graph in (False, True):
        torch.manual_seed(0)
        model = DNANet_UNet(2, (3, 5), 16, device="cuda", apply_allele_caller=False, dtype="bf16", norm="group", num_groups=4, activation="silu")
        model.fit(images, batch_size=4, num_epochs=3, learning_rate=1e-3, weight_decay=0.01, optimizer=optimizer, max_grad_norm=1.0,
                  use_scheduler=True, hip_graph=graph, validation_set=images[8:], min_delta=-99999)
        out.append(model._model.flat_params.cpu())
        assert len(model.predict_batch(images[:3])) == 3
    # the replayed step reads its learning rate from device memory in fp32: parameters agree to roundings of single steps
    assert float((out[0] - out[1]).abs().max()) <= 6 * (2.0 ** -22 + 1e-3 * 2.0 ** -6)


def test_fit_data_parallel_group_of_one(gpu_device):
    """A group norm has no batch statistics: the data-parallel fit of one rank is the plain one, sync_bn is refused."""
    import torch.distributed as dist
    from dnanet_amd.model import DNANet_UNet
    from dnanet_amd.data import SyntheticDataset
    images = list(SyntheticDataset(8, rows=5, width=256, seed=3))

    def fitted(**kw):
        torch.manual_seed(0)
        model = DNANet_UNet(2, (3, 5), 16, device="cuda", apply_allele_caller=False, norm="group", num_groups=4)
        model.fit(images, batch_size=4, num_epochs=2, learning_rate=1e-3, optimizer="adamw", max_grad_norm=1.0, hip_graph=False, **kw)
        return model._model.flat_params.cpu()

    plain = fitted()
    import os
    os.environ.setdefault("MASTER_ADDR", "127.0.0.1")
    os.environ["MASTER_PORT"] = "29617"
    dist.init_process_group("gloo", rank=0, world_size=1)
    try:
        assert torch.equal(fitted(data_parallel=True), plain)
        with pytest.raises(ValueError, match="sync_bn"):
            fitted(data_parallel=True, sync_bn=True)
    finally:
        dist.destroy_process_group()


def test_checkpoint_round_trip(gpu_device, tmp_path):
    from dnanet_amd.model import DNANet_UNet
    from dnanet_amd.data import SyntheticDataset
    images = list(SyntheticDataset(3, rows=5, width=256, seed=3))
    a = DNANet_UNet(2, (3, 5), 16, device="cuda", apply_allele_caller=False, norm="group", num_groups=4, activation="silu")
    a.save(tmp_path)
    b = DNANet_UNet(2, (3, 5), 16, device="cuda", apply_allele_caller=False, norm="group", num_groups=4, activation="silu")
    b.load(tmp_path)
    for p, q in zip(a.predict_batch(images), b.predict_batch(images)):
        assert (p.image == q.image).all()


def test_capture_before_any_other_pass(gpu_device):
    """A training step captured first of all, evaluation before its first replay: the model's group-norm workspace is zeroed when the
    step is captured, not when it is replayed."""
    from dnanet_amd.optim import HipAdamW
    from dnanet_amd.unet import GraphedTrainStep
    out = []
    for graphed in (False, True):
        m, x, t = make(2, 16, 5, 128, 3, 4, "silu", "bf16")
        opt = HipAdamW(m, lr=1e-3)
        m.train()
        if graphed:
            step = GraphedTrainStep(m, opt, x.cuda(), t.cuda())
        m.eval()
        with torch.no_grad():
            before = m(x.cuda()).clone()
        m.train()
        for _ in range(3):
            if graphed:
                step(x.cuda(), t.cuda())
            else:
                m.dice_forward(m(x.cuda()), t.cuda())
                m.backward()
                opt.step()
                opt.zero_grad()
        m.eval()
        with torch.no_grad():
            out.append((before, m(x.cuda()).clone()))
    assert torch.equal(out[0][0], out[1][0])
    # the replayed step reads its learning rate in fp32: parameters differ by 2^-24 of three steps of 1e-3, logits by what that and
    # bf16's roundings of such weights make of it: below one step of bf16 at the largest logit
    assert float((out[0][1] - out[1][1]).abs().max()) <= 2.0 ** -7 * float(out[0][1].abs().max())


def test_evaluation_captured_by_a_caller(gpu_device):
    """An evaluation captured into a caller's graph keeps its results when the model has meanwhile evaluated a larger batch."""
    m, x, _ = make(2, 16, 5, 128, 2, 4, "relu", "bf16")
    m.eval()
    x = x.cuda()
    with torch.no_grad():
        want = m(x).clone()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            got = m(x)
        for n in (5, 40):
            other = m(x[:1].expand(n, -1, -1, -1).contiguous())
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want) and torch.equal(other[-1], want[0])
