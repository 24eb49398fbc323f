"""The running mean of the training BatchNorm, to the last bit: the two products and their sum rounded one by one."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_running_mean_rounds_products_and_sum(gpu_device, dtype):
    from dnanet_amd.synthetic import make_batch
    from dnanet_amd.unet import HipUNet
    m = HipUNet(2, (3, 5), 16, "cuda", dtype=dtype)
    m.reset_parameters(torch.Generator().manual_seed(0))
    m.train()
    momentum = torch.tensor(0.1)
    for step in range(3):
        x, _ = make_batch(3, 5, 256, seed=step, unique=3)
        before = {u.bn: m.tensor(u.bn + ".running_mean").cpu().clone() for u in m.conv_units}
        m(torch.from_numpy(x).cuda())
        for u in m.conv_units:
            mean = m._saved[u.conv]["mean"][:u.cout].cpu()
            want = (1 - momentum) * before[u.bn] + momentum * mean
            assert torch.equal(m.tensor(u.bn + ".running_mean").cpu(), want), (step, u.bn)
