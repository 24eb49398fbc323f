"""Group norm and clipped AdamW, data parallel over two ranks that share the GPU (gloo, through the host): two halves of a batch are
the batch, and both ranks hold the same parameters bit for bit."""
import os
import socket

import pytest
import torch

pytestmark = pytest.mark.gpu
LR, CLIP = 1e-3, 0.05


def _net():
    from dnanet_amd.unet import HipUNet
    m = HipUNet(2, (3, 5), 16, "cuda", dtype="fp32", norm="group", num_groups=4, activation="silu")
    m.reset_parameters(torch.Generator().manual_seed(0))
    m._param_epoch += 1
    m.train()
    return m


def _batch():
    from dnanet_amd.synthetic import make_batch
    x, t = make_batch(8, 5, 256, seed=31, unique=8)
    return torch.from_numpy(x), torch.from_numpy(t)


def _optimizer(m, bits):
    from dnanet_amd.optim import HipAdamW
    return HipAdamW(m, lr=LR, weight_decay=0.01, state_bits=bits, max_grad_norm=CLIP, seed=11)


def _rank(rank, world, port, bits, out):
    import faulthandler
    import torch.distributed as dist
    from dnanet_amd.distributed import DataParallelTrainer, all_reduce_dice_sums
    faulthandler.dump_traceback_later(60, exit=True)      # a rank stuck in a collective ends (and says where) before pytest's limit
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    torch.cuda.set_device(0)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        m = _net()
        opt = _optimizer(m, bits)
        x, t = (v[rank * 4:rank * 4 + 4].cuda() for v in _batch())
        trainer = DataParallelTrainer(m, opt, min_bucket_elems=10000)
        sums = all_reduce_dice_sums(m.dice_forward(m.forward_train(x), t))
        m.backward(sums=sums, segment_hook=trainer.reducer.segment_done)
        trainer.reducer.finish()
        grads = m.flat_grads.cpu()
        opt.step()
        opt.zero_grad()
        first, norm = m.flat_params.cpu(), opt.grad_norm.cpu()
        for _ in range(2):
            trainer.step(x, t)
        torch.save({"grads": grads, "first": first, "norm": norm, "params": m.flat_params.cpu()}, f"{out}.{rank}")
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("bits", [32, 8])
def test_two_ranks_are_one(gpu_device, tmp_path, bits):
    import torch.multiprocessing as mp
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    out = str(tmp_path / "rank")
    mp.spawn(_rank, args=(2, port, bits, out), nprocs=2, join=True)
    a, b = (torch.load(f"{out}.{r}", weights_only=True) for r in range(2))
    for key in a:
        assert torch.equal(a[key], b[key]), key
    m = _net()
    opt = _optimizer(m, bits)
    x, t = (v.cuda() for v in _batch())
    m.dice_forward(m(x), t)
    m.backward()
    whole = m.flat_grads.cpu()
    # sums of the same products in another order: the bar of the BatchNorm net with synchronised statistics
    assert float((a["grads"] - whole).norm()) < 1e-5 * float(whole.norm())
    m.flat_grads.copy_(a["grads"])
    opt.step()
    assert torch.equal(opt.grad_norm.cpu(), a["norm"]) and float(a["norm"]) > CLIP
    assert torch.equal(m.flat_params.cpu(), a["first"])
    assert not torch.equal(a["params"], a["first"])
