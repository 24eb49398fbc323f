"""Group norm and AdamW: what is decided on the host -- argument checks of the C entry points and of the Python layer, the
parameter tree of a group-norm net, fit keywords, configuration files."""
import ctypes
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_group_norm_entry_points_refuse():
    from dnanet_amd import hip
    ws = hip.lib.dn_group_norm_workspace_bytes
    assert ws(2, 32, 5, 4096, 8, hip.BF16) > 0 and ws(0, 32, 5, 4096, 8, hip.F32) > 0
    for bad in ((2, 32, 5, 64, 5, 0), (2, 32, 5, 64, 0, 0), (2, 0, 5, 64, 1, 0), (2, 32, 0, 64, 8, 0), (2, 32, 5, 64, 8, 2), (-1, 32, 5, 64, 8, 0),
                (2, 32, 1 << 13, 1 << 13, 8, 0), (1 << 30, 64, 5, 64, 8, 0)):
        assert ws(*bad) == -1 and hip.lib.dn_last_error(), bad
    good = hip.DnTensor(4096, 4, 0, 32)
    vec = [4096] * 6

    def forward(x=good, a=good, n=2, groups=8, eps=1e-5, act=1, vectors=vec, work=4096, nbytes=1 << 30, dtype=0):
        g, b, *rest = vectors
        return hip.lib.dn_group_norm_act(x, a, n, 5, 64, groups, g, b, eps, act, *rest, work, nbytes, dtype, None)

    for kw in ({"x": hip.DnTensor(None, 4, 0, 32)}, {"x": hip.DnTensor(4097, 4, 0, 32)}, {"a": hip.DnTensor(4096, 4, 1, 32)},
               {"a": hip.DnTensor(4096, 4, -1, 32)}, {"a": hip.DnTensor(4096, 4, 0, 24)}, {"groups": 3}, {"eps": 0.0}, {"eps": -1.0},
               {"eps": float("nan")}, {"act": 3}, {"act": -1}, {"vectors": [None] + vec[1:]}, {"vectors": vec[:5] + [None]}, {"work": None},
               {"work": 4100}, {"nbytes": 64}, {"dtype": 7}):
        assert forward(**kw) == 1, kw
    assert forward(n=0) == 0, "an empty batch launches nothing"

    def backward(g=good, x=good, dx=good, n=2, groups=8, act=1, vectors=[4096] * 7, work=4096, nbytes=1 << 30, dtype=0):
        return hip.lib.dn_group_norm_act_backward(g, x, dx, n, 5, 64, groups, *vectors[:5], act, *vectors[5:], work, nbytes, dtype, None)

    for kw in ({"g": hip.DnTensor(None, 4, 0, 32)}, {"dx": hip.DnTensor(4096, 3, 0, 32)}, {"n": 0}, {"groups": 7}, {"act": 9},
               {"vectors": [4096] * 6 + [None]}, {"vectors": [None] + [4096] * 6}, {"work": None}, {"nbytes": 0}, {"dtype": -1}):
        assert backward(**kw) == 1, kw


def test_group_norm_refuses_tensors_that_share_memory():
    """32 channels of fp32 are 4 planes of 5 * 64 records of 32 bytes; two images of buffers of 4 (or 8) planes."""
    from dnanet_amd import hip
    plane, base = 5 * 64 * 32, 1 << 20
    x, apart = hip.DnTensor(base, 4, 0, 32), hip.DnTensor(1 << 24, 4, 0, 32)
    wide = [hip.DnTensor(base, 8, p, 32) for p in (0, 1, 3, 4)]

    def forward(x, a):
        return hip.lib.dn_group_norm_act(x, a, 2, 5, 64, 8, *[4096] * 2, 1e-5, 1, *[4096] * 5, 1 << 30, 0, None), hip.lib.dn_last_error()

    for a in (hip.DnTensor(base + 32, 4, 0, 32), hip.DnTensor(base - 32, 4, 0, 32), hip.DnTensor(base + 8 * plane - 32, 4, 0, 32),
              hip.DnTensor(base, 8, 0, 32), hip.DnTensor(base, 5, 1, 32)):
        rc, error = forward(x, a)
        assert rc == 1 and b"overlaps" in error, (a.base - base, error)
    for a in wide[1:3]:
        rc, error = forward(wide[0], a)
        assert rc == 1 and b"overlaps" in error, (a.plane0, error)

    def backward(g, x, dx, dgamma=1 << 26, dbeta=1 << 27):
        rc = hip.lib.dn_group_norm_act_backward(g, x, dx, 2, 5, 64, 8, *[4096] * 5, 1, dgamma, dbeta, 4096, 1 << 30, 0, None)
        return rc, hip.lib.dn_last_error()

    for args, word in (((apart, x, x), b"overlaps x"), ((apart, x, hip.DnTensor(base + 4 * plane, 4, 0, 32)), b"overlaps x"),
                       ((x, apart, hip.DnTensor(base + 32, 4, 0, 32)), b"overlaps g"), ((wide[0], apart, wide[1]), b"overlaps g"),
                       ((x, apart, x, 4096, 4096), b"dgamma and dbeta"), ((x, apart, x, 4096, 4096 + 31 * 4), b"dgamma and dbeta")):
        rc, error = backward(*args)
        assert rc == 1 and word in error, (args, error)


def test_sizes_that_no_launch_takes_are_refused():
    """A launch holds less than 2^32 threads."""
    from dnanet_amd import hip
    row = (hip.DnAdamwTensor * 1)(hip.DnAdamwTensor(4096, 4096, (1 << 34) + 1, 0, 0.0, 0, 0, 0))
    assert hip.lib.dn_adamw_step(row, 1, 4096, 4096, None, None, 32, 1e-3, 0.9, 0.999, 1e-8, 1, 0, None, 0, None) == 1
    assert hip.lib.dn_grad_norm_workspace_bytes(row, 1) == -1
    # one group of 2048 channels over 5 x 4096 points is more than a cluster of blocks: the form of three launches, 2^24 blocks
    x, a = hip.DnTensor(1 << 20, 128, 0, 2048), hip.DnTensor(1 << 60, 128, 0, 2048)
    assert hip.lib.dn_group_norm_act(x, a, 1 << 17, 5, 4096, 1, *[4096] * 2, 1e-5, 1, *[4096] * 5, 1 << 60, 1, None) == 1
    assert b"too many" in hip.lib.dn_last_error()


def test_adamw_entry_points_refuse():
    from dnanet_amd import hip

    def row(param=4096, grad=4096, n=8, state=0, decay=0.0, pd=0, gd=0):
        return (hip.DnAdamwTensor * 1)(hip.DnAdamwTensor(param, grad, n, state, decay, pd, gd, 0))

    def step(t, count=1, m=4096, v=4096, ms=None, vs=None, bits=32, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, number=1):
        return hip.lib.dn_adamw_step(t, count, m, v, ms, vs, bits, lr, b1, b2, eps, number, 0, None, 0, None)

    for t in (row(param=None), row(grad=None), row(n=-1), row(state=8), row(state=-256), row(pd=2), row(gd=-1), row(param=4098), row(grad=4097, gd=1),
              row(n=1 << 41)):
        assert step(t) == 1
    for kw in ({"m": None}, {"v": 4100}, {"bits": 16}, {"bits": 8}, {"b1": 1.0}, {"b2": -0.1}, {"eps": -1.0}, {"number": 0}, {"count": -1}):
        assert step(row(), **kw) == 1, kw
    assert step(row(n=0)) == 0 and step(None, count=0) == 0, "nothing to do: no launch"
    assert hip.lib.dn_grad_norm_workspace_bytes(row(n=1 << 20), 1) >= 8 * 256
    assert hip.lib.dn_grad_norm_workspace_bytes(row(grad=None), 1) == -1
    for out, norm, work, nbytes in ((None, 1.0, 4096, 1 << 20), (4096, 0.0, 4096, 1 << 20), (4096, float("nan"), 4096, 1 << 20),
                                    (4096, 1.0, None, 1 << 20), (4096, 1.0, 4096, 8), (4096, 1.0, 4100, 1 << 20)):
        assert hip.lib.dn_grad_norm(row(n=1 << 20), 1, norm, out, work, nbytes, None) == 1
    assert ctypes.sizeof(hip.DnAdamwTensor) == 48


def test_python_layer_refuses_host_tensors():
    from dnanet_amd.group_norm import group_norm_act
    from dnanet_amd.hip import DnTensor, PlaneBuffer
    from dnanet_amd.optim import HipAdamW
    with pytest.raises(ValueError, match="GPU"):
        HipAdamW([torch.zeros(4)])
    with pytest.raises(ValueError, match="device tensor"):
        PlaneBuffer.wrap(torch.zeros(1, 1, 1, 1, 8))
    with pytest.raises(TypeError, match="PlaneBuffer.ref"):
        group_norm_act(DnTensor(4096, 4, 0, 32), torch.ones(32), torch.zeros(32), 8)


def test_group_norm_net_parameter_tree(tmp_path):
    """The keys of the BatchNorm net without its statistics; checkpoints go round; what does not fit is refused."""
    from dnanet_amd.model import DNANet_UNet
    kw = dict(depth=2, kernel_size=(3, 5), num_filters=16, device="cpu")
    batch, group = DNANet_UNet(**kw), DNANet_UNet(**kw, norm="group", num_groups=4, activation="silu")
    keys = list(group._model.state_dict())
    assert keys == [k for k in batch._model.state_dict() if "running" not in k and "num_batches" not in k]
    assert group._model.flat_stats.numel() == 0 and group._model.flat_counts.numel() == 0
    group.save(tmp_path)
    other = DNANet_UNet(**kw, norm="group", num_groups=4, activation="silu")
    other.load(tmp_path)
    assert torch.equal(group._model.flat_params, other._model.flat_params)
    for bad in ({"norm": "layer"}, {"norm": "group", "num_groups": 3}, {"norm": "group", "num_groups": 0}, {"norm": "group", "activation": "gelu"},
                {"activation": "silu"}, {"norm": "group", "dtype": "bf16x3"}):
        with pytest.raises(ValueError):
            DNANet_UNet(**kw, **bad)


def test_fit_keywords():
    from dnanet_amd.model import DNANet_UNet
    m = DNANet_UNet(1, (3, 5), 8, device="cpu")
    with pytest.raises(ValueError, match="optimizer"):
        m.fit([], optimizer="sgd")
    with pytest.raises(ValueError, match="max_grad_norm"):
        m.fit([], max_grad_norm=1.0)
    with pytest.raises(ValueError, match="GPU"):
        m.fit([], optimizer="adamw")


def test_configuration_files():
    from dnanet_amd.config_io import load_config, load_training_config
    model = load_config(os.path.join(ROOT, "config", "models", "unet_groupnorm.yaml"))["model"]
    assert model["norm"] == "group" and model["num_filters"] % model["num_groups"] == 0
    training = load_training_config(os.path.join(ROOT, "config", "training", "segmentation_adamw.yaml"))
    assert training["optimizer"] == "adamw" and training["max_grad_norm"] > 0
