"""A group-norm workspace over the turn of its 32-bit epoch: every launch normalises with its own sums.

The workspace's first word is the epoch, 0 at first.  Results are compared bit by bit with those of a fresh workspace."""
import pytest
import torch

from test_group_norm_gpu import EPS, make

pytestmark = pytest.mark.gpu
WIDE, NARROW = (4, 32, 8, 5, 1024), (2, 64, 4, 5, 520)          # clusters of several blocks
TOP = (1 << 32) - 1


def epoch(ws, value=None):
    word = ws[:4].view(torch.int32)
    if value is not None:
        word.fill_(value - (1 << 32) if value >> 31 else value)
    return int(word.item()) & TOP


def passes(shape, dtype, ws, seed):
    """Forward and backward on inputs of ``seed``: one launch each that publishes words."""
    from dnanet_amd.group_norm import group_norm_act, group_norm_act_backward
    buf, _, gamma, beta = make(shape, dtype, seed=seed, offset=3.0)
    c, gamma = shape[1], gamma.cuda()
    kw = {} if ws is None else {"workspace": ws}
    a, stats = group_norm_act(buf.ref(c), gamma, beta.cuda(), shape[2], EPS, "silu", **kw)
    dx, dgamma, dbeta = group_norm_act_backward(a.ref(c), buf.ref(c), gamma, stats, **kw)
    return [x.cpu() for x in (a.data, stats.mean, stats.rstd, stats.scale, stats.shift, dx.data, dgamma, dbeta)]


def workspace(shape, dtype):
    from dnanet_amd import hip
    n, c, groups, h, w = shape
    return torch.zeros(hip.lib.dn_group_norm_workspace_bytes(n, c, h, w, groups, hip.BF16 if dtype == "bf16" else hip.F32),
                       dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_launches_around_the_turn(gpu_device, dtype):
    ws = workspace(WIDE, dtype)
    epoch(ws, TOP - 4)
    seen = []
    for seed in range(4):
        got, want = passes(WIDE, dtype, ws, seed), passes(WIDE, dtype, None, seed)
        assert all(torch.equal(x, y) for x, y in zip(got, want)), seed
        seen.append(epoch(ws))
    assert seen == [TOP - 2, 0, 2, 4], "two launches a round; tag 2^32 - 1 is the last one, the epoch after it is 0"


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_words_of_the_turn_before(gpu_device, dtype):
    """Words that a wide launch left with the first tags are not there any more when these tags come again."""
    ws = workspace(WIDE, dtype)
    passes(WIDE, dtype, ws, 0)
    assert epoch(ws) == 2
    epoch(ws, TOP - 2)
    passes(NARROW, dtype, ws, 1)
    assert epoch(ws) == 0
    for seed in (2, 3):
        got, want = passes(WIDE, dtype, ws, seed), passes(WIDE, dtype, None, seed)
        assert all(torch.equal(x, y) for x, y in zip(got, want)), seed
    assert epoch(ws) == 4


# byte offsets in a workspace: the count of listed places, the list
LISTED, LIST = 2 * 32 * 4, (3 + 16) * 32 * 4 + 16384 * 4 + 4096 * 4


@pytest.mark.parametrize("place,tag", [(0xFFFFFFF0, 0), (1 << 20, 0), (0, 0), (0, 1)])
def test_list_that_no_block_wrote(gpu_device, place, tag):
    """A list with a place outside the grid, with one that is done already, with one of another launch: all segments are right, the list
    is empty afterwards and the epoch is the next."""
    from dnanet_amd.group_norm import group_norm_act
    ws = workspace(WIDE, "bf16")
    for launch in range(3):
        buf, _, gamma, beta = make(WIDE, "bf16", seed=launch, offset=3.0)
        args = gamma.cuda(), beta.cuda(), WIDE[2], EPS, "relu"
        want, _ = group_norm_act(buf.ref(WIDE[1]), *args)
        if launch == 1:
            ws[LISTED:LISTED + 4].view(torch.int32).fill_(2)
            words = ws[LIST:LIST + 16].view(torch.int32)
            words.copy_(torch.tensor([place - (1 << 32) if place >> 31 else place, epoch(ws) + 1 + tag, 1, epoch(ws) + 1], dtype=torch.int32))
        got, _ = group_norm_act(buf.ref(WIDE[1]), *args, workspace=ws)
        assert torch.equal(got.data, want.data), launch
        assert epoch(ws) == launch + 1 and not ws[LISTED:LISTED + 4].any()
