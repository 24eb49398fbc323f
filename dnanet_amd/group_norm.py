"""GroupNorm with an activation on plane-record tensors: the batch-independent alternative to the BatchNorm2d + ReLU of a
``DoubleConv`` (reference ``unet_architecture.py:17,21``; a group norm has no counterpart there).

``y = act(group_norm(x))`` per image over ``groups`` groups of channels, statistics in fp32 or more, and its backward pass;
both run on the current stream of the tensors' device.  Tensors are ``PlaneBuffer.ref`` views (channels last inside 32-byte
records, see ``include/dnanet_hip.h``), the per-channel vectors fp32.
"""
from __future__ import annotations

from contextlib import nullcontext
from functools import lru_cache
from typing import Dict, Optional, Tuple

import torch

from . import hip
from .hip import DnTensor, PlaneBuffer

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2}      # DN_ACT_*


def parse_activation(activation: str) -> int:
    code = ACTIVATIONS.get(activation)
    if code is not None:
        return code
    try:
        return ACTIVATIONS[str(activation).lower()]
    except KeyError:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")


class GroupNormStats:
    """What a forward pass leaves for its backward pass: ``mean`` / ``rstd`` (N, groups), the fused ``scale`` / ``shift``
    (N, channels padded to 32), and how they were made.  The four lie one after the other in ``flat`` where a forward call
    made them, and become tensors of their own when they are asked for."""

    __slots__ = ("flat", "_parts", "_shape", "groups", "activation")

    def __init__(self, mean: torch.Tensor, rstd: torch.Tensor, scale: torch.Tensor, shift: torch.Tensor, groups: int, activation: str):
        self.flat, self._parts, self._shape = None, (mean, rstd, scale, shift), None
        self.groups, self.activation = groups, activation

    @staticmethod
    def floats(n: int, channels: int, groups: int) -> int:
        return 2 * n * (groups + hip.channel_pad(channels))

    @classmethod
    def from_flat(cls, flat: torch.Tensor, n: int, channels: int, groups: int, activation: str) -> "GroupNormStats":
        """Over ``floats(n, channels, groups)`` consecutive fp32 values."""
        self = cls.__new__(cls)
        self.flat, self._parts, self._shape = flat, None, (n, groups, hip.channel_pad(channels))
        self.groups, self.activation = groups, activation
        return self

    def _part(self, k: int) -> torch.Tensor:
        if self._parts is not None:
            return self._parts[k]
        n, groups, pad = self._shape
        flat = self.flat
        if k < 2:
            return flat.as_strided((n, groups), (groups, 1), flat.storage_offset() + k * n * groups)
        return flat.as_strided((n, pad), (pad, 1), flat.storage_offset() + n * (2 * groups + (k - 2) * pad))

    mean = property(lambda self: self._part(0))
    rstd = property(lambda self: self._part(1))
    scale = property(lambda self: self._part(2))
    shift = property(lambda self: self._part(3))

    def _spread(self, base: int) -> Tuple[int, int, int, int]:
        n, groups, pad = self._shape
        return base, base + 4 * n * groups, base + 8 * n * groups, base + 8 * n * groups + 4 * n * pad

    def _pointers(self, n: int, channels: int, groups: int, device: torch.device) -> Tuple[int, int, int, int]:
        """Device pointers of the four, checked against a call's sizes."""
        pad = hip.channel_pad(channels)
        if self._parts is None:
            if self._shape != (n, groups, pad):
                raise ValueError(f"stats.mean is of {self._shape[0]} images and {self._shape[1]} groups, the call of {n} and {groups}")
            return self._spread(_vector(self.flat, (2 * n * (groups + pad),), device, "stats.flat"))
        mean, rstd, scale, shift = self._parts
        return (_vector(mean, (n, groups), device, "stats.mean"), _vector(rstd, (n, groups), device, "stats.rstd"),
                _vector(scale, (n, pad), device, "stats.scale"), _vector(shift, (n, pad), device, "stats.shift"))


# torch.cuda.is_current_stream_capturing / current_device without their checks for a driver: 0.6 us of a call of 19
_capturing, _current_device = torch._C._cuda_isCurrentStreamCapturing, torch._C._cuda_getDevice

_workspaces: Dict[Tuple[int, int], torch.Tensor] = {}


def _workspace(device: torch.device, stream: int, nbytes: int) -> torch.Tensor:
    """Zero-filled before its first use, as the library asks.  Calls on one stream follow each other and share a workspace.  A
    call under HIP-graph capture gets one of its own inside the graph (zeroed there on every replay): two graphs captured on
    the same stream may be replayed at the same time."""
    if _capturing():
        return torch.zeros(nbytes, dtype=torch.uint8, device=device)
    ws = _workspaces.get((device.index, stream))
    if ws is None or ws.numel() < nbytes:
        ws = _workspaces[device.index, stream] = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
    return ws


_HERE = nullcontext()


def _on(device: torch.device):
    return _HERE if device.index == _current_device() else torch.cuda.device(device)


def _owner(ref: DnTensor, what: str) -> PlaneBuffer:
    buf = getattr(ref, "_owner", None)
    if not isinstance(buf, PlaneBuffer):
        raise TypeError(f"{what} must be a PlaneBuffer.ref(channels, plane0)")
    return buf


def _same(buf: PlaneBuffer, like: PlaneBuffer, what: str):
    if (buf.n, buf.h, buf.w, buf.dtype) != (like.n, like.h, like.w, like.dtype) or buf.data.device != like.data.device:
        raise ValueError(f"{what} is {(buf.n, buf.h, buf.w)} {buf.data.dtype} on {buf.data.device}, x is {(like.n, like.h, like.w)} "
                         f"{like.data.dtype} on {like.data.device}")


def _like(src: PlaneBuffer, channels: int) -> PlaneBuffer:
    """A new buffer of ``channels`` channels and the sizes of ``src``."""
    buf = PlaneBuffer.__new__(PlaneBuffer)
    buf.n, buf.planes_total, buf.h, buf.w, buf.dtype = src.n, hip.planes(channels, src.dtype), src.h, src.w, src.dtype
    buf.data = src.data.new_empty((buf.n, buf.planes_total, buf.h, buf.w, src.data.shape[4]))
    return buf


def _vector(t: torch.Tensor, shape, device, what: str) -> int:
    if t.dtype != torch.float32 or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous float32 tensor of shape {tuple(shape)} on {device}, got {tuple(t.shape)} {t.dtype} "
                         f"on {t.device}")
    return t.data_ptr()


def _given_workspace(ws: torch.Tensor, device) -> torch.Tensor:
    if ws.dtype != torch.uint8 or ws.device != device or not ws.is_contiguous():
        raise ValueError(f"workspace must be a contiguous uint8 tensor on {device}, got {ws.dtype} on {ws.device}")
    return ws


@lru_cache(maxsize=256)
def _need(n: int, channels: int, h: int, w: int, groups: int, dtype: int) -> int:
    nbytes = hip.lib.dn_group_norm_workspace_bytes(n, channels, h, w, groups, dtype)
    if nbytes < 0:
        raise ValueError(hip.lib.dn_last_error().decode())
    return nbytes


def group_norm_act(x: DnTensor, gamma: torch.Tensor, beta: torch.Tensor, groups: int, eps: float = 1e-5, activation: str = "relu",
                   out: Optional[DnTensor] = None, stats: Optional[GroupNormStats] = None, workspace: Optional[torch.Tensor] = None
                   ) -> Tuple[PlaneBuffer, GroupNormStats]:
    """``act(group_norm(x, groups, gamma, beta, eps))``.  ``out`` (default: a new buffer) may be ``x`` itself; ``stats``: where
    the statistics go (default: new tensors); ``workspace``: a caller's own (uint8, zeroed before its first use, one call at
    a time).  Returns the output's buffer and the statistics for the backward call."""
    src = _owner(x, "x")
    act, c, data = parse_activation(activation), x.channels, src.data
    n, h, w, dtype, dev = src.n, src.h, src.w, src.dtype, data.device
    need = _need(n, c, h, w, groups, dtype)
    shape = (c,)
    g, b = _vector(gamma, shape, dev, "gamma"), _vector(beta, shape, dev, "beta")
    if out is None:
        dst = _like(src, c)
        out = dst.ref(c)
    else:
        dst = _owner(out, "out")
        _same(dst, src, "out")
    if stats is None:
        stats = GroupNormStats.from_flat(gamma.new_empty(GroupNormStats.floats(n, c, groups)), n, c, groups, activation)
        vectors = stats._spread(stats.flat.data_ptr())
    else:
        vectors = stats._pointers(n, c, groups, dev)
    with _on(dev):
        stream = hip.raw_stream(dev)
        ws = _workspace(dev, stream, need) if workspace is None else _given_workspace(workspace, dev)
        hip.check(hip.lib.dn_group_norm_act(x, out, n, h, w, groups, g, b, eps, act, *vectors, ws.data_ptr(), ws.numel(), dtype, stream))
    stats.groups, stats.activation = groups, activation
    return dst, stats


def group_norm_act_backward(g: DnTensor, x: DnTensor, gamma: torch.Tensor, stats: GroupNormStats, out: Optional[DnTensor] = None,
                            dgamma: Optional[torch.Tensor] = None, dbeta: Optional[torch.Tensor] = None,
                            workspace: Optional[torch.Tensor] = None) -> Tuple[PlaneBuffer, torch.Tensor, torch.Tensor]:
    """``g`` = dL/d(output) -> (dL/dx, dL/dgamma, dL/dbeta).  ``x``, ``gamma``, ``stats``: as the forward call took and returned
    them.  ``out`` (default: a new buffer) may be ``g`` itself, not ``x``."""
    src, grad = _owner(x, "x"), _owner(g, "g")
    _same(grad, src, "g")
    c, dev, groups = x.channels, src.data.device, stats.groups
    need = _need(src.n, c, src.h, src.w, groups, src.dtype)
    ga = _vector(gamma, (c,), dev, "gamma")
    if out is None:
        dst = _like(src, c)
        out = dst.ref(c)
    else:
        dst = _owner(out, "out")
        _same(dst, src, "out")
        if dst.data.data_ptr() == src.data.data_ptr() and abs(out.plane0 - x.plane0) < hip.planes(c, src.dtype):
            raise ValueError("out must not overlap x")
    vectors = stats._pointers(src.n, c, groups, dev)
    if dgamma is None:
        dgamma = gamma.new_empty(c)
        dg = dgamma.data_ptr()
    else:
        dg = _vector(dgamma, (c,), dev, "dgamma")
    if dbeta is None:
        dbeta = gamma.new_empty(c)
        db = dbeta.data_ptr()
    else:
        db = _vector(dbeta, (c,), dev, "dbeta")
    with _on(dev):
        stream = hip.raw_stream(dev)
        ws = _workspace(dev, stream, need) if workspace is None else _given_workspace(workspace, dev)
        hip.check(hip.lib.dn_group_norm_act_backward(g, x, out, src.n, src.h, src.w, groups, ga, *vectors, parse_activation(stats.activation),
                                                     dg, db, ws.data_ptr(), ws.numel(), src.dtype, stream))
    return dst, dgamma, dbeta
