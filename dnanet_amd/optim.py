"""``HipAdamW``: AdamW (decoupled weight decay) over many tensors in one launch, moments in fp32 or in 8 bits.

Stands beside ``HipAdam`` (``unet.py``), which is the reference's ``torch.optim.Adam`` with coupled L2
(``trainable_unet.py:155-157``); AdamW has no counterpart there.  It takes a ``HipUNet`` or any list of fp32 / bf16 device
tensors with gradients, and optionally clips the gradients to a global norm, which stays on the device.
"""
from __future__ import annotations

import ctypes
from contextlib import nullcontext
from operator import attrgetter
from typing import Iterable, List, Optional, Sequence, Union

import torch

from . import hip
from ._layout import layout as _layout      # built from csrc/tensor_layout.cpp
from .hip import BF16, F32, DnAdamwTensor
from .params import ParameterTree

_DTYPE = {torch.float32: F32, torch.bfloat16: BF16}
_BLOCK = 256                     # elements of an 8-bit state block; a tensor's moments start at a multiple of it

_grad = attrgetter("grad")
# torch.cuda.is_current_stream_capturing / current_device without their checks for a driver: 0.6 us of a call of 13
_capturing, _current_device = torch._C._cuda_isCurrentStreamCapturing, torch._C._cuda_getDevice
_HERE = nullcontext()


def _blocks(n: int) -> int:
    return (n + _BLOCK - 1) // _BLOCK


class HipAdamW:
    """``torch.optim.AdamW`` semantics for tensors on one MI355X.

    ``params``: a ``HipUNet`` (its weights are decayed, biases and norm vectors are not; ``step`` also zeroes the gradient
    arena, as ``HipAdam``), a sequence of tensors, or a sequence of ``{"params": [...], "lr": ..., "weight_decay": ...}``
    groups.  Gradients are the tensors' ``.grad``, or a group's own list ``"grads"`` (fp32 accumulators of bf16 parameters,
    say).  Tensors without a gradient are left out of a step.

    ``state_bits``: 32 (fp32 moments) or 8 (e4m3 codes with a power-of-two scale per 256 elements, stochastic rounding from
    ``seed``, the step number, a tensor's place among the parameters and an element's in its tensor: the same run gives the same
    bits).  The moments of all tensors lie in the flat buffers
    ``exp_avg`` / ``exp_avg_sq``, in the order of the parameters, each tensor from a multiple of 256 elements on; with 8 bits
    they are ``float8_e4m3fn`` and belong to the per-block scales ``exp_avg_scale`` / ``exp_avg_sq_scale``.

    ``max_grad_norm``: scale the gradients by ``min(1, max_grad_norm / (norm + 1e-6))`` of their common 2-norm, which is
    left in ``grad_norm`` (a device scalar); the gradients themselves are not rewritten.  It may be set, changed and taken back (None)
    between steps."""

    def __init__(self, params: Union[ParameterTree, Iterable], lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, state_bits: int = 32, max_grad_norm: Optional[float] = None, seed: int = 0):
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits must be 32 or 8, got {state_bits!r}")
        if not 0 <= int(seed) < 1 << 32:
            raise ValueError(f"seed must fit 32 bits, got {seed!r}")
        self.model = params if isinstance(params, ParameterTree) else None
        if self.model is not None:
            named = [(key, self.model.tensor(key)) for key, _, kind in self.model.spec if kind == "param"]
            weights, vectors = ([key for key, t in named if (t.dim() == 4) is want] for want in (True, False))
            groups = [{"params": [self.model.tensor(key) for key in weights], "grads": [self.model.grad(key) for key in weights]},
                      {"params": [self.model.tensor(key) for key in vectors], "grads": [self.model.grad(key) for key in vectors],
                       "weight_decay": 0.0}]
        else:
            groups = list(params)
            if groups and not isinstance(groups[0], dict):
                groups = [{"params": groups}]
        self.param_groups: List[dict] = []
        self._given: List[Optional[torch.Tensor]] = []       # a parameter's own gradient tensor, None: its .grad
        for g in groups:
            unknown = set(g) - {"params", "grads", "lr", "betas", "eps", "weight_decay"}
            if unknown:
                raise ValueError(f"unknown keys in a parameter group: {sorted(unknown)}")
            group = {"params": list(g["params"]), "lr": g.get("lr", lr), "betas": tuple(g.get("betas", betas)), "eps": g.get("eps", eps),
                     "weight_decay": g.get("weight_decay", weight_decay)}
            if not (len(group["betas"]) == 2 and all(0 <= b < 1 for b in group["betas"]) and group["eps"] >= 0 and group["lr"] >= 0
                    and group["weight_decay"] >= 0):
                raise ValueError(f"bad hyper-parameters: lr {group['lr']}, betas {group['betas']}, eps {group['eps']}, "
                                 f"weight_decay {group['weight_decay']}")
            given = list(g.get("grads", [None] * len(group["params"])))
            if len(given) != len(group["params"]):
                raise ValueError(f"{len(given)} gradients for {len(group['params'])} parameters")
            self._given += given
            self.param_groups.append(group)
        self._all_given, self._none_given = all(g is not None for g in self._given), all(g is None for g in self._given)
        self._params: List[torch.Tensor] = [p for g in self.param_groups for p in g["params"]]
        if not self._params:
            raise ValueError("no parameters")
        self.device = getattr(self._params[0], "device", None)
        self._check_params()
        self.state_bits, self.seed = state_bits, int(seed)
        self.step_count = 0
        self._zeroed = False
        self._sizes = [p.numel() for p in self._params]
        self.offsets, at = [], 0                 # element at which a tensor's moments start
        for n in self._sizes:
            self.offsets.append(at)
            at += _blocks(n) * _BLOCK
        if state_bits == 32:
            self.exp_avg, self.exp_avg_sq = (torch.zeros(at, dtype=torch.float32, device=self.device) for _ in range(2))
        else:                                    # code 0 is 0.0
            self.exp_avg, self.exp_avg_sq = (torch.zeros(at, dtype=torch.uint8, device=self.device).view(torch.float8_e4m3fn) for _ in range(2))
        self.exp_avg_scale = self.exp_avg_sq_scale = None
        if state_bits == 8:
            self.exp_avg_scale, self.exp_avg_sq_scale = (torch.zeros(at // _BLOCK, dtype=torch.float32, device=self.device) for _ in range(2))
        self._clip = self._partial = None
        self.max_grad_norm = max_grad_norm
        self._made_for: tuple = ()               # layouts and decays that the table below was made for
        self._decays: List[float] = []
        self._table, self._slices = None, []

    @property
    def max_grad_norm(self) -> Optional[float]:
        return self._max_grad_norm

    @max_grad_norm.setter
    def max_grad_norm(self, value: Optional[float]):
        if value is not None and not value > 0:
            raise ValueError(f"max_grad_norm must be above zero, got {value!r}")
        if value is not None and self._clip is None:         # kept from then on: a captured step may hold them
            # sizes count here, pointers only have to be some
            whole = (DnAdamwTensor * len(self._params))(*[DnAdamwTensor(4096, 4096, n, 0, 0.0, F32, F32, 0) for n in self._sizes])
            nbytes = hip.lib.dn_grad_norm_workspace_bytes(whole, len(self._params))
            if nbytes < 0:
                hip.check(1)
            self._partial = torch.empty(nbytes // 8, dtype=torch.float64, device=self.device)
            self._clip = torch.zeros(2, dtype=torch.float32, device=self.device)
        self._max_grad_norm = value
        self.grad_norm = None if value is None else self._clip[0]

    def _check_params(self):
        spans = []
        for p in self._params:
            if not isinstance(p, torch.Tensor) or p.dtype not in _DTYPE or not p.is_cuda or p.device != self.device or not p.is_contiguous():
                raise ValueError("parameters must be contiguous float32 or bfloat16 tensors on one GPU, got "
                                 + (f"{tuple(p.shape)} {p.dtype} on {p.device}" if isinstance(p, torch.Tensor) else repr(type(p))))
            if p.numel():
                spans.append((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()))
        spans.sort()
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("parameters overlap in memory (a tensor listed twice?)")

    # ---- the tensor table: rebuilt when a parameter or a gradient lies elsewhere or is of another kind, or a decay is another one
    # than last time ---------------------------------------------------------------------------------------------------------
    def _refresh(self):
        decays = [g["weight_decay"] for g in self.param_groups]
        if self._table is not None and self.model is not None and decays == self._decays:
            return                               # a model's arenas stay where they are
        if self._all_given:
            grads = self._given
        elif self._none_given:
            grads = list(map(_grad, self._params))
        else:
            grads = [p.grad if g is None else g for p, g in zip(self._params, self._given)]
        # not the addresses alone: a tensor that keeps its own can become shorter, strided or one of another type (``p.data = p.data[:k]``,
        # ``resize_``, ``set_``), and a kernel that takes it for what it was writes past its end
        made_for = _layout(self._params + grads), decays
        if made_for == self._made_for:
            return
        self._check_params()
        for p, g, n in zip(self._params, grads, self._sizes):
            if p.numel() != n:
                raise ValueError(f"a parameter of {n} elements has become one of {p.numel()}: its moments do not fit, make a new optimizer")
            if g is None:
                continue
            if g.dtype not in _DTYPE or g.device != self.device or g.shape != p.shape or not g.is_contiguous():
                raise ValueError(f"gradient {tuple(g.shape)} {g.dtype} on {g.device} of a parameter {tuple(p.shape)}: contiguous float32 or "
                                 "bfloat16 of the parameter's shape, on its device, is required")
        rows, self._slices, k = [], [], 0
        for group in self.param_groups:
            start = len(rows)
            for p in group["params"]:
                g, at, number = grads[k], self.offsets[k], k
                k += 1
                if g is not None and p.numel():
                    rows.append(DnAdamwTensor(p.data_ptr(), g.data_ptr(), p.numel(), at, group["weight_decay"], _DTYPE[p.dtype],
                                              _DTYPE[g.dtype], number))
            self._slices.append((start, len(rows) - start))
        self._table = (DnAdamwTensor * max(1, len(rows)))(*rows)
        self._rows = len(rows)
        self._written = [p for p, g in zip(self._params, grads) if g is not None]
        self._made_for, self._decays = made_for, decays

    def _part(self, start: int):
        return ctypes.cast(ctypes.byref(self._table, start * ctypes.sizeof(DnAdamwTensor)), ctypes.POINTER(DnAdamwTensor))

    def frozen_constants(self) -> tuple:
        """Everything but the learning rate and the step number that a captured step has fixed."""
        first = self.param_groups[0]["lr"]
        return (tuple((g["betas"], g["eps"], g["weight_decay"], g["lr"] == first) for g in self.param_groups), self.max_grad_norm, self.seed)

    @torch.no_grad()
    def step(self, device_state: Optional[Sequence[torch.Tensor]] = None):
        """One update from the gradients at hand, queued on the current stream.  ``device_state = (hyper, step)``: learning
        rate, bias corrections and step number are read from / kept in device memory, for a captured step (one learning rate
        for all groups)."""
        groups = self.param_groups
        first = groups[0]
        same = all(g["lr"] == first["lr"] and g["betas"] == first["betas"] and g["eps"] == first["eps"] for g in groups[1:])
        capturing = _capturing()
        if device_state is None and capturing:
            raise RuntimeError("a captured step needs device_state: learning rate and step number would be frozen into the graph")
        if device_state is not None and not same:
            raise ValueError("a step with device_state needs one learning rate, betas and eps for all groups")
        self._refresh()
        lib = hip.lib
        state = (self.exp_avg.data_ptr(), self.exp_avg_sq.data_ptr(), hip.ptr(self.exp_avg_scale), hip.ptr(self.exp_avg_sq_scale),
                 self.state_bits)
        zero = 1 if self.model is not None else 0
        guard = _HERE if self.device.index == _current_device() else torch.cuda.device(self.device)
        with guard:
            stream = hip.raw_stream(self.device)
            clip = None
            if self._max_grad_norm is not None:
                clip = self._clip.data_ptr()
                hip.check(lib.dn_grad_norm(self._table, self._rows, self._max_grad_norm, clip, self._partial.data_ptr(),
                                           self._partial.numel() * 8, stream))
            if device_state is not None:
                hyper, step = device_state
                hip.check(lib.dn_adamw_step_graph(self._table, self._rows, *state, hip.ptr(hyper), hip.ptr(step), *first["betas"], first["eps"],
                                                  self.seed, clip, zero, stream))
            else:
                for g, (start, count) in [(first, (0, self._rows))] if same else zip(groups, self._slices):
                    hip.check(lib.dn_adamw_step(self._part(start), count, *state, g["lr"], *g["betas"], g["eps"], self.step_count + 1, self.seed,
                                                clip, zero, stream))
        self.step_count += 1
        if self.model is not None:
            self.model._param_epoch += 1
            self._zeroed = True
        elif not capturing:
            torch.autograd.graph.increment_version(self._written)    # the kernel's writes are in-place updates to autograd

    def zero_grad(self, set_to_none: bool = True):
        """A model's gradient arena was zeroed by ``step`` itself; ``.grad`` tensors are dropped (or zeroed), a group's own
        ``"grads"`` zeroed."""
        if self.model is not None:
            if not self._zeroed:
                self.model.flat_grads.zero_()
            self._zeroed = False
            return
        for p, g in zip(self._params, self._given):
            if g is not None:
                g.zero_()
            elif p.grad is not None:
                if set_to_none:
                    p.grad = None
                else:
                    p.grad.detach_().zero_()

    # ---- checkpoints ---------------------------------------------------------------------------------------------------
    def state_dict(self) -> dict:
        out = {"step": self.step_count, "state_bits": self.state_bits, "seed": self.seed, "sizes": [p.numel() for p in self._params],
               "exp_avg": self.exp_avg.clone(), "exp_avg_sq": self.exp_avg_sq.clone(),
               "param_groups": [{k: v for k, v in g.items() if k != "params"} for g in self.param_groups]}
        if self.state_bits == 8:
            out["exp_avg_scale"], out["exp_avg_sq_scale"] = self.exp_avg_scale.clone(), self.exp_avg_sq_scale.clone()
        return out

    def load_state_dict(self, state: dict):
        if state["state_bits"] != self.state_bits or list(state["sizes"]) != [p.numel() for p in self._params]:
            raise ValueError("the optimizer state is of other tensors or another state_bits")
        if len(state["param_groups"]) != len(self.param_groups):
            raise ValueError(f"the optimizer state has {len(state['param_groups'])} parameter groups, this optimizer {len(self.param_groups)}")
        for name in ("exp_avg", "exp_avg_sq") + (("exp_avg_scale", "exp_avg_sq_scale") if self.state_bits == 8 else ()):
            getattr(self, name).copy_(state[name])
        self.step_count, self.seed = int(state["step"]), int(state["seed"])
        for group, saved in zip(self.param_groups, state["param_groups"]):
            group.update(saved)
            group["betas"] = tuple(group["betas"])
