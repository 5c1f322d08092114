"""SodAdamW — AdamW over many tensors at once, with the moments in 32 or in 8
bits: one launch over every parameter of every type (csrc/adamw.hip).  The
same contract as SodSGD: fp32 masters of 16-bit parameters, the gradient
average and the loss-scale unscale folded in as ``grad_scale``, a device
multiplier that skips the step at 0, a device learning rate for captured steps.

The step, t counting a parameter's steps from one, in float32 with every
operation rounded by itself:

    g = float(grad) * (grad_scale * scale_t)
    m = b1*m + (1-b1)*g              v = b2*v + ((1-b2)*g)*g
    w = w*(1-lr*wd) - (lr/(1-b1^t)) * (m / (sqrt(v)*(1/sqrt(1-b2^t)) + eps))

Moments in 8 bits cost 2.03 bytes an element in place of 8.  A tensor is cut
into blocks of 256 elements in the order of its storage, each with two float32
scales, its largest |m| and its largest r = sqrt(v); m is a sign and 7 bits, 8
steps an octave, r 8 bits, 16 steps an octave, both over 15.9 octaves below
the scale.  Codes are rounded stochastically, by a hash of ``seed``, step,
tensor and element: a run repeats itself, and all ranks agree.

CPU path: ops.reference.adamw_step / adamw8_step, the same operations.
"""

from __future__ import annotations

from types import MappingProxyType
from typing import Iterable, Mapping

import torch

from . import conv, reference
from ._backend import ext

_BLOCK = 256  # elements of an 8-bit block (must match csrc/adamw.hip)
_NONE = torch.Tensor()
_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _padded(n: int) -> int:
    return -(-n // _BLOCK) * _BLOCK


def _in_storage(t: torch.Tensor) -> torch.Tensor:
    """The elements of a dense tensor in the order of its storage."""
    return t.as_strided((t.numel(),), (1,))


def _dense(t: torch.Tensor) -> bool:
    """Every element of one stretch of storage, each once."""
    if t.numel() == 0:
        return True
    want = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape)
                               if sz != 1):
        if stride != want:
            return False
        want *= size
    return True


def _order(t: torch.Tensor) -> "tuple[int, ...]":
    """The strides that matter."""
    return tuple(st if sz > 1 else 0 for st, sz in zip(t.stride(), t.shape))


def _checked(betas, eps) -> "tuple[tuple[float, float], float]":
    b1, b2 = betas
    if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
        raise ValueError(f"betas must lie in [0, 1), got {betas}")
    # as the step has it: a zero would make 0/0 of moments that are zero
    if not torch.tensor(float(eps), dtype=torch.float32) > 0.0:
        raise ValueError(f"eps must be positive in float32, got {eps}")
    return (float(b1), float(b2)), float(eps)


def _check_step(step) -> None:
    if step < 0 or step >= 2 ** 31 - 1:
        raise ValueError(f"step must lie in [0, 2^31 - 1), got {step}")


class SodAdamW:
    """``param_groups``: dicts ``{"params": [...], "weight_decay": float}``, the
    decay defaulting to ``weight_decay``.  ``state_bits``: 32 or 8.

    The states lie in flat tensors, every parameter's at a multiple of 256
    elements (the gaps are zero), in the groups' order: ``master`` (float32,
    the 16-bit parameters'; a float32 parameter is its own master) and, with
    32 bits, ``exp_avg`` and ``exp_avg_sq``, with 8 ``code_m``, ``code_r`` and
    ``scales`` [blocks, 2].  ``state[p]`` has the same memory cut into
    parameters.  They may be written in place, not replaced.

    A parameter whose gradient is None is left alone, its step count too.  A
    gradient that is not finite, or whose square is not, makes its block's
    moments not finite where they are held in 8 bits; ``ops.grad_norm`` gives
    the multiplier that skips such a step.

    A step may be captured into a graph; ``betas``, ``eps``, ``seed`` and host
    values of ``lr`` and ``grad_scale`` are then the capture's, the states, step
    counts and device scalars what they are at each replay.  Decay is too, once
    ``update_decay`` has handed a change of the groups' ``weight_decay`` over; an
    eager step does that by itself, one in a capture refuses."""

    def __init__(self, param_groups, betas: "tuple[float, float]" = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2,
                 state_bits: int = 32, seed: int = 0):
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits must be 32 or 8, got {state_bits}")
        self.betas, self.eps = _checked(betas, eps)
        self.state_bits = state_bits
        self.seed = int(seed) & 0xFFFFFFFF
        self.groups = []
        for g in param_groups:
            params = [p for p in g["params"] if p.requires_grad]
            self.groups.append({"params": params,
                                "weight_decay": float(g.get("weight_decay", weight_decay))})
        self._params = [p for g in self.groups for p in g["params"]]
        if len({id(p) for p in self._params}) != len(self._params):
            raise ValueError("a parameter appears twice")
        for p in self._params:
            if p.dtype not in _DTYPES:
                raise ValueError(f"parameters must be float32, bfloat16 or "
                                 f"float16, got {p.dtype}")
            if p.device != self._params[0].device:
                raise ValueError("parameters must be on one device")
            if not _dense(p):
                raise ValueError("parameters must be dense and without "
                                 f"overlaps, got strides {p.stride()} of {tuple(p.shape)}")
        self._looked_at = None
        self._check_apart(ValueError)
        self._shapes = [p.shape for p in self._params]
        self._orders = [_order(p) for p in self._params]
        self._dtypes = [p.dtype for p in self._params]
        self._grad_src = None
        self._allocate()
        self._make_plan()

    def _check_apart(self, error) -> None:
        """Where no parameter moved since the last look, nothing is done."""
        at = [p.data_ptr() for p in self._params]
        if at == self._looked_at:
            return
        spans = sorted((a, a + p.numel() * p.element_size())
                       for a, p in zip(at, self._params) if p.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise error("parameters overlap in memory")
        self._looked_at = at

    def _allocate(self) -> None:
        dev = self._params[0].device if self._params else torch.device("cpu")
        places = sum(_padded(p.numel()) for p in self._params)
        mplaces = sum(_padded(p.numel()) for p in self._params
                      if p.dtype != torch.float32)

        def zeros(n, dtype=torch.float32):
            return torch.zeros(n, dtype=dtype, device=dev)

        self._master = zeros(mplaces)
        if self.state_bits == 32:
            self._moments = [zeros(places), zeros(places)]
        else:
            self._moments = [zeros(places, torch.uint8),
                             zeros(places, torch.uint8),
                             zeros((places // _BLOCK, 2))]
        self.state: dict[torch.nn.Parameter, dict] = {}
        self._offsets, self._master_offsets, self._steps = [], [], []
        at = mat = 0
        masters, rounded = [], []
        for p in self._params:
            n, pad = p.numel(), _padded(p.numel())
            st = {}
            if p.dtype != torch.float32:
                st["master"] = self._master.as_strided(p.shape, p.stride(), mat)
                masters.append(st["master"])
                rounded.append(p.detach())
            if self.state_bits == 32:
                for k, f in zip(("exp_avg", "exp_avg_sq"), self._moments):
                    st[k] = f.as_strided(p.shape, p.stride(), at)
            else:
                for k, f in zip(("code_m", "code_r"), self._moments):
                    st[k] = f[at:at + pad]
                st["scales"] = self._moments[2][at // _BLOCK:(at + pad) // _BLOCK]
            self.state[p] = st
            self._offsets.append(at)
            self._master_offsets.append(mat if p.dtype != torch.float32 else -1)
            self._steps.append(0)           # CPU path; the GPU has its own
            at += pad
            mat += pad if p.dtype != torch.float32 else 0
        if masters:
            torch._foreach_copy_(masters, rounded)

    # -- flat states ---------------------------------------------------------
    @property
    def master(self) -> torch.Tensor:
        return self._master

    def _flat(self, bits: int, k: int) -> torch.Tensor:
        if self.state_bits != bits:
            raise AttributeError(f"the moments are held in {self.state_bits} bits")
        return self._moments[k]

    @property
    def exp_avg(self) -> torch.Tensor:
        return self._flat(32, 0)

    @property
    def exp_avg_sq(self) -> torch.Tensor:
        return self._flat(32, 1)

    @property
    def code_m(self) -> torch.Tensor:
        return self._flat(8, 0)

    @property
    def code_r(self) -> torch.Tensor:
        return self._flat(8, 1)

    @property
    def scales(self) -> torch.Tensor:
        return self._flat(8, 2)

    def moments(self) -> "tuple[torch.Tensor, torch.Tensor]":
        """The flat first and second moments: the float32 states themselves,
        or the values that the 8-bit codes stand for, in new bfloat16 tensors."""
        if self.state_bits == 32:
            return self._moments[0], self._moments[1]
        if self._master.is_cuda:
            m, v = ext().adamw8_decode(*self._moments)
            return m, v
        m, r = reference.adamw8_decode(*self._moments)
        return m.bfloat16(), (r * r).bfloat16()

    # -- gradients read elsewhere than in .grad ------------------------------
    # deferred-grad mode (reducer.defer): .grad is a fresh autograd tensor each
    # step, and the reducer's gather lands it in the stable bucket views given
    # here.  Without them a gradient that moved is seen, at the price of a new
    # table in front of the step.
    # What is given is taken as it is now; to change it, give another.
    @property
    def grad_src(self) -> "Mapping[torch.nn.Parameter, torch.Tensor] | None":
        return self._grad_src

    @grad_src.setter
    def grad_src(self, views) -> None:
        self._grad_src = None if views is None else MappingProxyType(dict(views))
        if self._plan is not None:
            views = views or {}
            self._plan.set_grads([views.get(p, _NONE) for p in self._params])

    def _decay(self) -> "list[float]":
        return [g["weight_decay"] for g in self.groups for _ in g["params"]]

    def _make_plan(self) -> None:
        """The kernel's tables, on the GPU: made ahead of the first step, which
        may be a captured one."""
        self._plan = None
        if self._params and self._params[0].is_cuda:
            self._plan = ext().AdamWPlan(self._params, self._decay(),
                                         self._offsets, self._master_offsets,
                                         self._master, self._moments)
            self._plan_wd = [g["weight_decay"] for g in self.groups]
            self._plan.set_steps(self._steps)
            self.grad_src = self._grad_src

    def update_decay(self) -> None:
        """Hand the groups' ``weight_decay`` to the device, where it changed:
        replays of a captured step go by it from here on, in the order of the
        current stream.  Not in a capture."""
        if self._plan is None:
            return
        wd = [g["weight_decay"] for g in self.groups]
        if wd != self._plan_wd:
            self._plan.set_decay(self._decay())
            self._plan_wd = wd

    def step(self, lr, grad_scale: float = 1.0,
             scale_t: "torch.Tensor | None" = None) -> None:
        """``lr`` and ``scale_t`` as in ``SodSGD.step``: ``scale_t``, a float32
        scalar on the parameters' device, is multiplied into ``grad_scale``
        and skips the whole step where it is 0; ``lr`` may be a device float32
        scalar, which a captured step reads anew on each replay."""
        if isinstance(lr, torch.Tensor) and lr.numel() != 1:
            raise RuntimeError(f"lr must be a scalar, got {tuple(lr.shape)}")
        if scale_t is not None and scale_t.numel() != 1:
            raise RuntimeError(f"scale_t must be a scalar, got {tuple(scale_t.shape)}")
        if not self._params:
            return
        if self._params[0].device != self._master.device:
            raise RuntimeError("the parameters have moved to another device "
                               "since the optimizer was made")
        if self._plan is None:
            self._step_cpu(lr, grad_scale, scale_t)
            return
        if [g["weight_decay"] for g in self.groups] != self._plan_wd:
            self.update_decay()
        lr_t = _NONE
        if isinstance(lr, torch.Tensor):
            if lr.is_cuda:
                lr, lr_t = 0.0, lr
            else:
                lr = float(lr)
        self._plan.step(lr, lr_t, *self.betas, self.eps, grad_scale,
                        _NONE if scale_t is None else scale_t, self.seed)
        # weights just changed: re-transpose every cached dgrad w_t in
        # one launch (sodkit/ops/conv.py _WtCache)
        conv._WtCache.refresh()

    @torch.no_grad()
    def _step_cpu(self, lr, grad_scale, scale_t) -> None:
        gs = torch.tensor(float(grad_scale))
        if scale_t is not None:
            if float(scale_t) == 0.0:
                return
            gs = gs * scale_t.to("cpu", torch.float32)
        grads = []
        for k, p in enumerate(self._params):
            grad = (self._grad_src or {}).get(p)
            grad = p.grad if grad is None else grad
            grads.append(grad)
            if (p.shape != self._shapes[k] or _order(p) != self._orders[k]
                    or p.dtype != self._dtypes[k]):
                raise RuntimeError(f"parameter {k} has changed its size, type or "
                                   f"layout since the optimizer was made")
            if grad is not None and (
                    grad.layout != torch.strided or grad.shape != p.shape
                    or grad.dtype not in _DTYPES or grad.device != p.device):
                raise RuntimeError(
                    f"the gradient of parameter {k} must be dense, of its "
                    f"size, on its device and float32, bfloat16 or float16")
        self._check_apart(RuntimeError)
        for k, (p, grad, wd) in enumerate(zip(self._params, grads, self._decay())):
            if grad is None or p.numel() == 0:
                continue
            grad = torch.empty_strided(p.shape, p.stride(), dtype=grad.dtype).copy_(grad)
            self._steps[k] += 1
            st = self.state[p]
            w = _in_storage(st["master"] if "master" in st else p.data)
            args = (float(lr), self._steps[k], self.betas, self.eps, wd, gs)
            if self.state_bits == 32:
                reference.adamw_step(_in_storage(p.data), _in_storage(grad), w,
                                     _in_storage(st["exp_avg"]),
                                     _in_storage(st["exp_avg_sq"]), *args)
            else:
                reference.adamw8_step(_in_storage(p.data), _in_storage(grad), w,
                                      st["code_m"], st["code_r"], st["scales"],
                                      *args, self.seed, k)

    def set_step(self, step: int) -> None:
        """Set every parameter's count of steps taken."""
        _check_step(step)
        self._steps = [int(step)] * len(self._params)
        if self._plan is not None:
            self._plan.set_steps(self._steps)

    # -- checkpointing (bitwise resume of optimizer state) -------------------
    def state_dict(self) -> dict:
        """References to the states, and each parameter's step count (which
        waits for the GPU)."""
        if self._plan is not None:
            self._steps = self._plan.get_steps()
        flat = [{**self.state[p], "step": t, "order": _order(p)}
                for p, t in zip(self._params, self._steps)]
        return {"kind": "adamw", "state_bits": self.state_bits,
                "betas": self.betas, "eps": self.eps, "seed": self.seed,
                "param_state": flat,
                "group_wd": [g["weight_decay"] for g in self.groups]}

    def load_state_dict(self, sd: dict) -> None:
        if sd.get("kind") != "adamw" or sd["state_bits"] != self.state_bits:
            raise ValueError(
                f"checkpoint holds the states of {sd.get('kind', 'sgd')}"
                + (f" in {sd['state_bits']} bits" if "state_bits" in sd else "")
                + f", not of adamw in {self.state_bits} bits")
        betas, eps = _checked(sd["betas"], sd["eps"])
        saved = sd["param_state"]
        if len(saved) != len(self._params) or len(sd["group_wd"]) != len(self.groups):
            raise ValueError(f"checkpoint holds {len(saved)} parameters in "
                             f"{len(sd['group_wd'])} groups, the optimizer "
                             f"{len(self._params)} in {len(self.groups)}")
        for k, (p, st) in enumerate(zip(self._params, saved)):
            mine = self.state[p]
            if set(st) - {"step", "order"} != set(mine) or any(
                    st[n].shape != mine[n].shape for n in mine):
                raise ValueError(f"checkpoint's state of parameter {k} does "
                                 f"not fit it")
            # codes lie in the order of the parameter's storage
            if self.state_bits == 8 and tuple(st["order"]) != _order(p):
                raise ValueError(f"checkpoint's 8-bit state of parameter {k} is "
                                 f"of another memory layout")
            _check_step(st["step"])
        self.betas, self.eps = betas, eps
        self.seed = int(sd["seed"]) & 0xFFFFFFFF
        for p, st in zip(self._params, saved):
            for n, t in self.state[p].items():
                t.copy_(st[n])
        self._steps = [int(st["step"]) for st in saved]
        for g, wd in zip(self.groups, sd["group_wd"]):
            g["weight_decay"] = wd
        if self._plan is not None:      # in place: captured steps live on
            self._plan.set_decay(self._decay())
            self._plan_wd = [g["weight_decay"] for g in self.groups]
            self._plan.set_steps(self._steps)

    def params(self) -> Iterable[torch.nn.Parameter]:
        for g in self.groups:
            yield from g["params"]
