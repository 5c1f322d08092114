"""Global gradient norm over many tensors at once, and from it the multiplier
of the optimizer's step: clipping, the dynamic loss scale and the skip of a
step whose gradients overflowed.  GPU: csrc/gradnorm.hip, nothing of it goes
through the host.  CPU: ops.reference.grad_norm."""

from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import reference
from ._backend import ext

_NONE = torch.Tensor()


def grad_norm(grads: Sequence[torch.Tensor], prescale: float = 1.0,
              max_norm: float = 0.0,
              loss_scale: Optional[torch.Tensor] = None,
              good_steps: Optional[torch.Tensor] = None,
              skips: Optional[torch.Tensor] = None,
              growth_interval: int = 500
              ) -> "tuple[torch.Tensor, torch.Tensor]":
    """``(norm, mult)``, float32 scalars on the gradients' device:

        norm = prescale * sqrt(sum of all squares) / loss_scale
        mult = min(1, max_norm / (norm + 1e-6)) / loss_scale

    ``mult`` is what ``SodSGD.step`` / ``SodAdamW.step`` take as ``scale_t``;
    it is 0 (skip the step) where the norm is infinite or NaN, and only there.
    ``max_norm`` 0 does not clip.  ``loss_scale``: a float32 scalar tensor, the
    scale that the gradients still carry.  With ``good_steps`` and ``skips``
    (float32 scalar tensors) the three are moved in place as a dynamic loss
    scale: halved, not below 1, after an overflow, which ``skips`` counts, and
    doubled, not above 65536, after ``growth_interval`` finite steps in a row;
    ``mult`` is of the scale before.

    Gradients may be float32, bfloat16 and float16, mixed, with any strides,
    on one device.  The sum is held in 64 bits, and how it is grouped goes by the
    sizes and by which gradients are neighbours in one storage, not by
    addresses: a repeated call, and every rank, gets the same bits."""
    if not isinstance(grads, list):
        grads = list(grads)
    if not grads:
        raise ValueError("grad_norm needs at least one gradient")
    if (good_steps is None) != (skips is None) or (
            good_steps is not None and loss_scale is None):
        raise ValueError("good_steps and skips come together, and with a "
                         "loss_scale")
    if growth_interval < 1:
        raise ValueError(f"growth_interval must be positive, got {growth_interval}")
    if loss_scale is not None:
        for t in (loss_scale, good_steps, skips):
            if t is not None and t.numel() != 1:
                raise ValueError(f"loss_scale, good_steps and skips must be a "
                                 f"scalar each, got {tuple(t.shape)}")
    if grads[0].is_cuda:
        norm, mult = ext().grad_norm(
            grads, prescale, max_norm,
            _NONE if loss_scale is None else loss_scale,
            _NONE if good_steps is None else good_steps,
            _NONE if skips is None else skips, growth_interval)
        return norm, mult
    return reference.grad_norm(grads, prescale, max_norm, loss_scale,
                               good_steps, skips, growth_interval)
