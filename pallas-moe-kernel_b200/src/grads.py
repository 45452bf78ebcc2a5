"""Global gradient norm and clipping over a list of tensors.

The expert MLP's backward (``train.py``) leaves f32 or bf16 gradients of every
expert; before the optimizer step they are scaled, together with the rest of
the model's, to a largest norm:

    norm = clip_grad_norm([w_up.grad, w_down.grad, ...], 1.0)

    norm = grad_norm(grads)                        # the two halves, to reduce the
    dist.all_reduce(...)                           # norm over ranks in between
    clip_grads(grads, 1.0, norm)

The reference is forward-only and has no counterpart.  One call takes the
whole list (one kernel for the norm and one for the scaling per 500 tensors),
is stream-ordered on the current stream and never synchronises the host: the
norm comes back as a device scalar.
"""

from __future__ import annotations

import math
from typing import Optional, Sequence

import torch

from . import _lib

__all__ = ["grad_norm", "clip_grads", "clip_grad_norm"]

_NORMS = {1.0: _lib.MOE_NORM_L1, 2.0: _lib.MOE_NORM_L2, math.inf: _lib.MOE_NORM_INF}


def _norm_code(norm_type) -> int:
    code = _NORMS.get(float(norm_type))
    if code is None:
        raise ValueError(f"norm_type {norm_type} (1, 2 or inf)")
    return code


def grad_norm(grads: Sequence[torch.Tensor], norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all tensors taken as one vector, a float32 scalar on their
    device: 2-norm, 1-norm or the largest absolute value (``math.inf``).

    float32, bfloat16 and float16 tensors of one CUDA device, of any size
    (empty ones count nothing); dense in any order of their dimensions, or
    equally spaced rows (a slice of the last dimension).  NaN and infinite
    elements come through.  An empty list has norm 0 (on the current device)."""
    return _lib.native().grad_norm(grads, _norm_code(norm_type))


def clip_grad_norm(grads: Sequence[torch.Tensor], max_norm: float, norm_type: float = 2.0, *,
                   out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Scales the tensors by ``min(1, max_norm / (norm + 1e-6))`` and returns
    the norm they had (see :func:`grad_norm`).

    In place, or into ``out``: tensors of the same shapes, of any of the three
    types (one rounding from the f32 product).  An output that shares memory
    with another output or with a gradient is refused (slices of one matrix
    that interleave are not).  In place nothing is written where the factor is
    1.  A NaN norm makes every result NaN, as the product says; check the
    returned norm to skip such a step."""
    return _lib.native().clip(grads, max_norm, _norm_code(norm_type), None, out)


def clip_grads(grads: Sequence[torch.Tensor], max_norm: float, total_norm: torch.Tensor, *,
               out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """The scaling of :func:`clip_grad_norm` with a norm known already (a
    float32 device scalar, reduced over ranks, say); returns it."""
    return _lib.native().clip(grads, max_norm, _lib.MOE_NORM_L2, total_norm, out)
