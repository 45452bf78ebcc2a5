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

import functools
import math
import operator
import struct
from array import array
from typing import Optional, Sequence

import torch

from . import _lib
from .kernel import _stream_handle, _stream_workspace
from .router import _ELEMS, _call, _scalars

__all__ = ["grad_norm", "clip_grads", "clip_grad_norm"]

_NORMS = {1.0: _lib.MOE_NORM_L1, 2.0: _lib.MOE_NORM_L2, math.inf: _lib.MOE_NORM_INF}

# moe_tensor_desc of include/moe_b200.h as 64-bit words: in, out, rows, cols,
# in_ld, out_ld, and the two element types in one.
_WORDS = 7

_ptrs = torch.Tensor.data_ptr
_numel = torch.Tensor.numel
_dense = torch.Tensor.is_contiguous
_device = torch.Tensor.get_device
_dtype = operator.attrgetter("dtype")


def _rows_of(t: torch.Tensor):
    """(rows, cols, row stride) of a tensor whose elements, in some order of
    its dimensions, are equally long contiguous rows at equal distances; None
    for other strides."""
    dims = sorted(((st, n) for st, n in zip(t.stride(), t.shape) if n > 1), reverse=True)
    cols = 1
    while dims and dims[-1][0] == cols:
        cols *= dims.pop()[1]
    if not dims:
        return 1, cols, cols
    ld = dims[-1][0]
    rows = 1
    while dims and dims[-1][0] == ld * rows:
        rows *= dims.pop()[1]
    return None if dims or ld < cols else (rows, cols, ld)


def _column(f, tensors) -> array:
    """f of every tensor as 64-bit words (array's own constructor takes twice as long from a list of ints)."""
    return array("q", struct.pack(f"{len(tensors)}q", *map(f, tensors)))


def _types(tensors) -> array:
    kinds = set(map(_dtype, tensors))
    if not kinds <= _ELEMS.keys():
        raise TypeError(f"gradients are float32, bfloat16 or float16, not {(kinds - _ELEMS.keys()).pop()}")
    if len(kinds) == 1:
        return array("q", [_ELEMS[kinds.pop()]]) * len(tensors)
    return array("q", [_ELEMS[t.dtype] for t in tensors])


def _describe(grads: Sequence[torch.Tensor], out: Optional[Sequence[torch.Tensor]]):
    """(descriptors, device) of the list; ``out`` None: the tensors themselves.
    Whole columns at a time: at hundreds of tensors this is the call's cost."""
    grads = list(grads)
    n = len(grads)
    outs = grads if out is None else list(out)
    if len(outs) != n:
        raise ValueError(f"{n} gradients and {len(outs)} outputs")
    if n == 0:
        return array("q"), None
    devices = set(map(_device, grads))
    if outs is not grads:
        devices.update(map(_device, outs))
    if len(devices) > 1 or -1 in devices:
        raise ValueError("gradients and outputs must be CUDA tensors on one device")
    d = array("q", bytes(8 * _WORDS * n))
    d[0::_WORDS] = d[1::_WORDS] = _column(_ptrs, grads)
    d[2::_WORDS] = array("q", [1]) * n
    d[3::_WORDS] = numel = _column(_numel, grads)
    types = outer = _types(grads)
    if outs is not grads:
        d[1::_WORDS] = _column(_ptrs, outs)
        outer = _types(outs)
        if numel != _column(_numel, outs):
            raise ValueError("an output has another shape than its gradient")
    if types.count(types[0]) == n == outer.count(outer[0]):
        d[6::_WORDS] = array("q", [types[0] | outer[0] << 32]) * n
    else:
        d[6::_WORDS] = array("q", [t | u << 32 for t, u in zip(types, outer)])
    if not all(map(_dense, grads)) or not (outs is grads or all(map(_dense, outs))):
        for i, (g, o) in enumerate(zip(grads, outs)):
            if not (g.is_contiguous() and o.is_contiguous()):
                d[_WORDS * i + 2:_WORDS * i + 6] = array("q", _strided(i, g, o))
    return d, grads[0].device


def _strided(i: int, g: torch.Tensor, o: torch.Tensor):
    """rows, cols and the two row strides of a pair that is not contiguous."""
    if g.shape != o.shape:
        raise ValueError(f"tensor {i}: an output of another shape than its gradient, {tuple(g.shape)}, {tuple(o.shape)}")
    # The elements' order in memory must be the same; the distance of the rows
    # may differ.
    dims = [x for x in range(g.dim()) if g.shape[x] > 1]
    rg, ro = _rows_of(g), _rows_of(o)
    if rg is not None and ro is not None and sorted(dims, key=g.stride) == sorted(dims, key=o.stride):
        if rg[0] == 1:
            rg = (ro[0], ro[1], ro[1])
        if ro[0] == 1:
            ro = (rg[0], rg[1], rg[1])
        if rg[:2] == ro[:2]:
            return rg[0], rg[1], rg[2], ro[2]
    raise ValueError(f"tensor {i}: strides {g.stride()} and {o.stride()} of shape {tuple(g.shape)} are not equally "
                     "spaced rows of one order")


def _norm_code(norm_type) -> int:
    code = _NORMS.get(float(norm_type))
    if code is None:
        raise ValueError(f"norm_type {norm_type} (1, 2 or inf)")
    return code


@functools.lru_cache(maxsize=4096)
def _space_bytes(n: int) -> int:
    return int(_lib.lib().moe_grad_norm_workspace_size(n))


def _space(dev, n: int):
    need = _space_bytes(n)
    return _stream_workspace(dev, _stream_handle(dev), need), need


def grad_norm(grads: Sequence[torch.Tensor], norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all tensors taken as one vector, a float32 scalar on their
    device: 2-norm, 1-norm or the largest absolute value (``math.inf``).

    float32, bfloat16 and float16 tensors of one CUDA device, of any size
    (empty ones count nothing); dense in any order of their dimensions, or
    equally spaced rows (a slice of the last dimension).  NaN and infinite
    elements come through.  An empty list has norm 0 (on the current device)."""
    code = _norm_code(norm_type)
    d, dev = _describe(grads, None)
    if dev is None:
        return torch.zeros((), dtype=torch.float32, device="cuda")
    norm = torch.empty_like(_scalars(dev)[1])
    ws, need = _space(dev, len(d) // _WORDS)
    _call(dev, _lib.lib().moe_grad_norm, d.buffer_info()[0], len(d) // _WORDS, code, norm.data_ptr(), ws.data_ptr(), need)
    return norm


def _clip(grads, max_norm, code, given, out):
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"max_norm {max_norm} must be at least 0")
    d, dev = _describe(grads, out)
    if dev is None:
        return given if given is not None else torch.zeros((), dtype=torch.float32, device="cuda")
    n, at = len(d) // _WORDS, d.buffer_info()[0]
    if given is not None:
        if given.device != dev or given.dtype != torch.float32 or given.numel() != 1:
            raise ValueError("total_norm must be a float32 scalar tensor on the gradients' device")
        _call(dev, _lib.lib().moe_clip_grads, at, n, code, max_norm, given.data_ptr(), None, None, 0)
        return given
    norm = torch.empty_like(_scalars(dev)[1])
    ws, need = _space(dev, len(d) // _WORDS)
    _call(dev, _lib.lib().moe_clip_grads, at, n, code, max_norm, None, norm.data_ptr(), ws.data_ptr(),
          need)
    return norm


def clip_grad_norm(grads: Sequence[torch.Tensor], max_norm: float, norm_type: float = 2.0, *,
                   out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Scales the tensors by ``min(1, max_norm / (norm + 1e-6))`` and returns
    the norm they had (see :func:`grad_norm`).

    In place, or into ``out``: tensors of the same sizes, of any of the three
    types (one rounding from the f32 product), that share no memory with the
    gradients.  In place nothing is written where the factor is 1.  A NaN norm
    makes every result NaN, as the product says; check the returned norm to
    skip such a step."""
    return _clip(grads, max_norm, _norm_code(norm_type), None, out)


def clip_grads(grads: Sequence[torch.Tensor], max_norm: float, total_norm: torch.Tensor, *,
               out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """The scaling of :func:`clip_grad_norm` with a norm known already (a
    float32 device scalar, reduced over ranks, say); returns it."""
    return _clip(grads, max_norm, _lib.MOE_NORM_L2, total_norm, out)
