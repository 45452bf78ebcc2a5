"""Routing and permutation around the fused expert MLP (torch CUDA tensors).

The reference's path starts from rows already sorted by expert plus their
``group_sizes`` (``src/kernel.py:85-95``; its benchmarks build the group
sizes directly).  These functions produce that input from router logits and
fold the expert outputs back per token, each one kernel of the library
(declared in ``include/moe_b200.h``):

    ids, w = route_topk(logits, k)                  # (T, k) experts and weights
    gs, src, inv = permute(ids, E)                  # stable sort of entries by expert
    xs = gather_rows(x, src, k)                     # X in expert order
    ys = fused_ragged_mlp(xs, w_up, w_down, gs)     # the reference's path
    y = combine_rows(ys, inv, w)                    # weighted sum per token

:func:`moe_layer` runs the five steps.  All calls are stream-ordered on the
current stream and never synchronise the host.
"""

from __future__ import annotations

import functools
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .kernel import _stream_handle, _stream_workspace


def _stream(dev) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


def route_topk(logits: torch.Tensor, k: int):
    """Top-k experts per token (larger logit first, ties to the lower expert
    id) and softmax weights over the selected logits.  ``logits`` (T, E)
    float32 on a CUDA device; returns (ids (T, k) int32, weights (T, k) f32)."""
    if not logits.is_cuda or logits.dim() != 2:
        raise ValueError("logits must be a 2-D CUDA tensor")
    logits = logits.float().contiguous()
    T, E = logits.shape
    ids = torch.empty((T, k), dtype=torch.int32, device=logits.device)
    w = torch.empty((T, k), dtype=torch.float32, device=logits.device)
    _lib.check(_lib.lib().moe_route_topk(logits.data_ptr(), T, E, k, ids.data_ptr(), w.data_ptr(),
                                         _stream(logits.device)))
    return ids, w


def permute(ids: torch.Tensor, num_experts: int, workspace: Optional[torch.Tensor] = None):
    """Stable counting sort of the entries ``i = t * k + j`` of ``ids`` (T, k)
    by expert.  Returns (group_sizes (E,), sorted_src (N,) entry index of each
    row in expert order, inverse (T, k) row of each entry, -1 if dropped)."""
    ids = ids.to(torch.int32).contiguous()
    dev = ids.device
    N = ids.numel()
    L = _lib.lib()
    gs = torch.empty(num_experts, dtype=torch.int32, device=dev)
    # Rows past sum(group_sizes), which dropped entries leave over, read as
    # entry 0: gather_rows takes every row of sorted_src.
    src = torch.zeros(N, dtype=torch.int32, device=dev)
    inv = torch.empty(ids.shape, dtype=torch.int32, device=dev)
    need = int(L.moe_permute_workspace_size(N, num_experts))
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
    _lib.check(L.moe_permute(ids.data_ptr(), N, num_experts, gs.data_ptr(), src.data_ptr(), inv.data_ptr(),
                             workspace.data_ptr(), workspace.numel(), _stream(dev)))
    return gs, src, inv


def gather_rows(x: torch.Tensor, sorted_src: torch.Tensor, k: int, out: Optional[torch.Tensor] = None):
    """Row r of the result is row ``sorted_src[r] // k`` of ``x`` (T, D)."""
    x = x.contiguous()
    rows = sorted_src.numel()
    if out is None:
        out = torch.empty((rows, x.shape[1]), dtype=x.dtype, device=x.device)
    row_bytes = x.shape[1] * x.element_size()
    _lib.check(_lib.lib().moe_gather_rows(x.data_ptr(), sorted_src.data_ptr(), rows, k, row_bytes, out.data_ptr(),
                                          _stream(x.device)))
    return out


def combine_rows(y_sorted: torch.Tensor, inverse: torch.Tensor, weights: torch.Tensor,
                 out: Optional[torch.Tensor] = None):
    """``y[t] = sum_j weights[t, j] * y_sorted[inverse[t, j]]`` (f32)."""
    T, k = inverse.shape
    D = y_sorted.shape[1]
    if out is None:
        out = torch.empty((T, D), dtype=torch.float32, device=y_sorted.device)
    _lib.check(_lib.lib().moe_combine_rows(y_sorted.contiguous().data_ptr(), inverse.contiguous().data_ptr(),
                                           weights.float().contiguous().data_ptr(), T, k, D, out.data_ptr(),
                                           _stream(y_sorted.device)))
    return out


# ----------------------------------------------------------------------------- training
class RouteTrain(NamedTuple):
    """Result of :func:`route_forward_train`."""
    ids: torch.Tensor           # (T, k) int32, -1: no expert
    weights: torch.Tensor       # (T, k) f32
    counts: torch.Tensor        # (sequences, E) int32: chosen entries per expert
    tokens: torch.Tensor        # (sequences,) int32: tokens that take part
    balance_loss: torch.Tensor  # f32 scalar
    z_loss: torch.Tensor        # f32 scalar


_ELEMS = {torch.float32: _lib.MOE_ELEM_F32, torch.bfloat16: _lib.MOE_ELEM_BF16, torch.float16: _lib.MOE_ELEM_F16}
_SCORING = {"softmax": 0, "sigmoid": 1}


def _elem(t: torch.Tensor, name: str) -> int:
    code = _ELEMS.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} is {t.dtype} (float32, bfloat16 or float16)")
    return code


def _on(dev, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, the other operands on {dev}")


# The calls below cost the host about as much as a small kernel runs: what
# torch.cuda wraps around these two is a third of a microsecond each.
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", torch.cuda.is_current_stream_capturing)


def _call(dev: torch.device, fn, *args) -> None:
    """One library call on ``dev`` and its current stream."""
    if dev.index == _current_device():
        rc = fn(*args, _stream_handle(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _stream_handle(dev))
    if rc:
        _lib.check(rc)


_COUNTERS: dict = {}


def _route_scratch(dev: torch.device, T: int, E: int, sequences: int, workspace: Optional[torch.Tensor]):
    """(workspace, its bytes, counters) of a routing on the current stream.
    Counters are zero between the calls of one stream (each call leaves them
    so); a call that a CUDA graph captures gets fresh ones, set to zero at
    each replay."""
    need, n = _route_space(T, E, sequences)
    key = (dev.index, _stream_handle(dev))
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = _stream_workspace(dev, key[1], need)
    if _capturing():
        return workspace, need, torch.zeros(n, dtype=torch.int32, device=dev)
    c = _COUNTERS.get(key)
    if c is None or c.numel() < n:
        c = _COUNTERS[key] = torch.zeros(max(n, 1024), dtype=torch.int32, device=dev)
    return workspace, need, c


_SCALARS: dict = {}


def _scalars(dev: torch.device):
    """An int32 and a float32 scalar on the device, for new_empty: half the
    host time of torch.empty with its keywords (1.3 against 2.3 us)."""
    s = _SCALARS.get(dev.index)
    if s is None:
        s = _SCALARS[dev.index] = (torch.empty((), dtype=torch.int32, device=dev), torch.empty((), device=dev))
    return s


def _route_args(logits, mask, sequences, scoring):
    """(logits with unit column stride, element type, row stride, mask pointer, scoring code, the mask's tensor)."""
    if not logits.is_cuda or logits.dim() != 2:
        raise ValueError("logits must be a 2-D CUDA tensor")
    code = _elem(logits, "logits")
    T, E = logits.shape
    ld, col = logits.stride()
    if E > 1 and col != 1 or T > 1 and ld < E:
        logits = logits.contiguous()
        ld = E
    if sequences < 1 or T % sequences:
        raise ValueError(f"{T} tokens are not {sequences} sequences of equal length")
    how = _SCORING.get(scoring)
    if how is None:
        raise ValueError(f"scoring {scoring!r} is not 'softmax' or 'sigmoid'")
    if mask is None:
        return logits, code, ld if T > 1 else E, None, how, None
    if mask.dtype != torch.bool or mask.numel() != T:
        raise ValueError(f"mask must be a bool tensor with one value per token ({T})")
    _on(logits.device, mask=mask)
    mask = mask.contiguous()
    return logits, code, ld if T > 1 else E, mask.data_ptr(), how, mask


@functools.lru_cache(maxsize=4096)
def _route_space(T: int, E: int, sequences: int):
    """(workspace bytes, counters) of a routing."""
    L = _lib.lib()
    return int(L.moe_route_train_workspace_size(T, E, sequences)), int(L.moe_route_train_counters(T, E, sequences))


def route_forward_train(logits: torch.Tensor, k: int, *, ids: Optional[torch.Tensor] = None,
                        mask: Optional[torch.Tensor] = None, sequences: int = 1, scoring: str = "softmax",
                        normalize: bool = True, workspace: Optional[torch.Tensor] = None) -> RouteTrain:
    """Top-k routing with the balance and z losses and per-expert counts.

    ``logits`` (T, E) float32, bfloat16 or float16; the T tokens are
    ``sequences`` runs of equal length.  Per token, with p = softmax(logits),
    s = sigmoid(logits) and q = p (``scoring="softmax"``) or s / sum(s)
    (``"sigmoid"``): the k largest logits (ties to the lower expert id) and
    their scores p or s, divided by their sum with ``normalize``;

        balance_loss = mean over sequences of sum_e (c_e E / (k N)) mean_t(q_te)
        z_loss       = mean over tokens of logsumexp(logits)^2

    with c_e the entries that chose expert e in a sequence of N tokens.
    ``mask`` (T,) bool: tokens where it is False (padding) take no part - ids
    -1, weights 0 - and neither does a token whose logits are all -inf.  An
    expert whose logit is -inf is never chosen; its slots get id -1.  ``ids``
    (T, k): experts chosen elsewhere, to be used in place of the top k.

    ``permute`` drops the -1 entries and reports them in the device status
    word.  The gradient is :func:`route_backward`; ``train.route_topk_train``
    puts both under autograd."""
    logits, code, ld, mask_ptr, how, mask = _route_args(logits, mask, sequences, scoring)
    dev = logits.device
    T, E = logits.shape
    if ids is not None:
        if tuple(ids.shape) != (T, k):
            raise ValueError(f"ids is {tuple(ids.shape)}, expected {(T, k)}")
        _on(dev, ids=ids)
        if ids.dtype.is_floating_point or ids.dtype == torch.bool:
            raise TypeError(f"ids are {ids.dtype}, not integers")
        if ids.dtype == torch.int64:
            ids = ids.clamp(-1, E)             # far values stay out of range in 32 bits
        ids = ids.to(torch.int32).contiguous()
    if not 1 <= k <= min(16, E) or E > 1024:
        raise ValueError(f"k={k}, E={E}: 1 <= k <= min(16, E) and E <= 1024 are supported")
    i32, f32 = _scalars(dev)
    o_ids, o_weights, o_counts = i32.new_empty((T, k)), f32.new_empty((T, k)), i32.new_empty((sequences, E))
    o_tokens, balance, z = i32.new_empty(sequences), torch.empty_like(f32), torch.empty_like(f32)
    workspace, need, counters = _route_scratch(dev, T, E, sequences, workspace)
    _call(dev, _lib.lib().moe_route_train, logits.data_ptr(), code, ld, T, E, k, sequences, mask_ptr,
          None if ids is None else ids.data_ptr(), how, normalize, o_ids.data_ptr(), o_weights.data_ptr(),
          o_counts.data_ptr(), o_tokens.data_ptr(), balance.data_ptr(), z.data_ptr(), workspace.data_ptr(), need,
          counters.data_ptr())
    return RouteTrain(o_ids, o_weights, o_counts, o_tokens, balance, z)


def route_backward(logits: torch.Tensor, routed: RouteTrain, *, d_weights: Optional[torch.Tensor] = None,
                   d_balance: Optional[torch.Tensor] = None, d_z: Optional[torch.Tensor] = None,
                   mask: Optional[torch.Tensor] = None, sequences: int = 1, scoring: str = "softmax",
                   normalize: bool = True) -> torch.Tensor:
    """Gradient (T, E) with respect to the logits, in their type, for upstream
    gradients of the weights (T, k) and of the two losses (scalars on the
    device); a gradient that is None counts as zero.  ``routed`` is the
    forward's result for the same logits and options."""
    logits, code, ld, mask_ptr, how, mask = _route_args(logits, mask, sequences, scoring)
    dev = logits.device
    T, E = logits.shape
    ids, weights, counts, tokens = routed[:4]
    k = ids.shape[-1]
    if (ids.shape != (T, k) or weights.shape != (T, k) or counts.shape != (sequences, E) or tokens.shape != (sequences,)
            or not ids.get_device() == weights.get_device() == counts.get_device() == tokens.get_device() == dev.index):
        raise ValueError(f"routed has ids {tuple(ids.shape)}, weights {tuple(weights.shape)}, counts "
                         f"{tuple(counts.shape)} and tokens {tuple(tokens.shape)} on {ids.device}, expected {(T, k)}, "
                         f"{(T, k)}, {(sequences, E)} and {(sequences,)} on {dev}")
    if not (ids.dtype == counts.dtype == tokens.dtype == torch.int32 and weights.dtype == torch.float32
            and ids.is_contiguous() and weights.is_contiguous() and counts.is_contiguous() and tokens.is_contiguous()):
        raise TypeError("routed's tensors must be as route_forward_train returns them: int32 and float32, contiguous")
    if d_weights is not None:
        if d_weights.shape != (T, k) or d_weights.device != dev:
            raise ValueError(f"d_weights is {tuple(d_weights.shape)} on {d_weights.device}, expected {(T, k)} on {dev}")
        d_weights = d_weights.to(torch.float32).contiguous()
    for g in (d_balance, d_z):
        if g is not None and (g.numel() != 1 or g.dtype != torch.float32 or g.device != dev):
            raise ValueError("d_balance and d_z must be float32 scalar tensors on the logits' device")
    d = logits.new_empty((T, E))
    _call(dev, _lib.lib().moe_route_backward, logits.data_ptr(), code, ld, T, E, k, sequences, mask_ptr, how,
          normalize, ids.data_ptr(), weights.data_ptr(), counts.data_ptr(), tokens.data_ptr(),
          None if d_weights is None else d_weights.data_ptr(), None if d_balance is None else d_balance.data_ptr(),
          None if d_z is None else d_z.data_ptr(), d.data_ptr())
    return d


def _rows(t: torch.Tensor, name: str) -> torch.Tensor:
    if not t.is_cuda or t.dim() != 2:
        raise ValueError(f"{name} must be a 2-D CUDA tensor")
    if t.shape[1] % 4 or t.shape[1] == 0:
        raise ValueError(f"{name} has rows of {t.shape[1]} elements: a positive multiple of 4 is needed")
    if not t.is_contiguous():
        return t.contiguous()
    # A contiguous view may start anywhere in its storage; the kernels read
    # four elements at a time.
    return t.clone() if t.data_ptr() % (4 * t.element_size()) else t


def combine_rows_backward(dy: torch.Tensor, y_sorted: torch.Tensor, inverse: torch.Tensor, weights: torch.Tensor,
                          group_sizes: torch.Tensor, *, dtype: torch.dtype = torch.float32
                          ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Backward of :func:`combine_rows` for the upstream gradient ``dy``
    (T, D): (dys, dw) with ``dys[inverse[t, j]] = weights[t, j] * dy[t]`` in
    ``dtype`` - rows past ``sum(group_sizes)`` zero - and the f32 weights'
    gradient ``dw[t, j] = <dy[t], y_sorted[inverse[t, j]]>``, 0 at dropped
    entries.  bfloat16 ``dys`` are what the experts' backward multiplies."""
    code = _elem(dy, "dy")
    dy, y_sorted = _rows(dy, "dy"), _rows(y_sorted, "y_sorted")
    dev = dy.device
    T, k = inverse.shape
    N, D = y_sorted.shape
    if dy.shape != (T, D) or weights.shape != (T, k):
        raise ValueError(f"dy {tuple(dy.shape)}, weights {tuple(weights.shape)}: expected {(T, D)} and {(T, k)}")
    if y_sorted.dtype != torch.float32 or inverse.dtype != torch.int32:
        raise TypeError("y_sorted must be float32 and inverse int32")
    if dtype not in _ELEMS:
        raise TypeError(f"dtype {dtype} (float32, bfloat16 or float16)")
    _on(dev, y_sorted=y_sorted, inverse=inverse, weights=weights, group_sizes=group_sizes)
    inverse, weights = inverse.contiguous(), weights.to(torch.float32).contiguous()
    gs = group_sizes.to(torch.int32).contiguous()
    dys = torch.empty_like(y_sorted, dtype=dtype)
    dw = torch.empty_like(weights)
    _call(dev, _lib.lib().moe_combine_rows_backward, dy.data_ptr(), code, y_sorted.data_ptr(), inverse.data_ptr(),
          weights.data_ptr(), gs.data_ptr(), T, k, D, N, gs.numel(), dys.data_ptr(), _ELEMS[dtype], dw.data_ptr())
    return dys, dw


def gather_rows_backward(dxs: torch.Tensor, inverse: torch.Tensor, *, dtype: Optional[torch.dtype] = None
                         ) -> torch.Tensor:
    """Backward of :func:`gather_rows`: ``dx[t] = sum_j dxs[inverse[t, j]]``,
    summed in f32 in slot order, in ``dtype`` (default: ``dxs``'s)."""
    code = _elem(dxs, "dxs")
    dxs = _rows(dxs, "dxs")
    dev = dxs.device
    T, k = inverse.shape
    N, D = dxs.shape
    dtype = dxs.dtype if dtype is None else dtype
    if inverse.dtype != torch.int32:
        raise TypeError("inverse must be int32")
    if dtype not in _ELEMS:
        raise TypeError(f"dtype {dtype} (float32, bfloat16 or float16)")
    _on(dev, inverse=inverse)
    inverse = inverse.contiguous()
    dx = dxs.new_empty((T, D), dtype=dtype)
    _call(dev, _lib.lib().moe_gather_rows_backward, dxs.data_ptr(), code, inverse.data_ptr(), T, k, D, N,
          dx.data_ptr(), _ELEMS[dtype])
    return dx


def moe_layer(x: torch.Tensor, logits: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, k: int, *,
              w_up_scale: Optional[torch.Tensor] = None, w_down_scale: Optional[torch.Tensor] = None):
    """A whole MoE expert layer: top-k routing of ``x`` (T, D) by ``logits``
    (T, E), the fused expert MLP over the expert-sorted rows, and the
    weighted combine.  Returns (y (T, D) f32, group_sizes)."""
    from .kernel import fused_ragged_mlp
    E = w_up.shape[0]
    ids, w = route_topk(logits, k)
    gs, src, inv = permute(ids, E)
    xs = gather_rows(x, src, k)
    ys = fused_ragged_mlp(xs, w_up, w_down, gs, w_up_scale=w_up_scale, w_down_scale=w_down_scale)
    return combine_rows(ys, inv, w), gs
