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

from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib


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
    row in expert order - 0 past the last routed row -, inverse (T, k) row of
    each entry, -1 if dropped)."""
    ids = ids.to(torch.int32).contiguous()
    dev = ids.device
    N = ids.numel()
    L = _lib.lib()
    gs = torch.empty(num_experts, dtype=torch.int32, device=dev)
    src = torch.empty(N, dtype=torch.int32, device=dev)
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


def _score(scoring: str) -> int:
    code = _SCORING.get(scoring)
    if code is None:
        raise ValueError(f"scoring {scoring!r} is not 'softmax' or 'sigmoid'")
    return code


def _out_elem(dtype: torch.dtype) -> int:
    code = _ELEMS.get(dtype)
    if code is None:
        raise TypeError(f"dtype {dtype} (float32, bfloat16 or float16)")
    return code


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
    return RouteTrain._make(_lib.native().route_forward(logits, k, ids, mask, sequences, _score(scoring), normalize,
                                                        workspace))


def route_backward(logits: torch.Tensor, routed: RouteTrain, *, d_weights: Optional[torch.Tensor] = None,
                   d_balance: Optional[torch.Tensor] = None, d_z: Optional[torch.Tensor] = None,
                   mask: Optional[torch.Tensor] = None, sequences: int = 1, scoring: str = "softmax",
                   normalize: bool = True) -> torch.Tensor:
    """Gradient (T, E) with respect to the logits, in their type, for upstream
    gradients of the weights (T, k) and of the two losses (scalars on the
    device); a gradient that is None counts as zero.  ``routed`` is the
    forward's result for the same logits and options."""
    return _lib.native().route_backward(logits, *routed[:4], d_weights, d_balance, d_z, mask, sequences,
                                        _score(scoring), normalize)


def combine_rows_backward(dy: torch.Tensor, y_sorted: torch.Tensor, inverse: torch.Tensor, weights: torch.Tensor,
                          group_sizes: torch.Tensor, *, dtype: torch.dtype = torch.float32
                          ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Backward of :func:`combine_rows` for the upstream gradient ``dy``
    (T, D): (dys, dw) with ``dys[inverse[t, j]] = weights[t, j] * dy[t]`` in
    ``dtype`` - zero in every row that no entry maps to, past
    ``sum(group_sizes)`` or of entries dropped after :func:`permute` - and the
    f32 weights' gradient ``dw[t, j] = <dy[t], y_sorted[inverse[t, j]]>``, 0 at
    dropped entries.  bfloat16 ``dys`` are what the experts' backward
    multiplies."""
    return _lib.native().combine_backward(dy, y_sorted, inverse, weights, group_sizes, _out_elem(dtype))


def gather_rows_backward(dxs: torch.Tensor, inverse: torch.Tensor, *, dtype: Optional[torch.dtype] = None
                         ) -> torch.Tensor:
    """Backward of :func:`gather_rows`: ``dx[t] = sum_j dxs[inverse[t, j]]``,
    summed in f32 in slot order, in ``dtype`` (default: ``dxs``'s)."""
    return _lib.native().gather_backward(dxs, inverse, -1 if dtype is None else _out_elem(dtype))


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
