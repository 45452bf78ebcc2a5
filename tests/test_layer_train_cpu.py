"""CPU tests of the steps that train a whole MoE layer: the oracle's formulas
against differentiation in float64 and against differences, and the argument
checks of the C ABI and of the Python entry points (all before device work)."""

import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import moe_oracle as orc
from src import _lib, grads, router

CASES = [(scoring, normalize, sequences, masked, given) for scoring in ("softmax", "sigmoid")
         for normalize in (True, False) for sequences, masked, given in ((1, False, False), (3, True, False), (2, True, True))]


def _inputs(sequences, masked, given, seed=0):
    rng = np.random.default_rng(seed)
    T, E, k = 12, 7, 3
    x = rng.standard_normal((T, E)) * 2
    x[4, [0, 5]] = -np.inf
    mask = rng.random(T) < 0.7 if masked else None
    ids = np.stack([rng.permutation(E)[:k] for _ in range(T)]).astype(np.int32) if given else None
    if given:
        ids[1, 0], ids[2, 1], ids[3, :2] = -1, E, 6         # dropped, out of range, one expert twice
    return x, mask, ids, rng.standard_normal((T, k)), T, E, k


def _loss(x, mask, ids, dw, k, sequences, scoring, normalize):
    """The scalar whose gradient is wanted, in torch float64, from ids fixed beforehand."""
    T, E = x.shape
    allowed = torch.isfinite(x)
    low = torch.where(allowed, x, -math.inf)
    keep = torch.ones(T, dtype=torch.bool) if mask is None else torch.from_numpy(mask)
    score = torch.softmax(low, 1) if scoring == "softmax" else torch.where(allowed, torch.sigmoid(x), 0)
    on = torch.from_numpy((ids >= 0) & (ids < E)) & keep[:, None]
    at = torch.from_numpy(np.where((ids >= 0) & (ids < E), ids, 0)).long()
    w = torch.where(on, score.gather(1, at), 0)
    if normalize:
        w = w / torch.where(w.sum(1, keepdim=True) > 0, w.sum(1, keepdim=True), 1)
    q = score / score.sum(1, keepdim=True)
    L = T // sequences
    balance, live = 0.0, 0
    for s in range(sequences):
        rows = slice(s * L, (s + 1) * L)
        n = int(keep[rows].sum())
        if n == 0:
            continue
        live += 1
        c = torch.bincount(at[rows][on[rows]], minlength=E).double()
        balance = balance + (c * E / (k * n) * torch.where(keep[rows][:, None], q[rows], 0).sum(0) / n).sum()
    lse = torch.logsumexp(low, 1)
    z = torch.where(keep, lse ** 2, 0).sum() / max(int(keep.sum()), 1)
    return (w * torch.from_numpy(dw)).sum() + 0.7 * balance / max(live, 1) + 0.3 * z, balance / max(live, 1), z, w


@pytest.mark.parametrize("scoring,normalize,sequences,masked,given", CASES)
def test_oracle_gradient_matches_autograd_and_differences(scoring, normalize, sequences, masked, given):
    x, mask, ids, dw, T, E, k = _inputs(sequences, masked, given)
    r = orc.route_train(x, k, ids, mask, sequences, scoring, normalize)
    xt = torch.from_numpy(np.where(np.isfinite(x), x, 0)).requires_grad_()
    xin = torch.where(torch.from_numpy(np.isfinite(x)), xt, -math.inf)
    fixed = r["ids"] if ids is None else ids
    loss, balance, z, w = _loss(xin, mask, fixed, dw, k, sequences, scoring, normalize)
    np.testing.assert_allclose(r["weights"], w.detach().numpy(), rtol=1e-12, atol=1e-14)
    assert r["balance"] == pytest.approx(balance.item(), rel=1e-12)
    assert r["z"] == pytest.approx(z.item(), rel=1e-12)
    g, = torch.autograd.grad(loss, xt)
    g = torch.where(torch.from_numpy(np.isfinite(x)), g, 0).numpy()
    d, scale = orc.route_train_backward(r, dw, 0.7, 0.3)
    np.testing.assert_allclose(d, g, rtol=1e-11, atol=1e-13)
    assert np.all(np.abs(d) <= scale * (1 + 1e-12))
    # Central differences: truncation h^2 |l'''| / 6 and cancellation 2^-52 |l| / h, both below 1e-8 here.
    h = 1e-5
    for t, e in ((0, 0), (3, 2), (4, 1), (7, 6), (11, 3)):
        step = np.zeros_like(x)
        step[t, e] = h
        hi, lo = (_loss(torch.from_numpy(x + s * step), mask, fixed, dw, k, sequences, scoring, normalize)[0].item()
                  for s in (1, -1))
        assert abs((hi - lo) / (2 * h) - d[t, e]) < 1e-8


def test_oracle_route_matches_route_topk():
    rng = np.random.default_rng(1)
    logits = np.round(rng.standard_normal((50, 16)) * 4).astype(np.float32) / 4          # ties
    ids, w = orc.route_topk(logits, 5)
    r = orc.route_train(logits, 5)
    assert np.array_equal(r["ids"], ids)
    np.testing.assert_allclose(r["weights"], w, rtol=1e-6)
    assert r["balance"] >= 0 and r["counts"].sum() == 250 and r["tokens"][0] == 50


def test_oracle_row_gradients_are_transposes():
    """<dys, ys'> + <dw, w'> of the two forms against combine_rows itself (it is bilinear)."""
    rng = np.random.default_rng(2)
    T, k, D, E = 9, 3, 8, 5
    ids = np.stack([rng.permutation(E)[:k] for _ in range(T)]).astype(np.int32)
    ids[2] = -1
    gs, src, inv = orc.permute_by_expert(ids, E)
    inv = inv.reshape(T, k)
    ys, w, dy = rng.standard_normal((T * k, D)), rng.random((T, k)), rng.standard_normal((T, D))
    dys, dw = orc.combine_rows_backward(dy, ys, inv, w)
    y = orc.combine_rows(ys, inv.reshape(-1), w, k).astype(np.float64)
    lhs = (dy * y).sum()
    assert (dys * ys).sum() == pytest.approx(lhs, rel=1e-6) and (dw * w).sum() == pytest.approx(lhs, rel=1e-6)
    assert np.all(dys[int(gs.sum()):] == 0)
    dxs = rng.standard_normal((T * k, D))
    x = rng.standard_normal((T, D))
    xs = np.zeros((T * k, D))
    xs[:len(src)] = x[src // k]
    n = int(gs.sum())
    assert (orc.gather_rows_backward(dxs, inv) * x).sum() == pytest.approx((dxs[:n] * xs[:n]).sum(), rel=1e-12)


# ----------------------------------------------------------------------------- refusals
def _null():
    return ctypes.c_void_p(0)


def test_route_abi_refusals():
    L = _lib.lib()
    p = ctypes.c_void_p(256)

    def call(elem=0, ld=8, T=4, E=8, k=2, S=1, scoring=0, logits=p, out=p, ws=p, nbytes=1 << 20):
        return L.moe_route_train(logits, elem, ld, T, E, k, S, None, None, scoring, 1, out, out, out, out, out, out, ws,
                                 nbytes, p, None)
    assert call(k=0) == call(k=9) == call(k=17, E=64, ld=64) == call(E=1025, ld=1025) == call(T=-1) == -1
    assert call(T=1 << 30, k=2) == -1                                   # T k reaches 2^31
    assert call(S=3) == call(S=0) == call(ld=7) == call(scoring=2) == -1
    assert call(elem=3) == -3
    assert call(logits=_null()) == -1 and b"null" in L.moe_last_error()
    assert call(nbytes=16) == -4 and call(ws=_null()) == -4
    assert call(ws=ctypes.c_void_p(264)) == -7
    assert call(logits=ctypes.c_void_p(258)) == -7

    def back(elem=0, T=4, E=8, k=2, S=1, logits=p, d=p):
        return L.moe_route_backward(logits, elem, E, T, E, k, S, None, 0, 1, p, p, p, p, None, None, None, d, None)
    assert back(k=0) == back(S=3) == back(d=_null()) == -1
    assert back(elem=-1) == -3
    assert back(d=ctypes.c_void_p(258)) == -7
    assert back(T=0) == 0
    assert L.moe_route_train_workspace_size(10, 8, 3) == 0 and L.moe_route_train_workspace_size(12, 8, 3) > 0


def test_row_abi_refusals():
    L = _lib.lib()
    p = ctypes.c_void_p(256)

    def comb(T=4, k=2, D=8, rows=8, E=2, dy=p, a=0, b=0):
        return L.moe_combine_rows_backward(dy, a, p, p, p, p, T, k, D, rows, E, p, b, p, None)
    assert comb(T=-1) == comb(k=0) == comb(D=6) == comb(D=0) == comb(rows=-1) == comb(E=0) == comb(dy=_null()) == -1
    assert comb(a=3) == comb(b=9) == -3
    assert comb(dy=ctypes.c_void_p(260)) == -7
    assert comb(T=0, rows=0) == 0

    def gath(T=4, k=2, D=8, rows=8, x=p, a=0, b=0):
        return L.moe_gather_rows_backward(x, a, p, T, k, D, rows, p, b, None)
    assert gath(T=-1) == gath(k=0) == gath(D=10) == gath(x=_null()) == -1
    assert gath(a=-1) == -3 and gath(x=ctypes.c_void_p(264)) == -7
    assert gath(T=0) == 0


class _Desc(ctypes.Structure):
    _fields_ = [("inp", ctypes.c_void_p), ("out", ctypes.c_void_p), ("rows", ctypes.c_int64), ("cols", ctypes.c_int64),
                ("in_ld", ctypes.c_int64), ("out_ld", ctypes.c_int64), ("in_type", ctypes.c_int32),
                ("out_type", ctypes.c_int32)]


def test_gradient_list_abi_refusals():
    L = _lib.lib()
    p = ctypes.c_void_p(256)

    def norm(n=1, kind=2, ws=p, nbytes=1 << 20, **kw):
        d = _Desc(256, 256, 1, 10, 10, 10, 0, 0)
        for name, v in kw.items():
            setattr(d, name, v)
        return L.moe_grad_norm(ctypes.byref(d), n, kind, p, ws, nbytes, None)
    assert norm(n=-1) == norm(kind=0) == norm(kind=4) == norm(rows=-1) == norm(inp=0) == -1
    assert norm(rows=2, in_ld=9) == -1
    assert norm(in_type=3) == -3
    assert norm(rows=1 << 30, cols=1 << 30, in_ld=1 << 30) == -2
    assert norm(inp=258) == -7 and norm(ws=ctypes.c_void_p(8)) == -7
    assert norm(nbytes=8) == -4

    def clip(max_norm=1.0, **kw):
        d = _Desc(256, 256, 1, 10, 10, 10, 0, 0)
        for name, v in kw.items():
            setattr(d, name, v)
        return L.moe_clip_grads(ctypes.byref(d), 1, 2, max_norm, None, p, p, 1 << 20, None)
    assert clip(-1.0) == clip(math.nan) == clip(out=0) == clip(rows=2, out_ld=3) == -1
    assert clip(out_type=5) == -3 and clip(out=257) == -7
    def pair(a, b, na, nb):                                        # outputs at a and b, of na and nb f32
        d = (_Desc * 2)(_Desc(4096, a, 1, na, na, na, 0, 0), _Desc(8192, b, 1, nb, nb, nb, 0, 0))
        return L.moe_clip_grads(d, 2, 2, 1.0, None, p, p, 8, None)
    assert pair(256, 256, 1, 1) == pair(256, 260, 2, 1) == pair(260, 256, 1, 2) == -1
    assert b"share memory" in L.moe_last_error()
    assert clip(out_type=1) == clip(rows=2, out_ld=12) == -1       # in place, but not the same elements
    assert pair(256, 260, 1, 1) == pair(260, 256, 1, 1) == pair(256, 256, 0, 1) == -4      # apart: the workspace is next
    assert L.moe_grad_norm_workspace_size(-1) == 0 and L.moe_grad_norm_workspace_size(1000) > L.moe_grad_norm_workspace_size(1)


def test_python_refusals_without_a_gpu():
    with pytest.raises(ValueError, match="CUDA"):
        router.route_forward_train(torch.zeros(4, 8), 2)
    with pytest.raises(ValueError, match="CUDA"):
        router.gather_rows_backward(torch.zeros(4, 8), torch.zeros((2, 2), dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        grads.grad_norm([torch.zeros(4)])
    with pytest.raises(ValueError, match="norm_type"):
        grads.grad_norm([torch.zeros(4)], 3)
    with pytest.raises(ValueError, match="max_norm"):
        grads.clip_grad_norm([torch.zeros(4)], -1.0)
    from src import train
    with pytest.raises(ValueError, match="activation"):
        train.moe_layer_train(torch.zeros(4, 8), torch.zeros(4, 2), torch.zeros(2, 8, 8), torch.zeros(2, 8, 8), 1,
                              activation="relu")


@pytest.mark.parametrize("shape,view,want", [
    ((6, 8), lambda t: t, (1, 48, 48)),
    ((6, 8), lambda t: t.t(), (1, 48, 48)),
    ((6, 8), lambda t: t[:, :5], (6, 5, 8)),
    ((2, 6, 8), lambda t: t[:, :, 2:6], (12, 4, 8)),
    ((2, 6, 8), lambda t: t[:, :4], (2, 32, 48)),
    ((2, 6, 8), lambda t: t[:, :4, :4], None),
    ((6, 8), lambda t: t[:, ::2], (24, 1, 2)),
    ((8,), lambda t: t[:1].expand(5), None),
    ((), lambda t: t, (1, 1, 1)),
])
def test_rows_of_strided_tensors(shape, view, want):
    assert _lib.native().tensor_rows(view(torch.zeros(shape))) == want
