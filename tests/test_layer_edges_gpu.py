"""Edges of routing and of a layer's training step: tokens that take no part at
the end of a batch, batches without any, gradients of bf16 logits, two graphs
and a user's workspace."""

import math

import pytest
import torch

from src import _lib, grads, router, train
from src.kernel import swiglu_interleave

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k", [(1, 8, 2), (33, 60, 6), (700, 256, 8), (97, 1000, 16)])
def test_last_token_without_an_expert(T, E, k, scoring):
    x = torch.randn((T, E), generator=_gen(T), device=DEV)
    x[T - 1] = -math.inf
    dw = torch.full((T, k), math.nan, device=DEV)
    dw[:T - 1] = 1.0
    one = torch.ones((), device=DEV)
    for mask in (None, torch.ones(T, dtype=torch.bool, device=DEV)):
        r = router.route_forward_train(x, k, mask=mask, scoring=scoring)
        d = router.route_backward(x, r, d_weights=dw, d_balance=one, d_z=one, mask=mask, scoring=scoring)
        assert torch.all(r.ids[T - 1] == -1) and torch.all(r.weights[T - 1] == 0) and torch.all(d[T - 1] == 0)
        assert r.tokens.item() == T - 1 and int(r.counts.sum()) == (T - 1) * k
        assert torch.isfinite(r.balance_loss) and torch.isfinite(r.z_loss) and torch.isfinite(d).all()


def _layer(T, D, F, E, swiglu, seed):
    g = _gen(seed)
    r = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    ups = [(r(E, D, F) / D ** 0.5).bfloat16() for _ in range(2 if swiglu else 1)]
    return r(T, D).bfloat16(), r(D, E) / D ** 0.5, ups, (r(E, F, D) / F ** 0.5).bfloat16(), r(T, D)


@pytest.mark.parametrize("swiglu", [False, True])
def test_a_batch_without_tokens_that_count(swiglu):
    T, D, F, E, k = 40, 256, 256, 4, 2
    x, wr, ups, wd, dy = _layer(T, D, F, E, swiglu, 1)
    w_in = swiglu_interleave(*ups) if swiglu else ups[0]
    leaves = [t.detach().clone().requires_grad_() for t in (x, x.float() @ wr, w_in, wd)]
    y, routed = train.moe_layer_train(*leaves, k, activation="swiglu" if swiglu else "gelu",
                                      mask=torch.zeros(T, dtype=torch.bool, device=DEV))
    ((y * dy).sum() + routed.balance_loss + routed.z_loss).backward()
    assert torch.all(y == 0) and routed.balance_loss.item() == 0 and routed.z_loss.item() == 0
    for t in leaves:
        assert torch.all(t.grad == 0)
    assert grads.clip_grad_norm([t.grad for t in leaves], 1.0).item() == 0
    _lib.device_status(reset=True)


def test_gradient_of_bf16_logits():
    """Within 1e-2 in the 2-norm of float64 differentiation (bf16 operands, each rounded by at most 2^-8)."""
    T, D, F, E, k = 96, 256, 256, 4, 2
    x, wr, ups, wd, dy = _layer(T, D, F, E, False, 2)
    logits = (x.float() @ wr).bfloat16().requires_grad_()
    y, routed = train.moe_layer_train(x, logits, ups[0], wd, k)
    ((y * dy).sum() + routed.balance_loss).backward()
    ld = logits.detach().double().requires_grad_()
    at = routed.ids.long()
    p = torch.softmax(ld, 1)
    w = p.gather(1, at)
    w = w / w.sum(1, keepdim=True)
    ref = torch.zeros((T, D), dtype=torch.double, device=DEV)
    for e in range(E):
        h = torch.nn.functional.gelu(x.double() @ ups[0][e].double(), approximate="tanh") @ wd[e].double()
        ref = ref + (w * (at == e)).sum(1, keepdim=True) * h
    f = torch.bincount(at.reshape(-1), minlength=E) * E / (k * T)
    want, = torch.autograd.grad((ref * dy.double()).sum() + (f * p.mean(0)).sum(), ld)
    assert logits.grad.dtype == torch.bfloat16
    assert ((logits.grad.double() - want).norm() / want.norm()).item() <= 1e-2


def test_two_graphs_replayed_on_two_streams():
    """Each capture has workspaces and counters of its own: replays that overlap do not meet."""
    xs = [torch.randn((30000, 64), generator=_gen(i), device=DEV) for i in (3, 4)]
    ts = [[torch.randn(n, generator=_gen(n), device=DEV) for n in (400_000, 33)] for _ in xs]
    want = [router.route_forward_train(x, 4) for x in xs]
    norms = [grads.grad_norm(t) for t in ts]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for x, t in zip(xs, ts):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append((*router.route_forward_train(x, 4), grads.grad_norm(t)))
    for _ in range(6):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for out, r, n in zip(outs, want, norms):
        assert all(torch.equal(a, b) for a, b in zip(out, (*r, n)))


def test_workspace_of_the_caller():
    x = torch.randn((20000, 64), generator=_gen(5), device=DEV)
    want = router.route_forward_train(x, 4)
    for ws in (torch.empty(1 << 20, dtype=torch.uint8, device=DEV), torch.empty(8, dtype=torch.uint8, device=DEV),
               torch.empty(1 << 20, dtype=torch.uint8)):                # enough; too small; elsewhere: one of the library's
        assert all(torch.equal(a, b) for a, b in zip(router.route_forward_train(x, 4, workspace=ws), want))
    with pytest.raises(_lib.MoeError, match="aligned"):
        router.route_forward_train(x, 4, workspace=torch.empty((1 << 20) + 8, dtype=torch.uint8, device=DEV)[8:])
