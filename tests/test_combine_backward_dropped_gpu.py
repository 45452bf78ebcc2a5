"""Backward of combine where entries were dropped after the permutation: every
row that no entry maps to is zero, wherever it lies."""

import numpy as np
import pytest
import torch

from oracle import moe_oracle as orc
from src import router

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _junk(shape, dtype):
    """Leaves NaN in the memory that the next tensor of this size takes."""
    del_me = [torch.full(shape, float("nan"), dtype=dtype, device=DEV) for _ in range(3)]
    torch.cuda.synchronize()
    del del_me


@pytest.mark.parametrize("out_t", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,k,D,E,drop,extra", [(1, 1, 4, 2, 1.0, 0), (5, 2, 8, 4, 0.4, 3), (70, 3, 60, 5, 0.3, 0),
                                                (129, 9, 1020, 32, 0.1, 7), (40, 8, 1024, 64, 0.0, 1),
                                                (64, 2, 2052, 8, 0.5, 0), (300, 4, 16, 16, 0.99, 40)])
def test_rows_without_an_entry_are_zero(T, k, D, E, drop, extra, out_t):
    rng = np.random.default_rng(T + D)
    ids = np.stack([rng.permutation(E)[:k] for _ in range(T)]).astype(np.int32)
    gs, _, inv = router.permute(torch.from_numpy(ids).to(DEV), E)
    inv = torch.where(torch.from_numpy(rng.random((T, k)) < drop).to(DEV), -1, inv)      # over an expert's capacity
    rows = T * k + extra
    dy = torch.randn((T, D), device=DEV)
    ys = torch.randn((rows, D), device=DEV)
    w = torch.rand((T, k), device=DEV)
    _junk((rows, D), out_t)
    dys, dw = router.combine_rows_backward(dy, ys, inv, w, gs, dtype=out_t)
    ref, refw = orc.combine_rows_backward(*(t.double().cpu().numpy() for t in (dy, ys)), inv.cpu().numpy(),
                                          w.double().cpu().numpy())
    got = dys.double().cpu().numpy()
    tol = U * np.abs(ref) + HALF_STEP[out_t] * (1 + U) * np.abs(ref) + (2.0 ** -25 if out_t == torch.float16 else 0)
    assert np.all(np.abs(got - ref) <= tol)
    mapped = np.zeros(rows, bool)
    mapped[inv[inv >= 0].cpu().numpy()] = True
    assert np.all(got[~mapped] == 0)
    _, mag = orc.combine_rows_backward(*(np.abs(t.double().cpu().numpy()) for t in (dy, ys)), inv.cpu().numpy(),
                                       w.double().cpu().numpy())
    assert np.all(np.abs(dw.double().cpu().numpy() - refw) <= (D / 32 + 18) * U * mag)   # D / 32 groups a thread, 18 more
    assert torch.all(dw[inv < 0] == 0)


@pytest.mark.parametrize("T,k,D", [(1_100_001, 2, 512), (300_000, 2, 8), (100_001, 2, 1024), (40_000, 16, 32), (8192, 8, 256)])
def test_many_rows(T, k, D):
    """Rows in a random order, a tenth of the entries dropped, bits for bits (weights are powers of two)."""
    g = torch.Generator(device=DEV)
    g.manual_seed(D)
    N = T * k
    inv = torch.randperm(N, generator=g, device=DEV).to(torch.int32).view(T, k)
    inv = torch.where(torch.rand((T, k), generator=g, device=DEV) < 0.1, -1, inv)
    dy = torch.randn((T, D), generator=g, device=DEV).bfloat16()
    ys = torch.ones((N, D), device=DEV)
    w = torch.full((T, k), 0.5, device=DEV)
    gs = torch.full((8,), N // 8, dtype=torch.int32, device=DEV)
    _junk((N, D), torch.bfloat16)
    dys, _ = router.combine_rows_backward(dy, ys, inv, w, gs, dtype=torch.bfloat16)
    want = torch.zeros((N, D), dtype=torch.bfloat16, device=DEV)
    at, entry = inv.reshape(-1), torch.arange(N, device=DEV)
    on = at >= 0
    want[at[on].long()] = dy[entry[on] // k] * 0.5
    assert torch.equal(dys, want)


def test_in_a_graph():
    """Captured with one set of dropped entries, replayed with others."""
    T, k, D = 200, 4, 512
    inv = torch.randperm(T * k, device=DEV).to(torch.int32).view(T, k)
    dy, ys, w = torch.randn((T, D), device=DEV), torch.randn((T * k, D), device=DEV), torch.rand((T, k), device=DEV)
    gs = torch.full((4,), T, dtype=torch.int32, device=DEV)
    static = inv.clone()
    router.combine_rows_backward(dy, ys, static, w, gs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dys, dw = router.combine_rows_backward(dy, ys, static, w, gs)
    for share in (0.5, 0.0, 1.0):
        static.copy_(torch.where(torch.rand((T, k), device=DEV) < share, -1, inv))
        dys.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        want, want_w = router.combine_rows_backward(dy, ys, static, w, gs)
        assert torch.equal(dys, want) and torch.equal(dw, want_w) and torch.isfinite(dys).all()
