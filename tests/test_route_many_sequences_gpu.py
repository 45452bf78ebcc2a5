"""Routing of very many short sequences: values, and a time that grows with
the tokens and not with the square of the sequences."""

import pytest
import torch

from src import router

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U = 2.0 ** -24


@pytest.mark.parametrize("sequences,L,E,k", [(4097, 3, 8, 2), (9000, 1, 60, 6), (5000, 33, 24, 3), (20000, 2, 256, 8),
                                             (4500, 1, 1000, 16)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_many_sequences_match_float64(sequences, L, E, k, scoring):
    g = torch.Generator(device=DEV)
    g.manual_seed(sequences)
    T = sequences * L
    x = torch.randn((T, E), generator=g, device=DEV)
    mask = torch.rand(T, generator=g, device=DEV) < 0.7
    mask[:L] = False                                               # a sequence of padding only
    dw = torch.randn((T, k), generator=g, device=DEV)
    how = {"mask": mask, "sequences": sequences, "scoring": scoring}
    one = torch.ones((), device=DEV)
    r = router.route_forward_train(x, k, **how)
    d = router.route_backward(x, r, d_weights=dw, d_balance=one, d_z=one, **how)
    # The definition in float64 with the chosen experts fixed, differentiated.
    ids = r.ids.long().clamp(min=0)
    assert torch.equal(torch.where(mask[:, None], x, 0).topk(k, 1).values[mask], x.gather(1, ids)[mask])
    xd = x.double().requires_grad_()
    s = torch.softmax(xd, 1) if scoring == "softmax" else torch.sigmoid(xd)
    w = s.gather(1, ids)
    w = w / w.sum(1, keepdim=True) * mask[:, None]
    hot = torch.zeros((T, E), device=DEV, dtype=torch.double).scatter_(1, ids, 1.0) * mask[:, None]
    c = hot.view(sequences, L, E).sum(1)
    assert torch.equal(r.counts.double(), c)
    n = mask.view(sequences, L).sum(1)
    assert torch.equal(r.tokens.long(), n)
    q = (s / s.sum(1, keepdim=True) * mask[:, None]).view(sequences, L, E).sum(1)
    nn = n.clamp(min=1).double()[:, None]
    balance = (c * E / (k * nn) * q / nn).sum() / (n > 0).sum()
    z = torch.where(mask, torch.logsumexp(xd, 1) ** 2, 0).sum() / mask.sum()
    ref, = torch.autograd.grad(balance + z + (w * dw).sum(), xd)
    span = float(x.max() - x.min()) + float(x.abs().max())
    # As for fewer sequences: scores within (span + 80) u, f32 sums over the few rows of a block, the rest in f64.
    tol = (2 * (span + 80) + L + 50) * U
    assert abs(r.balance_loss.item() - balance.item()) <= tol * balance.item()
    assert abs(r.z_loss.item() - z.item()) <= 2 * tol * (z.item() + 1)
    # Each element is a sum of terms of at most: weights w (|dw| + <|dw|, w>) <= 2 |dw| max, the losses' share per token
    # q (|f| + <|f|, q>) / (S' n) <= 2 max f and 2 |lse| p / N.
    size = 2 * dw.abs().amax(1, keepdim=True).double() + (2 * c.max() * E / k + 2 * (span + 10)) / mask.sum()
    assert torch.all((d.double() - ref).abs() <= 8 * (span + 80 + k + E / 8) * U * size)
    assert torch.all(d[~mask] == 0) and torch.all(r.ids[~mask] == -1)


def test_time_does_not_grow_with_the_square():
    """One token a sequence against one sequence: the same rows, so tens of microseconds either way (a scan of all
    sequences by every block's every warp takes tens of milliseconds here)."""
    T, E, k = 131072, 8, 2
    x = torch.randn((T, E), device=DEV)
    one = torch.ones((), device=DEV)
    r = router.route_forward_train(x, k, sequences=T)
    best = float("inf")
    for _ in range(4):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        router.route_backward(x, r, d_balance=one, d_z=one, sequences=T)
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b))
    assert best < 3.0, f"{best} ms"
