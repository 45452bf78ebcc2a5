"""Clipping of tensors that share memory: refused with nothing written; what only interleaves is scaled once."""

import pytest
import torch

from src import _lib, grads

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def test_shared_memory_is_refused():
    m = torch.ones((50, 64), device=DEV)
    norm = grads.grad_norm([m])
    a, b = torch.ones(100, device=DEV), torch.ones(100, device=DEV)
    flat = torch.ones(101, device=DEV)
    for ts, out in (([m[:, :20], m[:, 10:30]], None), ([m[:, :20], m[3]], None), ([a, b], [b, a]), ([a, b], [b, b.clone()]),
                    ([flat[1:]], [flat[:-1]]), ([m, m], [m, m])):
        for call in (lambda: grads.clip_grad_norm(ts, 0.5, out=out), lambda: grads.clip_grads(ts, 0.5, norm, out=out)):
            with pytest.raises(_lib.MoeError, match="share"):
                call()
    with pytest.raises(_lib.MoeError, match="norm"):
        grads.clip_grads([a], 0.5, a[7])
    torch.cuda.synchronize()
    assert all(torch.all(t == 1) for t in (m, a, b, flat))


def test_interleaved_slices_are_scaled_once():
    m = torch.ones((50, 64), device=DEV)
    parts = [m[:, 40:], m[:, :20], m[:, 20:40]]
    total = grads.clip_grad_norm(parts, 20.0)
    assert total.item() == pytest.approx(3200 ** 0.5, rel=1e-6)
    # One factor for all: 20 / norm rounds three times at most.
    assert torch.all((m - 20 / 3200 ** 0.5).abs() <= 20 / 3200 ** 0.5 * 8 * 2.0 ** -24)
    rows = torch.ones((6, 128), device=DEV)
    grads.clip_grad_norm([rows[::2], rows[1::2]], 1.0, out=[rows[::2], rows[1::2]])
    assert rows.norm().item() == pytest.approx(1.0, rel=1e-5)
