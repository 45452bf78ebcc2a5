"""Clipping tells autograd what it changed, like every in-place operation."""

import pytest
import torch

from src import grads

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def test_a_saved_gradient_that_is_clipped_is_an_error():
    g = torch.ones(1000, device=DEV)
    w = torch.ones(1000, device=DEV, requires_grad=True)
    loss = (w * g).sum()                                           # saves g
    grads.clip_grad_norm([g], 0.5)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()


def test_version_counters():
    g, h = torch.ones(1000, device=DEV), torch.ones((30, 40), device=DEV)[:, 3:20]
    out = [torch.empty_like(g), torch.empty((30, 17), dtype=torch.bfloat16, device=DEV)]
    before = [t._version for t in (g, h, *out)]
    grads.grad_norm([g, h])
    assert [t._version for t in (g, h, *out)] == before
    grads.clip_grad_norm([g, h], 0.5, out=out)
    assert [t._version - v for t, v in zip((g, h, *out), before)] == [0, 0, 1, 1]
    norm = grads.clip_grad_norm([g, h], 0.5)
    assert [t._version - v for t, v in zip((g, h, *out), before)] == [1, 1, 1, 1]
    grads.clip_grads([g], 0.5, norm)
    assert g._version - before[0] == 2 and norm._version == 0
    with torch.inference_mode():
        t = torch.ones(10, device=DEV)
        grads.clip_grad_norm([t], 1.0)
        assert t.norm().item() == pytest.approx(1.0, rel=1e-5)
