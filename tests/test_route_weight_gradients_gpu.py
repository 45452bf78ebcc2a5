"""The normalised weights' gradient where it cancels: a weight that is always
one has gradient zero, and an upstream gradient that is the same for all of a
row's weights moves nothing, although the weights themselves are rounded."""

import numpy as np
import pytest
import torch

from oracle import moe_oracle as orc
from src import router

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U = 2.0 ** -24


def _case(T, E, k, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    x = 1.5 * torch.randn((T, E), generator=g, device=DEV)
    return x, torch.randn((T, k), generator=g, device=DEV), torch.randint(0, E, (T, k), generator=g, device=DEV,
                                                                          dtype=torch.int32)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E", [1, 8, 13, 60, 256, 1000])
def test_a_single_choice_has_no_gradient(E, scoring):
    x, dw, given = _case(300, E, 1, E)
    for ids in (None, given):
        r = router.route_forward_train(x, 1, ids=ids, scoring=scoring)
        assert torch.all(router.route_backward(x, r, d_weights=dw, scoring=scoring) == 0)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,k", [(8, 2), (13, 5), (60, 6), (256, 8), (300, 16)])
def test_what_all_weights_share_moves_nothing(E, k, scoring):
    x, dw, given = _case(200, E, k, E + k)
    x[5] = -float("inf")
    x[6, 1:] = -float("inf")                                       # one expert left: the other slots are empty
    for ids in (None, given):
        r = router.route_forward_train(x, k, ids=ids, scoring=scoring)
        same = torch.full((200, k), 3.7, device=DEV)
        assert torch.all(router.route_backward(x, r, d_weights=same, scoring=scoring) == 0)
        far = dw + 1e5
        d = router.route_backward(x, r, d_weights=far, scoring=scoring)
        ref = orc.route_train(x.double().cpu().numpy(), k, None if ids is None else ids.cpu().numpy(), scoring=scoring)
        far = far.double().cpu().numpy()
        refd, _ = orc.route_train_backward(ref, far)
        # Any common value may be taken off first, the first filled slot's here: what is left rounds once, the
        # weights are off by 2 (span + 80 + k) u each and enter twice, k + 8 roundings in sums and products.
        first = far[np.arange(200), np.argmax(ref["ids"] >= 0, axis=1)]
        _, scale = orc.route_train_backward(ref, far - first[:, None])
        fin = x[torch.isfinite(x)]
        span = float(fin.max() - fin.min()) + float(fin.abs().max())
        tol = (4 * (span + 80 + k) + k + 10) * U * scale + 1e-37
        assert np.all(np.abs(d.double().cpu().numpy() - refd) <= tol)
