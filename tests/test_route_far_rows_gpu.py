"""Routing of rows whose logits are finite and far from zero, between the
16-bit range and the end of f32: usual mask constants (-1e9, -1e10, -1e30) and
runaway logits, against the float64 oracle."""

import math

import numpy as np
import pytest
import torch

from oracle import moe_oracle as orc
from src import router

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
F32_MAX = 2.0 ** 128 * (1 - 2.0 ** -24)

# A score: the difference to the row's maximum rounds once, log2 e and the
# product once each (3 u |x|, and |x| < 88 where the score does not vanish), exp
# is off by at most 2 steps (4 u), sums, logistic and division by 12 u more, and
# a sum over 20 experts by at most 64 u.
SCORE = (3 * 88 + 16 + 64) * U


def _np(t):
    return t.detach().double().cpu().numpy()


def _close(got, ref, bound, dtype=torch.float32):
    got = _np(got)
    tol = bound + HALF_STEP[dtype] * (np.abs(ref) + bound)
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], ref[bad][:5], tol[bad][:5])


def _rows(value, dtype):
    g = torch.Generator(device=DEV)
    g.manual_seed(31)
    x = (torch.randn((48, 20), generator=g, device=DEV) * 1.5).to(dtype)
    x[5] = value                                                   # a row masked throughout
    step = abs(value) * torch.finfo(dtype).eps
    x[6] = value - step * torch.randint(0, 3, (20,), generator=g, device=DEV)      # a few neighbouring values
    x[7, 4:11] = value                                             # some experts masked, or some run away
    x[8] = value
    x[8, 3] = -math.inf
    x[47] = value
    return x, torch.randn((48, 4), generator=g, device=DEV), torch.randint(-1, 20, (48, 4), generator=g, device=DEV,
                                                                           dtype=torch.int32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("value", [1e5, 1e6, 2.0 ** 20, 1.5 * 2.0 ** 20, 1e9, 1e10, 1e12, 1e18, 1e20, 1e30, 9e37, 1.5e38])
@pytest.mark.parametrize("sign", [1, -1])
def test_route_far_rows(value, sign, dtype):
    x, dw, given = _rows(sign * value, dtype)
    one = torch.ones((), device=DEV)
    for scoring in ("softmax", "sigmoid"):
        for normalize in (True, False):
            for ids in (None, given):
                how = {"scoring": scoring, "normalize": normalize}
                r = router.route_forward_train(x, 4, ids=ids, **how)
                ref = orc.route_train(_np(x), 4, None if ids is None else ids.cpu().numpy(), **how)
                assert np.array_equal(r.ids.cpu().numpy(), ref["ids"])
                assert np.array_equal(r.counts.cpu().numpy(), ref["counts"]) and r.tokens.item() == 48
                _close(r.weights, ref["weights"], 2 * (SCORE + 4 * U) * ref["weights"] + 2.0 ** -126)
                over = (48 + 16) * U                               # f32 sums over the tokens
                assert abs(r.balance_loss.item() - ref["balance"]) <= (2 * SCORE + over + 2 * U) * ref["balance"]
                lse_err = SCORE + (3 * np.abs(ref["lse"]) + 4) * U  # sum, ln 2 and product round once each
                # The z loss where lse^2 summed over the rows, and its gradient, are f32 numbers.
                in_range = value <= 1e18
                if in_range:
                    z_tol = (2 * np.abs(ref["lse"]) * lse_err).sum() / 48 + (over + 3 * U) * ref["z"]
                    assert abs(r.z_loss.item() - ref["z"]) <= z_tol
                elif ref["z"] > F32_MAX:
                    assert r.z_loss.item() == math.inf
                d = router.route_backward(x, r, d_weights=dw, d_balance=one, d_z=one if in_range else None, **how)
                refd, scale = orc.route_train_backward(ref, _np(dw), 1.0, 1.0 if in_range else 0.0)
                lse_part = 2 * lse_err[:, None] / 48 * ref["p"] if in_range else 0.0
                _close(d, refd, 4 * (SCORE + (4 + 20 / 8 + 8) * U) * scale + lse_part + 1e-37, dtype)
