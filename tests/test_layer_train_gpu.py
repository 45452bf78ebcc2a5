"""The steps that train a whole MoE layer, on the GPU against the float64
oracle: routing with its losses and gradient, the backward of combine and
gather, gradient norms and clipping, and all of them together around the
expert MLP.

Tolerances count roundings.  u = 2^-24 is half a step of f32; a rounding to a
16-bit type is off by half a step of it (2^-9 relative to the next power of
two, so at most 2^-8 of the value, for bf16; 2^-11 for f16; below f16's
normal range half of 2^-24 absolute)."""

import math

import numpy as np
import pytest
import torch

from oracle import moe_oracle as orc
from src import _lib, grads, router, train
from src.kernel import swiglu_interleave

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F16_SUBNORMAL = 2.0 ** -25


def _np(t):
    return t.detach().double().cpu().numpy()


def _close(got, ref, bound, dtype=torch.float32):
    """|got - ref| <= bound (rounding in f32, absolute) + half a step of the type."""
    got, ref = _np(got), np.asarray(ref)
    tol = np.asarray(bound) + HALF_STEP[dtype] * (np.abs(ref) + np.asarray(bound))
    if dtype == torch.float16:
        tol = tol + F16_SUBNORMAL
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], ref[bad][:5], np.broadcast_to(tol, ref.shape)[bad][:5])


# ----------------------------------------------------------------------------- routing
def _check_route(logits, k, dw, *, ids=None, mask=None, sequences=1, scoring="softmax", normalize=True, d_balance=0.7,
                 d_z=0.3):
    """Forward and backward of one routing against the oracle; returns both."""
    how = {"mask": mask, "sequences": sequences, "scoring": scoring, "normalize": normalize}
    r = router.route_forward_train(logits, k, ids=ids, **how)
    scalar = lambda v: None if v is None else torch.tensor(v, device=DEV)  # noqa: E731
    d = router.route_backward(logits, r, d_weights=dw, d_balance=scalar(d_balance), d_z=scalar(d_z), **how)
    torch.cuda.synchronize()
    x = _np(logits)
    E = x.shape[1]
    ref = orc.route_train(x, k, None if ids is None else ids.cpu().numpy(), None if mask is None else mask.cpu().numpy(),
                          sequences, scoring, normalize)
    assert np.array_equal(r.ids.cpu().numpy(), ref["ids"])
    assert np.array_equal(r.counts.cpu().numpy(), ref["counts"])
    assert np.array_equal(r.tokens.cpu().numpy(), ref["tokens"])
    # A score: the argument of exp is rounded once (u |x - max|), exp is off by
    # at most 2 steps (4 u), logistic sums and divisions by 2 steps more, and a
    # sum of n positive terms by n u; weights divide two such.
    fin = x[np.isfinite(x)]
    span = float(fin.max() - fin.min()) + float(np.abs(fin).max()) if fin.size else 0.0
    score = (span + 16 + 64) * U                       # lane sums: at most 32 + 5 additions, 64 with slack
    _close(r.weights, ref["weights"], 2 * (score + k * U) * ref["weights"] + 2.0 ** -126)
    T = x.shape[0]
    over = (T + 16) * U                                # the f32 sums over tokens
    assert abs(r.balance_loss.item() - ref["balance"]) <= (2 * score + over + 2 * U) * ref["balance"] + 1e-30
    # lse: the logarithm's argument is off by `score`, the sum rounds once more.
    lse_err = score + (np.abs(ref["lse"]) + 4) * U
    z_tol = (2 * np.abs(ref["lse"]) * lse_err)[ref["keep"]].sum() / ref["total"] + (over + 3 * U) * ref["z"]
    assert abs(r.z_loss.item() - ref["z"]) <= z_tol + 1e-30
    refd, scale = orc.route_train_backward(ref, None if dw is None else _np(dw), d_balance or 0.0, d_z or 0.0)
    lse_part = abs(d_z or 0.0) * 2 * lse_err[:, None] / ref["total"] * ref["p"]
    _close(d, refd, 4 * (score + (k + E / 8 + 8) * U) * scale + lse_part + 1e-37, logits.dtype)
    assert torch.all(d[torch.from_numpy(~ref["keep"]).to(DEV)] == 0)
    assert torch.all(d[torch.isneginf(logits)] == 0)
    return r, d, ref


def _logits(T, E, dtype, seed, scale=1.5):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    x = torch.randn((T, E), generator=g, device=DEV) * scale + torch.randn(E, generator=g, device=DEV)
    return x.to(dtype), torch.randn((T, min(16, E)), generator=g, device=DEV)


@pytest.mark.parametrize("scoring,normalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("T,E,k,dtype", [(1, 1, 1, torch.float32), (1, 8, 2, torch.float32), (37, 8, 8, torch.bfloat16),
                                         (130, 13, 3, torch.float16), (65, 32, 4, torch.float32), (50, 60, 6, torch.float16),
                                         (33, 128, 16, torch.bfloat16), (96, 256, 8, torch.float32),
                                         (17, 300, 7, torch.bfloat16), (21, 1000, 16, torch.float32),
                                         (9, 1024, 2, torch.float16), (700, 2, 1, torch.bfloat16)])
def test_route_matches_oracle(T, E, k, dtype, scoring, normalize):
    x, dw = _logits(T, E, dtype, T + E)
    _check_route(x, k, dw[:, :k], scoring=scoring, normalize=normalize)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k,sequences", [(96, 8, 2, 6), (96, 64, 6, 96), (60, 256, 8, 4), (1600, 16, 4, 2)])
def test_route_masks_sequences_and_given_ids(T, E, k, sequences, scoring):
    x, dw = _logits(T, E, torch.float32, T + E)
    g = torch.Generator(device=DEV)
    g.manual_seed(T)
    mask = torch.rand(T, generator=g, device=DEV) < 0.6
    mask[:T // sequences] = False                                  # a sequence of padding only
    x[~mask] = float("nan")                                        # what is masked is never looked at
    x[T // 2:, E // 2:] = -math.inf                                # experts that a token may not use
    x[T - 1] = -math.inf                                           # nothing left
    if mask[T - 1] and sequences > 1:
        assert T // sequences >= 1
    r, _, _ = _check_route(x, k, dw[:, :k], mask=mask, sequences=sequences, scoring=scoring)
    assert torch.all(r.ids[~mask] == -1) and torch.all(r.weights[~mask] == 0)
    ids = torch.randint(-1, E + 1, (T, k), generator=g, device=DEV, dtype=torch.int32)   # -1, E, repeats
    ids[0, :] = 0
    y = torch.where(torch.isnan(x), 0.25, x)
    _check_route(y, k, dw[:, :k], ids=ids, mask=mask, sequences=sequences, scoring=scoring)
    _check_route(y, k, dw[:, :k], ids=ids, mask=mask, sequences=sequences, scoring=scoring, normalize=False)


def test_route_everything_masked_or_empty():
    x, dw = _logits(20, 8, torch.bfloat16, 0)
    for logits, mask in ((x, torch.zeros(20, dtype=torch.bool, device=DEV)), (torch.full_like(x, -math.inf), None)):
        r, d, _ = _check_route(logits, 2, dw[:, :2], mask=mask, sequences=4)
        assert r.balance_loss.item() == 0 and r.z_loss.item() == 0 and torch.all(d == 0)
    r = router.route_forward_train(x[:0], 2, sequences=3)
    assert r.ids.shape == (0, 2) and torch.all(r.counts == 0) and torch.all(r.tokens == 0)
    assert r.balance_loss.item() == 0 and r.z_loss.item() == 0
    assert router.route_backward(x[:0], r, d_z=torch.ones((), device=DEV), sequences=3).shape == (0, 8)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("shift", [-300.0, 80.0])
def test_route_far_logits(shift, scoring):
    """Rows far from zero: sigmoids that leave the f32 range keep their ratios, exponentials do not overflow."""
    x, dw = _logits(40, 24, torch.float32, 3)
    _check_route(x + shift, 4, dw[:, :4], scoring=scoring)


def test_route_lowest_value_and_single_parts():
    x, dw = _logits(64, 16, torch.float32, 4)
    x[::2, 3:9] = torch.finfo(torch.float32).min                   # masked by the type's lowest value: finite
    r = router.route_forward_train(x, 12)
    ref = orc.route_train(_np(x), 12)
    assert np.array_equal(r.ids.cpu().numpy(), ref["ids"])
    assert torch.isfinite(r.weights).all() and torch.isfinite(r.balance_loss) and torch.isfinite(r.z_loss)
    y = _logits(64, 16, torch.float32, 5)[0]
    for parts in ({"dw": dw[:, :3], "d_balance": None, "d_z": None}, {"dw": None, "d_balance": 0.5, "d_z": None},
                  {"dw": None, "d_balance": None, "d_z": 0.5}):
        _check_route(y, 3, parts["dw"], d_balance=parts["d_balance"], d_z=parts["d_z"])
    r = router.route_forward_train(y, 3)
    assert torch.all(router.route_backward(y, r) == 0)


@pytest.mark.parametrize("scoring,normalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_route_rows_of_the_lowest_value(dtype, scoring, normalize):
    """Rows masked throughout by the type's lowest value are rows of equal logits; their product with log2 e is not finite."""
    x, dw = _logits(48, 20, dtype, 14)
    x[5] = torch.finfo(dtype).min
    x[6] = torch.finfo(dtype).min
    x[6, 7] = 0.5
    x[7] = torch.finfo(dtype).max / 2
    dw = dw[:, :4]
    r = router.route_forward_train(x, 4, scoring=scoring, normalize=normalize)
    d = router.route_backward(x, r, d_weights=dw, d_balance=torch.ones((), device=DEV), scoring=scoring,
                              normalize=normalize)
    ref = orc.route_train(_np(x), 4, scoring=scoring, normalize=normalize)
    refd, scale = orc.route_train_backward(ref, _np(dw), 1.0)
    assert np.array_equal(r.ids.cpu().numpy(), ref["ids"]) and r.tokens.item() == 48
    # Arguments of exp up to 15 from the maximum (others vanish in 64 bits too): as in _check_route, 2 (15 + 80 + k) u.
    _close(r.weights, ref["weights"], 2 * 100 * U * ref["weights"] + 2.0 ** -126)
    assert abs(r.balance_loss.item() - ref["balance"]) <= 2 * 160 * U * ref["balance"]
    _close(d, refd, 4 * 120 * U * scale + 1e-37, dtype)


def test_route_nan_is_never_chosen_and_reaches_the_losses():
    x, _ = _logits(32, 8, torch.float32, 6)
    x[5, 2] = float("nan")
    r = router.route_forward_train(x, 3)
    assert 2 not in r.ids[5].tolist() and torch.all(r.ids >= 0)
    assert torch.isnan(r.balance_loss) and torch.isnan(r.z_loss)
    assert torch.isfinite(r.weights).all()
    x[7] = float("nan")                                            # nothing to choose from: takes no part
    x[5, 2] = 0.0
    r = router.route_forward_train(x, 3)
    assert torch.all(r.ids[7] == -1) and r.tokens.item() == 31 and torch.isfinite(r.balance_loss)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_route_strides_and_alignment(dtype):
    """Column slices, odd row strides, an offset start, a transposed matrix: the same values, the same results."""
    base, dw = _logits(70, 64, dtype, 7)
    want = router.route_forward_train(base, 4)
    d_want = router.route_backward(base, want, d_weights=dw[:, :4])
    wide = torch.zeros((70, 71), dtype=dtype, device=DEV)
    wide[:, 3:67] = base
    flat = torch.zeros(70 * 64 + 1, dtype=dtype, device=DEV)
    flat[1:] = base.reshape(-1)
    for view in (wide[:, 3:67], flat[1:].view(70, 64), base.t().contiguous().t()):
        assert torch.equal(view, base)
        got = router.route_forward_train(view, 4)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert torch.equal(router.route_backward(view, got, d_weights=dw[:, :4]), d_want)
    one = base[:1].expand(5, 64)                                   # rows that share memory
    assert torch.equal(router.route_forward_train(one, 4).ids, want.ids[:1].expand(5, 4))


def test_route_repeats_bit_for_bit_and_agrees_with_route_topk():
    x, dw = _logits(20000, 64, torch.float32, 8)
    a, b = (router.route_forward_train(x, 6) for _ in range(2))
    for p, q in zip(a, b):
        assert torch.equal(p, q)
    da, db = (router.route_backward(x, a, d_weights=dw[:, :6], d_balance=torch.ones((), device=DEV)) for _ in range(2))
    assert torch.equal(da, db)
    ids, w = router.route_topk(x, 6)
    assert torch.equal(ids, a.ids)
    torch.testing.assert_close(w, a.weights, rtol=1e-5, atol=1e-7)
    gs, _, _ = router.permute(a.ids, 64)
    assert torch.equal(gs, a.counts[0])


@pytest.mark.parametrize("T,E,k", [(40000, 8, 2), (30011, 256, 8)])
def test_route_long_batches(T, E, k):
    """Many blocks: sums over tokens against float64 torch on the same logits."""
    x, dw = _logits(T, E, torch.float32, 9)
    r = router.route_forward_train(x, k)
    d = router.route_backward(x, r, d_balance=torch.ones((), device=DEV), d_z=torch.ones((), device=DEV))
    p = torch.softmax(x.double(), 1)
    lse = torch.logsumexp(x.double(), 1)
    c = torch.bincount(r.ids.reshape(-1).long(), minlength=E).double()
    f = c * E / (k * T)
    assert torch.equal(r.counts[0].double(), c) and r.tokens.item() == T
    # Sums over tokens: a lane adds at most T / (8 warps x 148 blocks) + 1 rows
    # in f32 and the rest in f64; each p within (span + 80) u (see _check_route).
    span = float(x.max() - x.min()) + float(x.abs().max())
    tol = (2 * (span + 80) + T / 1000 + 50) * U
    assert abs(r.balance_loss.item() - float((f * p.mean(0)).sum())) <= tol * float((f * p.mean(0)).sum())
    assert abs(r.z_loss.item() - float((lse ** 2).mean())) <= 2 * tol * float((lse ** 2 + lse.abs()).mean())
    fc = f - 1
    ref = (p * (fc - (p * fc).sum(1, keepdim=True)) + 2 * lse[:, None] * p) / T
    mag = (p * (fc.abs() + (p * fc.abs()).sum(1, keepdim=True)) + 2 * (lse.abs() + 1)[:, None] * p) / T
    assert torch.all((d.double() - ref).abs() <= 8 * (span + 80 + E / 8) * U * mag)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k,sequences", [(12000, 256, 8, 3), (6000, 1000, 4, 2), (50000, 16, 2, 5), (2400, 64, 6, 800)])
def test_route_long_sequences(T, E, k, sequences, scoring):
    """Several sequences of many blocks each (and many of few), padded: losses and counts against float64 torch."""
    x, _ = _logits(T, E, torch.float32, T)
    L = T // sequences
    mask = torch.arange(L, device=DEV)[None] < torch.linspace(0, 1.2, sequences, device=DEV)[:, None] * L
    r = router.route_forward_train(x, k, mask=mask, sequences=sequences, scoring=scoring)
    keep = mask.reshape(T)
    s = torch.softmax(x.double(), 1) if scoring == "softmax" else torch.sigmoid(x.double())
    q = torch.where(keep[:, None], s / s.sum(1, keepdim=True), 0).view(sequences, L, E).sum(1)
    seq = (torch.arange(T, device=DEV) // L)[:, None] * E
    c = torch.bincount((seq + r.ids.long())[keep].reshape(-1), minlength=sequences * E).view(sequences, E)
    n = keep.view(sequences, L).sum(1)
    assert torch.equal(r.counts.long(), c) and torch.equal(r.tokens.long(), n) and torch.all(r.ids[~keep] == -1)
    nn = n.clamp(min=1).double()[:, None]
    want = float((c * E / (k * nn) * q / nn).sum() / (n > 0).sum())
    lse = torch.logsumexp(x.double(), 1)[keep]
    span = float(x.max() - x.min()) + float(x.abs().max())
    tol = (2 * (span + 80) + T / 1000 + 50) * U                    # see test_route_long_batches
    assert abs(r.balance_loss.item() - want) <= tol * want
    assert abs(r.z_loss.item() - float((lse ** 2).mean())) <= 2 * tol * float((lse ** 2 + lse.abs()).mean())


@pytest.mark.parametrize("scoring,normalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("E,k", [(8, 8), (20, 16), (40, 3), (130, 16)])
def test_route_given_repeats(E, k, scoring, normalize):
    """One expert several times in a row, in neighbouring slots and in slots that one lane holds."""
    x, dw = _logits(60, E, torch.float32, E + k)
    g = torch.Generator(device=DEV)
    g.manual_seed(k)
    ids = torch.randint(0, min(E, 4), (60, k), generator=g, device=DEV, dtype=torch.int32)
    ids[::3] = ids[::3, :1]
    dw = torch.randn((60, k), generator=g, device=DEV)
    _check_route(x, k, dw, ids=ids, scoring=scoring, normalize=normalize)
    r = router.route_forward_train(x, k, ids=ids, scoring=scoring, normalize=normalize)
    a, b = (router.route_backward(x, r, d_weights=dw, scoring=scoring, normalize=normalize) for _ in range(2))
    assert torch.equal(a, b)


def test_route_two_streams_at_once():
    """Calls that overlap on two streams, each with workspaces and counters of its own."""
    xs = [_logits(30000, 256, torch.float32, 20)[0], _logits(20000, 128, torch.bfloat16, 21)[0]]
    want = [router.route_forward_train(x, 8) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(8):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(router.route_forward_train(xs[i], 8))
    torch.cuda.synchronize()
    for i in (0, 1):
        for r in got[i]:
            for a, b in zip(r, want[i]):
                assert torch.equal(a, b)


def test_route_on_another_stream_and_in_a_graph():
    x, dw = _logits(500, 64, torch.float32, 10)
    how = {"sequences": 5, "scoring": "sigmoid"}
    one = torch.ones((), device=DEV)

    def step(x):
        r = router.route_forward_train(x, 4, **how)
        return (*r, router.route_backward(x, r, d_weights=dw[:, :4], d_balance=one, d_z=one, **how))
    want = step(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step(x)
    s.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for seed in (11, 12):
        new, _ = _logits(500, 64, torch.float32, seed)
        static.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step(new)):
            assert torch.equal(a, b)


def test_route_python_refusals():
    x = torch.zeros((4, 8), device=DEV)
    with pytest.raises(ValueError, match="sequences"):
        router.route_forward_train(x, 2, sequences=3)
    with pytest.raises(ValueError, match="scoring"):
        router.route_forward_train(x, 2, scoring="tanh")
    with pytest.raises(ValueError, match="k="):
        router.route_forward_train(x, 9)
    with pytest.raises(TypeError):
        router.route_forward_train(x.double(), 2)
    with pytest.raises(ValueError, match="mask"):
        router.route_forward_train(x, 2, mask=torch.ones(3, dtype=torch.bool, device=DEV))
    with pytest.raises(ValueError, match="cpu"):
        router.route_forward_train(x, 2, mask=torch.ones(4, dtype=torch.bool))
    with pytest.raises(ValueError, match="ids"):
        router.route_forward_train(x, 2, ids=torch.zeros((4, 3), dtype=torch.int32, device=DEV))
    r = router.route_forward_train(x, 2)
    with pytest.raises(ValueError, match="d_weights"):
        router.route_backward(x, r, d_weights=torch.zeros((4, 3), device=DEV))
    with pytest.raises(ValueError, match="d_balance"):
        router.route_backward(x, r, d_balance=torch.zeros(2, device=DEV))
    with pytest.raises(ValueError, match="routed"):
        router.route_backward(x[:3], r)
    with pytest.raises(TypeError, match="routed"):
        router.route_backward(x, r._replace(weights=r.weights.half()))
    with pytest.raises(TypeError, match="ids"):
        router.route_forward_train(x, 2, ids=torch.zeros((4, 2), device=DEV))


def test_route_offsets_past_32_bits_and_wide_ids():
    """Rows four billion elements from the first, and ids that 32 bits would wrap."""
    base = torch.zeros((4400, 1_000_000), dtype=torch.bfloat16, device=DEV)
    x, dw = _logits(4400, 64, torch.bfloat16, 13)
    base[:, :64] = x
    want = router.route_forward_train(x, 6)
    got = router.route_forward_train(base[:, :64], 6)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert torch.equal(router.route_backward(base[:, :64], got, d_weights=dw[:, :6]),
                       router.route_backward(x, want, d_weights=dw[:, :6]))
    ids = want.ids.long()
    ids[0, 0], ids[1, 1] = 2 ** 32 + 3, -(2 ** 32) + 5
    far = router.route_forward_train(x, 6, ids=ids)
    assert far.ids[0, 0].item() == -1 and far.ids[1, 1].item() == -1


# ----------------------------------------------------------------------------- rows
def _routing(T, k, E, drop, seed):
    rng = np.random.default_rng(seed)
    ids = np.stack([rng.permutation(E)[:k] for _ in range(T)]).astype(np.int32) if T else np.zeros((0, k), np.int32)
    ids[rng.random(T) < drop] = -1
    gs, _, inv = orc.permute_by_expert(ids, E)
    return (torch.from_numpy(np.ascontiguousarray(inv.reshape(T, k))).to(DEV, torch.int32),
            torch.from_numpy(np.asarray(gs)).to(DEV, torch.int32))


ROWS = [(1, 1, 4, 1, 0.0), (3, 2, 8, 4, 0.0), (70, 3, 60, 5, 0.3), (33, 16, 128, 16, 0.1), (129, 9, 1020, 32, 0.1),
        (40, 8, 1024, 64, 0.0), (5, 2, 7168, 8, 1.0), (64, 2, 2052, 8, 0.2)]


@pytest.mark.parametrize("T,k,D,E,drop", ROWS)
@pytest.mark.parametrize("dy_t,out_t", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32),
                                        (torch.float16, torch.float16), (torch.float32, torch.float32)])
def test_combine_backward_matches_oracle(T, k, D, E, drop, dy_t, out_t):
    inv, gs = _routing(T, k, E, drop, T + D)
    g = torch.Generator(device=DEV)
    g.manual_seed(D)
    dy = torch.randn((T, D), generator=g, device=DEV).to(dy_t)
    ys = torch.randn((T * k, D), generator=g, device=DEV)
    ys[int(gs.sum()):] = float("nan")                              # rows nobody maps to are not looked at
    w = torch.rand((T, k), generator=g, device=DEV)
    dys, dw = router.combine_rows_backward(dy, ys, inv, w, gs, dtype=out_t)
    torch.cuda.synchronize()
    ysn = np.nan_to_num(_np(ys))
    ref, refw = orc.combine_rows_backward(_np(dy), ysn, inv.cpu().numpy(), _np(w))
    assert dys.dtype == out_t
    _close(dys, ref, U * np.abs(ref), out_t)
    _, mag = orc.combine_rows_backward(np.abs(_np(dy)), np.abs(ysn), inv.cpu().numpy(), _np(w))
    # A thread adds D / (4 x 8) groups at most (8 threads a token is the least), 4 roundings each at the start,
    # then 5 + 8 additions across threads.
    _close(dw, refw, (D / 32 + 4 + 13) * U * mag)
    assert torch.all(dys[int(gs.sum()):] == 0) and torch.all(dw[inv < 0] == 0)


@pytest.mark.parametrize("T,k,D,E,drop", ROWS)
@pytest.mark.parametrize("in_t,out_t", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32),
                                        (torch.float16, torch.float16), (torch.float32, torch.float32)])
def test_gather_backward_matches_oracle(T, k, D, E, drop, in_t, out_t):
    inv, gs = _routing(T, k, E, drop, T + D)
    g = torch.Generator(device=DEV)
    g.manual_seed(D)
    dxs = torch.randn((T * k, D), generator=g, device=DEV).to(in_t)
    dxs[int(gs.sum()):] = float("nan")
    dx = router.gather_rows_backward(dxs, inv, dtype=out_t)
    torch.cuda.synchronize()
    x = np.nan_to_num(_np(dxs))
    _close(dx, orc.gather_rows_backward(x, inv.cpu().numpy()),
           k * U * orc.gather_rows_backward(np.abs(x), inv.cpu().numpy()), out_t)
    assert dx.dtype == out_t and torch.all(dx[(inv < 0).all(1)] == 0)


def test_rows_strides_bad_indexes_and_refusals():
    T, k, D, E = 50, 2, 64, 4
    inv, gs = _routing(T, k, E, 0.2, 1)
    dy, ys, w = torch.randn((T, D), device=DEV), torch.randn((T * k, D), device=DEV), torch.rand((T, k), device=DEV)
    want = router.combine_rows_backward(dy, ys, inv, w, gs)
    wide = torch.zeros((T, D + 3), device=DEV)
    wide[:, 1:D + 1] = dy
    flat = torch.zeros(T * k * D + 2, device=DEV)
    flat[2:] = ys.reshape(-1)
    got = router.combine_rows_backward(wide[:, 1:D + 1], flat[2:].view(T * k, D), inv.t().contiguous().t(),
                                       w.t().contiguous().t(), gs.long())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # dy that is one row for all tokens (the gradient of a mean).
    same = router.combine_rows_backward(dy[:1].expand(T, D), ys, inv, w, gs)
    assert torch.equal(same[0], router.combine_rows_backward(dy[:1].repeat(T, 1), ys, inv, w, gs)[0])
    assert torch.equal(router.gather_rows_backward(flat[2:].view(T * k, D), inv), router.gather_rows_backward(ys, inv))
    bad = inv.clone()
    bad[3, 0], bad[4, 1], bad[5, 0] = T * k, 2 ** 31 - 1, -7           # outside: dropped
    dropped = torch.where((bad >= 0) & (bad < T * k), bad, -1)
    assert torch.equal(router.combine_rows_backward(dy, ys, bad, w, gs)[1],
                       router.combine_rows_backward(dy, ys, dropped, w, gs)[1])
    assert torch.equal(router.gather_rows_backward(ys, bad), router.gather_rows_backward(ys, dropped))
    empty = torch.zeros((0, k), dtype=torch.int32, device=DEV)
    dys, dw = router.combine_rows_backward(dy[:0], ys, empty, w[:0], torch.zeros_like(gs))
    assert torch.all(dys == 0) and dw.shape == (0, k)
    assert router.gather_rows_backward(ys, empty).shape == (0, D)
    with pytest.raises(ValueError, match="multiple of 4"):
        router.gather_rows_backward(ys[:, :30], inv)
    with pytest.raises(TypeError):
        router.combine_rows_backward(dy, ys.bfloat16(), inv, w, gs)
    with pytest.raises(TypeError):
        router.gather_rows_backward(ys, inv.long())
    with pytest.raises(ValueError):
        router.combine_rows_backward(dy, ys, inv, w[:3], gs)
    with pytest.raises(TypeError):
        router.gather_rows_backward(ys, inv, dtype=torch.float64)


def test_rows_past_32_bits():
    T, k, D = 270_000, 2, 8192                                     # 4.4 billion elements of expert rows
    inv = torch.arange(T * k - 1, -1, -1, dtype=torch.int32, device=DEV).view(T, k)
    dxs = torch.zeros((T * k, D), dtype=torch.bfloat16, device=DEV)
    dxs[0], dxs[-1], dxs[-2] = 1.0, 2.0, 3.0
    dx = router.gather_rows_backward(dxs, inv)
    assert torch.all(dx[0] == 5.0) and torch.all(dx[-1] == 1.0) and dx[1:-1].abs().max().item() == 0
    del dxs, dx
    ys = torch.zeros((T * k, D), device=DEV)
    ys[-1], ys[0] = 2.0, 1.0
    dy = torch.zeros((T, D), dtype=torch.bfloat16, device=DEV)
    dy[0], dy[-1] = 1.0, 0.5
    w = torch.full((T, k), 0.25, device=DEV)
    gs = torch.tensor([T * k], dtype=torch.int32, device=DEV)
    dys, dw = router.combine_rows_backward(dy, ys, inv, w, gs, dtype=torch.bfloat16)
    assert dw[0].tolist() == [2.0 * D, 0.0] and dw[-1].tolist() == [0.0, 0.5 * D]
    assert torch.all(dys[-2:] == 0.25) and torch.all(dys[:2] == 0.125) and dys[2:-2].abs().max().item() == 0


# ----------------------------------------------------------------------------- gradient norm and clipping
def _tensors(sizes, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return [(torch.randn(n, generator=g, device=DEV) * scale).to(dtype) for n in sizes]


def _norm_tol(norm_type):
    # 32 terms summed in f32: the term rounds once, four chains of 8 and two
    # more additions (11 u), half of it after the root; the result rounds once.
    return {1: 12 * U, 2: 7 * U, math.inf: 0.0}[norm_type]


@pytest.mark.parametrize("norm_type", [1, 2, math.inf])
@pytest.mark.parametrize("sizes", [[1], [7, 1, 3], [33, 8192, 8193, 5], [100_003], [0, 17, 0], [3] * 49, [11] * 501,
                                   [2_000_001, 31]])
@pytest.mark.parametrize("dtype,out_t", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                         (torch.float16, torch.bfloat16), (torch.float32, torch.float16)])
def test_clip_matches_oracle(sizes, norm_type, dtype, out_t):
    ts = _tensors(sizes, dtype, sum(sizes))
    ref = [_np(t) for t in ts]
    want = orc.grad_norm(ref, norm_type)
    assert abs(grads.grad_norm(ts, norm_type).item() - want) <= _norm_tol(norm_type) * want
    for max_norm in (0.3 * want, 2.0 * want + 1.0, 0.0):
        out = [torch.full(t.shape, 7.0, dtype=out_t, device=DEV) for t in ts]
        norm = grads.clip_grad_norm(ts, max_norm, norm_type, out=out)
        assert abs(norm.item() - want) <= _norm_tol(norm_type) * want
        for o, c in zip(out, orc.clip_grads(ref, max_norm, want)):
            # The factor: the norm's error, one rounding of its own; the product rounds once more.
            _close(o, c, (_norm_tol(norm_type) + 3 * U) * np.abs(c), out_t)
        for t, r in zip(ts, ref):
            assert np.array_equal(_np(t), r)                       # the gradients are left alone
    mine = [t.clone() for t in ts]
    grads.clip_grad_norm(mine, 0.3 * want, norm_type)
    for o, c in zip(mine, orc.clip_grads(ref, 0.3 * want, want)):
        _close(o, c, (_norm_tol(norm_type) + 3 * U) * np.abs(c), dtype)
    mine = [t.clone() for t in ts]
    grads.clip_grad_norm(mine, 2.0 * want + 1.0, norm_type)
    assert all(torch.equal(a, b) for a, b in zip(mine, ts))


@pytest.mark.parametrize("scale", [1e-30, 1e-19, 1e15, 1e30])
@pytest.mark.parametrize("norm_type", [1, 2])
def test_norm_over_the_whole_range(scale, norm_type):
    """Squares that would vanish or overflow in f32."""
    ts = _tensors([5000, 77], torch.float32, 1, scale)
    ts[0][100:4000] = 0
    want = orc.grad_norm([_np(t) for t in ts], norm_type)
    assert abs(grads.grad_norm(ts, norm_type).item() - want) <= _norm_tol(norm_type) * want
    ts[0][:3] = torch.tensor([1e-38, 1e-30, 0.0], device=DEV)
    want = orc.grad_norm([_np(t) for t in ts], norm_type)
    assert abs(grads.grad_norm(ts, norm_type).item() - want) <= _norm_tol(norm_type) * want


@pytest.mark.parametrize("norm_type", [1, 2, math.inf])
def test_norm_of_nan_infinite_and_zero(norm_type):
    ts = _tensors([10_000, 50], torch.bfloat16, 2)
    ts[0][7777] = float("nan")
    assert math.isnan(grads.grad_norm(ts, norm_type).item())
    out = [torch.empty_like(t) for t in ts]
    grads.clip_grad_norm(ts, 1.0, norm_type, out=out)
    assert all(torch.isnan(o).all() for o in out)
    ts[0][7777] = -math.inf
    assert grads.clip_grad_norm(ts, 1.0, norm_type, out=out).item() == math.inf
    assert torch.isnan(out[0][7777]) and torch.all(out[1] == 0)
    zero = [torch.zeros(1000, device=DEV), torch.zeros(3, device=DEV)]
    assert grads.clip_grad_norm(zero, 1.0, norm_type).item() == 0 and torch.all(zero[0] == 0)
    nan = [torch.full((64,), float("nan"), device=DEV)]
    assert math.isnan(grads.grad_norm(nan, norm_type).item())


def test_clip_strides_offsets_and_given_norm():
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    flat = torch.randn(100_000, generator=g, device=DEV)
    fused = torch.randn((6, 40, 64), generator=g, device=DEV)
    odd = torch.randn((50, 33), generator=g, device=DEV).bfloat16()
    views = [flat[1:5000], flat[5001:5002], flat[5005:90_001], fused[..., :32], fused[..., 32:], odd[:, 3:20], odd.t()[30:]]
    ref = [_np(v) for v in views]
    want = orc.grad_norm(ref)
    before = (flat[0].item(), flat[5000].item(), flat[90_001:].clone(), odd[:, :3].clone(), odd[:, 20:30].clone())
    assert abs(grads.grad_norm(views).item() - want) <= _norm_tol(2) * want
    out = [torch.zeros((2,) + v.shape, device=DEV)[1] for v in views[:3]] + [v.clone() for v in views[3:]]
    grads.clip_grad_norm(views, 0.5 * want, out=out[:6] + [torch.zeros_like(views[6])])
    for o, c in zip(out[:6], orc.clip_grads(ref, 0.5 * want, want)):
        _close(o, c, (_norm_tol(2) + 3 * U) * np.abs(c), o.dtype)
    norm = grads.clip_grad_norm(views, 0.5 * want)
    for v, c in zip(views, orc.clip_grads(ref, 0.5 * want, want)):
        _close(v, c, (_norm_tol(2) + 3 * U) * np.abs(c), v.dtype)
    after = (flat[0].item(), flat[5000].item(), flat[90_001:], odd[:, :3], odd[:, 20:30])
    assert before[:2] == after[:2] and all(torch.equal(a, b) for a, b in zip(before[2:], after[2:]))
    assert abs(norm.item() - want) <= _norm_tol(2) * want
    total = torch.tensor(4.0, device=DEV)                          # a norm from elsewhere
    t = torch.ones(100, device=DEV)
    assert grads.clip_grads([t], 1.0, total) is total
    _close(t, np.full(100, 1 / (4 + 1e-6)), 3 * U * 0.25)


def test_clip_past_32_bits():
    """More elements than 32 bits count: dense, and rows that are a slice."""
    t = torch.zeros(2 ** 32 + 1003, dtype=torch.bfloat16, device=DEV)
    t[0], t[2 ** 32 + 5], t[-1] = 3.0, 4.0, 12.0
    assert grads.clip_grad_norm([t], 6.5).item() == 13.0
    # 6.5 / (13 + 1e-6) is 0.5 less 4e-8 of it: each product rounds to half of its element.
    assert t[0].item() == 1.5 and t[2 ** 32 + 5].item() == 2.0 and t[-1].item() == 6.0
    rows = t[:2 ** 32].view(2, 2 ** 31)[:, :2 ** 31 - 8]
    rows[0, -1], rows[1, -1] = 4.0, -6.0
    rows[0, 0] = 12.0
    assert grads.clip_grad_norm([rows], 7.0).item() == 14.0
    assert rows[0, -1].item() == 2.0 and rows[1, -1].item() == -3.0 and rows[0, 0].item() == 6.0


def test_clip_large_lists_take_the_other_path():
    """Above 155 MB the norm has a launch of its own and every block takes one unit."""
    ts = _tensors([30_000_001, 17, 12_345_678], torch.float32, 5)
    want = float(torch.cat(ts).double().square().sum().sqrt())
    out = [torch.empty_like(t, dtype=torch.bfloat16) for t in ts]
    norm = grads.clip_grad_norm(ts, 0.3 * want, out=out)
    assert abs(norm.item() - want) <= _norm_tol(2) * want
    for o, t in zip(out, ts):
        ref = t.double() * (0.3 * want / (want + 1e-6))
        assert torch.all((o.double() - ref).abs() <= ref.abs() * (2.0 ** -8 + 20 * U))
    again = [torch.empty_like(o) for o in out]
    assert torch.equal(norm, grads.clip_grad_norm(ts, 0.3 * want, out=again))
    assert all(torch.equal(a, b) for a, b in zip(out, again))
    assert grads.grad_norm(ts, math.inf).item() == max(t.abs().max().item() for t in ts)


def test_clip_repeats_on_streams_and_in_a_graph():
    ts = _tensors([300_000, 17, 40_001], torch.float32, 4)
    out = [torch.empty_like(t, dtype=torch.bfloat16) for t in ts]
    want = grads.clip_grad_norm(ts, 1.0, out=out).clone()
    ref = [o.clone() for o in out]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = grads.clip_grad_norm(ts, 1.0, out=out)
    s.synchronize()
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(out, ref))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = grads.clip_grad_norm(ts, 1.0, out=out)
    for step in range(2):
        for t in ts:
            t.mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        again = [torch.empty_like(o) for o in out]
        assert torch.equal(norm, grads.clip_grad_norm(ts, 1.0, out=again))
        assert all(torch.equal(a, b) for a, b in zip(out, again))


def test_clip_refusals():
    t = torch.ones(100, device=DEV)
    with pytest.raises(_lib.MoeError, match="twice"):
        grads.clip_grad_norm([t, t], 1.0)
    with pytest.raises(_lib.MoeError, match="twice"):
        grads.clip_grad_norm([t[:60], t[50:]], 1.0)
    grads.clip_grad_norm([t[:50], t[50:]], 100.0)
    assert grads.grad_norm([t, t]).item() == pytest.approx(math.sqrt(200), rel=1e-6)
    with pytest.raises(TypeError):
        grads.grad_norm([t.double()])
    with pytest.raises(ValueError, match="device"):
        grads.grad_norm([t, torch.ones(3)])
    with pytest.raises(ValueError, match="outputs"):
        grads.clip_grad_norm([t], 1.0, out=[])
    with pytest.raises(ValueError, match="shape"):
        grads.clip_grad_norm([t], 1.0, out=[torch.ones(99, device=DEV)])
    with pytest.raises(ValueError, match="strides"):
        grads.grad_norm([t[:1].expand(4)])
    with pytest.raises(ValueError, match="total_norm"):
        grads.clip_grads([t], 1.0, torch.ones((), device=DEV, dtype=torch.float64))
    assert grads.grad_norm([]).item() == 0 and grads.clip_grad_norm([], 1.0).item() == 0


# ----------------------------------------------------------------------------- the layer
def _layer_inputs(T, D, F, E, swiglu, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    x = r(T, D).bfloat16()
    wr = r(D, E) / D ** 0.5
    ups = [(r(E, D, F) / D ** 0.5).bfloat16() for _ in range(2 if swiglu else 1)]
    return x, wr, ups, (r(E, F, D) / F ** 0.5).bfloat16(), r(T, D)


def _layer_ref(x, logits, ups, wd, ids, keep, dy, swiglu, sequences, T, E, k):
    """The layer in torch float64 with the chosen experts fixed: (y, balance, z, gradients of the loss)."""
    leaves = [t.detach().double().requires_grad_() for t in (x, logits, *ups, wd)]
    xd, ld, *upd, wdd = leaves
    on = ids >= 0
    at = ids.clamp(min=0).long()
    w = torch.where(on, torch.softmax(ld, 1).gather(1, at), 0)
    w = w / torch.where(w.sum(1, keepdim=True) > 0, w.sum(1, keepdim=True), 1)
    y = torch.zeros_like(xd)
    for e in range(E):
        h = [xd @ u[e] for u in upd]
        h = torch.nn.functional.silu(h[0]) * h[1] if swiglu else torch.nn.functional.gelu(h[0], approximate="tanh")
        y = y + (w * (on & (at == e))).sum(1, keepdim=True) * (h @ wdd[e])
    p = torch.where(keep[:, None], torch.softmax(ld, 1), 0)
    L = T // sequences
    n = keep.view(sequences, L).sum(1)
    c = torch.stack([torch.bincount(at[s * L:(s + 1) * L][on[s * L:(s + 1) * L]], minlength=E) for s in range(sequences)])
    nn = n.clamp(min=1).double()[:, None]
    balance = (c * E / (k * nn) * p.view(sequences, L, E).sum(1) / nn).sum() / (n > 0).sum()
    z = torch.where(keep, torch.logsumexp(ld, 1) ** 2, 0).sum() / n.sum()
    loss = (y * dy.double()).sum() + 3.0 * balance + 2.0 * z
    return y, balance, z, torch.autograd.grad(loss, leaves)


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("T,D,F,E,k,sequences,padded", [(192, 256, 256, 4, 2, 1, False), (300, 256, 512, 8, 3, 3, True)])
def test_layer_trains_like_the_oracle(T, D, F, E, k, sequences, padded, swiglu):
    """Forward, losses and every gradient of one step, then clipping: within 1e-2 in the 2-norm (bf16 operands and
    intermediates, each rounded by at most 2^-8, errors adding as squares), losses within f32 rounding."""
    x, wr, ups, wd, dy = _layer_inputs(T, D, F, E, swiglu, T)
    mask = None
    if padded:
        mask = (torch.arange(T, device=DEV) % (T // sequences)) < 70
    logits = (x.float() @ wr).detach().requires_grad_()
    x.requires_grad_()
    w_in = (swiglu_interleave(*ups) if swiglu else ups[0]).detach().requires_grad_()
    wd.requires_grad_()
    y, routed = train.moe_layer_train(x, logits, w_in, wd, k, activation="swiglu" if swiglu else "gelu", mask=mask,
                                      sequences=sequences)
    ((y * dy).sum() + 3.0 * routed.balance_loss + 2.0 * routed.z_loss).backward()
    norm = grads.grad_norm([t.grad for t in (x, logits, w_in, wd)])
    torch.cuda.synchronize()
    keep = torch.ones(T, dtype=torch.bool, device=DEV) if mask is None else mask
    ry, rb, rz, rg = _layer_ref(x, logits, ups, wd, routed.ids, keep, dy, swiglu, sequences, T, E, k)
    rel = lambda a, b: ((a.double() - b).norm() / b.norm()).item()  # noqa: E731
    assert rel(y, ry) <= 1e-2
    assert routed.balance_loss.item() == pytest.approx(rb.item(), rel=1e-5)
    assert routed.z_loss.item() == pytest.approx(rz.item(), rel=1e-5)
    ref = [rg[0], rg[1]] + ([torch.from_numpy(orc.swiglu_interleave(_np(rg[2]), _np(rg[3]))).to(DEV)] if swiglu else [rg[2]]) \
        + [rg[-1]]
    for name, t, r in zip(("x", "logits", "w_in", "w_down"), (x, logits, w_in, wd), ref):
        assert t.grad.dtype == t.dtype
        assert rel(t.grad, r) <= 1e-2, name
    assert norm.item() == pytest.approx(math.sqrt(sum(float(t.grad.double().square().sum()) for t in (x, logits, w_in, wd))),
                                        rel=1e-6)
    if mask is not None:
        assert torch.all(y[~mask] == 0) and torch.all(x.grad[~mask] == 0) and torch.all(logits.grad[~mask] == 0)
        assert _lib.device_status(reset=True) == 16                # permute's report of dropped entries
    else:
        assert _lib.device_status(reset=True) == 0


def test_layer_autograd_parts_and_refusals():
    T, D, F, E, k = 64, 256, 256, 4, 2
    x, wr, ups, wd, dy = _layer_inputs(T, D, F, E, False, 9)
    logits = (x.float() @ wr).requires_grad_()
    r = train.route_topk_train(logits, k)
    (r.balance_loss * 2).backward(retain_graph=True)               # one output alone
    alone = logits.grad.clone()
    logits.grad = None
    d = router.route_backward(logits, r, d_balance=torch.full((), 2.0, device=DEV))
    assert torch.equal(alone, d)
    assert not r.ids.requires_grad and not r.counts.requires_grad
    with torch.no_grad():
        y, _ = train.moe_layer_train(x, logits, ups[0], wd, k)
    y2, _ = router.moe_layer(x, logits.detach(), ups[0], wd, k)
    assert float((y - y2).norm() / y2.norm()) <= 1e-5              # weights' exponentials differ by a few steps
    with pytest.raises(ValueError, match="logits"):
        train.moe_layer_train(x, logits[:3], ups[0], wd, k)
    with pytest.raises(TypeError):
        train.moe_layer_train(x.float(), logits, ups[0], wd, k)


def test_layer_step_in_a_graph():
    """Routing, experts, backward and clipping captured once and replayed on new tokens."""
    T, D, F, E, k = 128, 256, 256, 4, 2
    x, wr, ups, wd, dy = _layer_inputs(T, D, F, E, False, 10)
    static = x.clone()
    bf16 = [torch.empty((E, D, F), dtype=torch.bfloat16, device=DEV), torch.empty((E, F, D), dtype=torch.bfloat16, device=DEV)]

    def step(x, out):
        logits = x.float() @ wr
        r = router.route_forward_train(logits, k)
        gs, src, inv = router.permute(r.ids, E)
        xs = router.gather_rows(x, src, k)
        ys, a = train.forward_train(xs, ups[0], wd, gs)
        y = router.combine_rows(ys, inv, r.weights)
        dys, dw = router.combine_rows_backward(dy, ys, inv, r.weights, gs, dtype=torch.bfloat16)
        dxs, dwu, dwd = train.backward(xs, ups[0], wd, gs, a, dys)
        dx = router.gather_rows_backward(dxs, inv, dtype=torch.bfloat16)
        d = router.route_backward(logits, r, d_weights=dw, d_balance=torch.full((), 0.01, device=DEV))
        norm = grads.clip_grad_norm([dwu, dwd], 1.0, out=out)
        return y, dx, d, norm
    step(static, bf16)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static, bf16)
    for seed in (1, 2):
        new = _layer_inputs(T, D, F, E, False, seed)[0]
        static.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        mine = [torch.empty_like(t) for t in bf16]
        want = step(new, mine)
        torch.cuda.synchronize()
        for a, b in zip((*out, *bf16), (*want, *mine)):
            assert torch.equal(a, b)
    del graph
    assert _lib.device_status(reset=True) == 0


def test_layer_backward_in_a_graph():
    """An autograd step captured whole, on leaves without an eager graph, and replayed."""
    T, D, F, E, k = 128, 256, 256, 4, 2
    x0, wr, ups, wd, dy = _layer_inputs(T, D, F, E, False, 11)

    def leaves(x):
        return [t.detach().clone().requires_grad_() for t in (x, wr, ups[0], wd)]

    def step(x, wr, wu, wd):
        y, routed = train.moe_layer_train(x, x.float() @ wr, wu, wd, k)
        loss = (y * dy).sum() + 0.01 * routed.balance_loss
        return torch.autograd.grad(loss, (x, wr, wu, wd))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(*leaves(x0))                                          # warm-up; its graph is gone at the return
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    static = leaves(x0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for seed in (1, 2):
        new = _layer_inputs(T, D, F, E, False, seed)[0]
        with torch.no_grad():
            static[0].copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step(*leaves(new))):
            assert torch.equal(a, b)
    del graph


def test_layer_second_derivatives_are_refused():
    T, D, F, E, k = 64, 256, 256, 4, 2
    x, wr, ups, wd, dy = _layer_inputs(T, D, F, E, False, 12)
    logits = (x.float() @ wr).requires_grad_()
    r = train.route_topk_train(logits, k)
    d, = torch.autograd.grad(r.balance_loss, logits, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()
    with pytest.raises(ValueError, match="token"):
        train.moe_layer_train(x[:0], logits[:0], ups[0], wd, k)


def test_layer_with_bf16_logits_and_frozen_inputs():
    """Gradients in the leaves' own types; tokens or router that take none; an upstream gradient that is one row for all."""
    T, D, F, E, k = 96, 256, 256, 4, 2
    x, wr, ups, wd, _ = _layer_inputs(T, D, F, E, False, 15)
    logits = (x.float() @ wr).bfloat16().requires_grad_()
    wu, wdn = ups[0].clone().requires_grad_(), wd.clone().requires_grad_()
    y, routed = train.moe_layer_train(x, logits, wu, wdn, k)
    (y.sum() + routed.balance_loss).backward()
    assert logits.grad.dtype == torch.bfloat16 and wu.grad.dtype == torch.bfloat16 and x.grad is None
    dy = torch.ones((T, D), device=DEV)
    _, rb, _, rg = _layer_ref(x, logits, ups, wd, routed.ids, torch.ones(T, dtype=torch.bool, device=DEV), dy, False, 1,
                              T, E, k)
    assert routed.balance_loss.item() == pytest.approx(rb.item(), rel=1e-5)
    # _layer_ref's loss has the losses' weights 3 and 2; the experts' gradients do not depend on them.
    for name, t, r in (("w_up", wu, rg[2]), ("w_down", wdn, rg[3])):
        assert ((t.grad.double() - r).norm() / r.norm()).item() <= 1e-2, name
    leaf = x.clone().requires_grad_()
    y, _ = train.moe_layer_train(leaf, logits.detach(), ups[0], wd, k)
    y.sum().backward()
    assert leaf.grad.dtype == torch.bfloat16
    assert ((leaf.grad.double() - rg[0]).norm() / rg[0].norm()).item() <= 1e-2
    _lib.device_status(reset=True)
