"""The operators that train a mixture-of-experts layer around its expert MLP, as measured cases.

Four kinds of case, each one pass through an operator as a training program calls it:

  route    router logits -> top-k experts, their weights, per-expert counts, the balance loss and the
           z loss, and the gradient of all of them with respect to the logits.  With ``given`` the
           experts were chosen elsewhere and only the two losses are trained on.
  combine  backward of the weighted sum over a token's experts: gradients of the expert outputs (in
           expert order) and of the weights.
  gather   backward of the gather of token rows into expert order: the sum over a token's experts.
  clip     the global norm of a set of gradients and the gradients scaled to a largest norm, written
           to the optimizer's buffers.

``run`` computes each of them with elementary torch operations (``own = False``) or through the
package's entry points (``own = True``) on the same inputs; ``exact`` gives the definition in 64 bits.
"""

import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}

BALANCE_GRAD = 1e-2   # upstream gradients of the two losses: their usual coefficients
Z_GRAD = 1e-3


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # The last few tokens of a fine-tuning batch through a small router: launch latency.
        {"name": "route_T16_E8_k2", "op": "route", "T": 16, "E": 8, "k": 2, "type": "f32", "scoring": "softmax",
         "normalize": True, "sequences": 1, "pad": 0.0, "limited": False, "given": False},
        # The 8-expert top-2 layer at its benchmark's batch, bf16 logits (ties are common).
        {"name": "route_T16384_E8_k2_bf16", "op": "route", "T": 16384, "E": 8, "k": 2, "type": "bf16",
         "scoring": "softmax", "normalize": True, "sequences": 1, "pad": 0.0, "limited": False, "given": False},
        # The 256-expert top-8 layer at its benchmark's batch, sequences padded to one length.
        {"name": "route_T8192_E256_k8_padded", "op": "route", "T": 8192, "E": 256, "k": 8, "type": "f32",
         "scoring": "softmax", "normalize": True, "sequences": 4, "pad": 0.2, "limited": False, "given": False},
        # Odd sizes; experts outside a token's allowed groups carry -inf; weights keep the full softmax.
        {"name": "route_T4099_E60_k6_limited", "op": "route", "T": 4099, "E": 60, "k": 6, "type": "f16",
         "scoring": "softmax", "normalize": False, "sequences": 1, "pad": 0.05, "limited": True, "given": False},
        # The losses of a large accumulated batch whose experts another rule chose, per sequence.
        {"name": "loss_T131072_E256_k8_sigmoid", "op": "route", "T": 131072, "E": 256, "k": 8, "type": "bf16",
         "scoring": "sigmoid", "normalize": True, "sequences": 32, "pad": 0.1, "limited": False, "given": True},
        # Combine backward of a handful of tokens: latency.
        {"name": "combine_T64_k2_D512", "op": "combine", "T": 64, "k": 2, "D": 512, "E": 8, "type": "f32",
         "out": "f32", "pad": 0.0},
        # Combine backward of the 256-expert layer: HBM traffic of 65536 rows.
        {"name": "combine_T8192_k8_D7168", "op": "combine", "T": 8192, "k": 8, "D": 7168, "E": 256, "type": "f32",
         "out": "bf16", "pad": 0.0},
        # Gather backward of the 8-expert layer.
        {"name": "gather_T16384_k2_D4096", "op": "gather", "T": 16384, "k": 2, "D": 4096, "E": 8, "type": "f32",
         "out": "bf16", "pad": 0.0},
        # Gather backward, odd sizes with dropped tokens.
        {"name": "gather_T333_k3_D1020_dropped", "op": "gather", "T": 333, "k": 3, "D": 1020, "E": 13, "type": "bf16",
         "out": "f32", "pad": 0.1},
        # A small layer's gradients: latency.
        {"name": "clip_small", "op": "clip", "tensors": 5, "total": 50_000, "type": "f32", "out": "f32",
         "norm": "2", "flat": False},
        # A whole model's bucket of gradients: many tensors of uneven sizes, views of one flat buffer.
        {"name": "clip_200_flat_bf16", "op": "clip", "tensors": 200, "total": 60_000_000, "type": "bf16", "out": "bf16",
         "norm": "2", "flat": True},
        # The expert gradients of the 8-expert layer (dW_up and dW_down, D=4096, F=14336), f32 from the
        # backward kernels, to the bf16 gradients of its bf16 weights.
        {"name": "clip_experts_E8_D4096_F14336", "op": "clip", "tensors": 2, "total": 2 * 8 * 4096 * 14336, "type": "f32",
         "out": "bf16", "norm": "2", "flat": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 0.5 / hi)))))


def draw(rng):
    while True:
        case = _drawn(rng)
        if work(case)["bytes"] <= max(work(c)["bytes"] for c in listed() if c["op"] == case["op"]):
            return case


def _drawn(rng):
    op = rng.choice(("route", "route", "combine", "gather", "clip"))
    kind = lambda: rng.choice(("f32", "bf16", "f16"))  # noqa: E731
    if op == "route":
        E = _log_int(rng, 2, 1024)
        T = _log_int(rng, 1, min(131072, 131072 * 256 // E))
        sequences = min(T, _log_int(rng, 1, 64)) if rng.random() < 0.5 else 1
        return {"op": op, "T": max(1, T // sequences) * sequences, "E": E, "k": rng.randint(1, min(16, E)), "type": kind(),
                "scoring": rng.choice(("softmax", "sigmoid")), "normalize": rng.random() < 0.7, "sequences": sequences,
                "pad": rng.choice((0.0, 0.03, 0.3)), "limited": rng.random() < 0.3, "given": rng.random() < 0.3}
    if op in ("combine", "gather"):
        D = 4 * _log_int(rng, 1, 2048)
        k = rng.randint(1, 16)
        T = _log_int(rng, 1, min(32768, 8192 * 8 * 7168 // (k * D)))
        return {"op": op, "T": T, "k": k, "D": D, "E": max(k, _log_int(rng, 2, 512)), "type": kind(),
                "out": kind(), "pad": rng.choice((0.0, 0.0, 0.1))}
    total = _log_int(rng, 100, 400_000_000)
    return {"op": op, "tensors": min(_log_int(rng, 1, 300) if total < 100_000_000 else rng.randint(1, 50), total // 50),
            "total": total, "type": kind(), "out": kind(), "norm": rng.choice(("2", "2", "inf", "1")), "flat": True}


# ----------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _routing(T, k, E, pad, g):
    """(T, k) distinct experts per token, skewed towards low ids, some tokens dropped, and the expert order:
    row of each entry (-1: dropped) and group sizes."""
    score = torch.rand((T, E), generator=g, device=DEV) - torch.linspace(0, 0.3, E, device=DEV)
    ids = score.topk(k, dim=1).indices
    if pad:
        ids = torch.where(torch.rand((T, 1), generator=g, device=DEV) < pad, E, ids)
    flat = ids.reshape(-1)
    order = torch.argsort(flat, stable=True)
    inverse = torch.empty_like(flat)
    inverse[order] = torch.arange(T * k, device=DEV)
    inverse = torch.where(flat < E, inverse, -1).to(torch.int32).view(T, k)
    return inverse, torch.bincount(flat, minlength=E + 1)[:E].to(torch.int32)


def _sizes(tensors, total, seed):
    """Uneven tensor sizes of a given sum: most small, a few large, odd ones among them."""
    r = torch.Generator()
    r.manual_seed(seed)
    share = torch.exp(2.0 * torch.randn(tensors, generator=r, dtype=torch.float64))
    sizes = [max(1, int(s)) for s in (share / share.sum() * (total - tensors)).tolist()]
    sizes[0] += max(0, total - sum(sizes))
    return sizes


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    if case["op"] == "route":
        T, E, k = case["T"], case["E"], case["k"]
        skew = torch.randn(E, generator=g, device=DEV)
        logits = 1.5 * torch.randn((T, E), generator=g, device=DEV) + skew
        if case["limited"]:  # each token may use the experts of half the groups of four
            allowed = torch.rand((T, (E + 3) // 4), generator=g, device=DEV) < 0.5
            logits = torch.where(allowed.repeat_interleave(4, dim=1)[:, :E], logits, -math.inf)
        s["logits"] = logits.to(TYPES[case["type"]])
        s["mask"] = None
        if case["pad"]:  # sequences padded at their ends
            L = T // case["sequences"]
            keep = (1 - 2 * case["pad"] * torch.rand((case["sequences"], 1), generator=g, device=DEV)) * L
            s["mask"] = (torch.arange(L, device=DEV)[None] < keep.ceil()).reshape(T)
        s["ids"] = None
        if case["given"]:
            noise = torch.rand((T, E), generator=g, device=DEV)
            ids = (torch.sigmoid(s["logits"].float()) + 0.5 * noise).topk(k, dim=1).indices.to(torch.int32)
            s["ids"] = ids if s["mask"] is None else torch.where(s["mask"][:, None], ids, -1)
        scale = 1024.0 * T if case["type"] == "f16" else 1.0    # f16 gradients come with a loss scale
        s["d_weights"] = None if case["given"] else torch.randn((T, k), generator=g, device=DEV) * (scale / T)
        s["d_balance"] = torch.tensor(BALANCE_GRAD * scale, device=DEV)
        s["d_z"] = torch.tensor(Z_GRAD * scale, device=DEV)
    elif case["op"] == "combine":
        T, k, D = case["T"], case["k"], case["D"]
        s["inverse"], s["group_sizes"] = _routing(T, k, case["E"], case["pad"], g)
        s["y_sorted"] = torch.randn((T * k, D), generator=g, device=DEV)
        w = torch.rand((T, k), generator=g, device=DEV) + 0.1
        s["weights"] = w / w.sum(1, keepdim=True)
        s["dy"] = (torch.randn((T, D), generator=g, device=DEV) / 64).to(TYPES[case["type"]])
    elif case["op"] == "gather":
        T, k, D = case["T"], case["k"], case["D"]
        s["inverse"], _ = _routing(T, k, case["E"], case["pad"], g)
        s["dxs"] = (torch.randn((T * k, D), generator=g, device=DEV) / 64).to(TYPES[case["type"]])
    else:
        sizes = _sizes(case["tensors"], case["total"], seed if case["flat"] else 7)
        if case["tensors"] == 2:
            sizes = [case["total"] // 2, case["total"] - case["total"] // 2]
        flat = torch.randn(sum(sizes), generator=g, device=DEV).mul_(1e-2).to(TYPES[case["type"]])
        s["out_flat"] = torch.empty(sum(sizes), dtype=TYPES[case["out"]], device=DEV)
        s["grads"] = list(flat.split(sizes))
        s["out"] = list(s["out_flat"].split(sizes))
        s["norm_type"] = float(case["norm"])
        # About 0.37 of the norm that these gradients have, so that they are scaled.
        n = sum(sizes)
        s["max_norm"] = {"2": 0.37e-2 * math.sqrt(n), "1": 0.3e-2 * n, "inf": 1e-2}[case["norm"]]
    return s


# ----------------------------------------------------------------------------- the definitions
def _route(s, real):
    """ids, weights, counts, tokens, losses and the gradient of the logits in the type ``real``."""
    E, k, S = s["E"], s["k"], s["sequences"]
    logits = s["logits"].to(real)
    T = logits.shape[0]
    keep = (logits > -math.inf).any(1)
    if s["mask"] is not None:
        keep = keep & s["mask"]
    safe = torch.where(keep[:, None], logits, 0)
    if s["ids"] is None:
        top, ids = torch.sort(safe, dim=1, descending=True, stable=True)
        top, ids = top[:, :k], ids[:, :k]
        ids = torch.where((top > -math.inf) & keep[:, None], ids, -1)
    else:
        ids = torch.where(keep[:, None], s["ids"].long(), -1)
    chosen = ids >= 0
    at = ids.clamp(min=0)
    m = safe.amax(1, keepdim=True)
    e = torch.exp(safe - m)
    total = e.sum(1, keepdim=True)
    p = e / total
    lse = (m + torch.log(total))[:, 0]
    if s["scoring"] == "softmax":
        score, q, slope = p, p, None
        raw = torch.where(chosen, torch.exp(safe.gather(1, at) - torch.where(chosen, safe.gather(1, at), -math.inf)
                                            .amax(1, keepdim=True).clamp(min=torch.finfo(real).min)), 0)
    else:
        score = torch.sigmoid(safe)
        sum_score = score.sum(1, keepdim=True)
        q = score / sum_score
        slope = torch.sigmoid(-safe)             # d log(sigmoid) / d logit
        raw = torch.where(chosen, score.gather(1, at), 0)
    if s["normalize"]:
        weights = raw / raw.sum(1, keepdim=True).clamp(min=torch.finfo(real).tiny)
    else:
        weights = torch.where(chosen, score.gather(1, at), 0)
    seq = torch.arange(T, device=logits.device) // (T // S)
    tokens = torch.zeros(S, dtype=torch.int64, device=logits.device).index_add_(0, seq, keep.long())
    cell = torch.where(chosen, seq[:, None] * E + at, S * E).reshape(-1)
    counts = torch.bincount(cell, minlength=S * E + 1)[:S * E].view(S, E)
    n = tokens.clamp(min=1).to(real)[:, None]
    live = (tokens > 0).sum().clamp(min=1).to(real)
    f = counts.to(real) * E / (k * n)
    mean_q = torch.where(keep[:, None], q, 0).view(S, T // S, E).sum(1) / n
    balance = (f * mean_q).sum() / live
    all_tokens = tokens.sum().clamp(min=1).to(real)
    z = torch.where(keep, lse * lse, 0).sum() / all_tokens
    # Gradient.  Since sum(q) = 1 any constant may be taken off f: f - 1 keeps what matters in few bits.
    fc = ((counts * E - k * tokens[:, None]).to(real) / (k * n))[seq]
    scale = s["d_balance"].to(real) / (live * n[seq])
    centred = q * (fc - (fc * q).sum(1, keepdim=True))
    d = scale * (centred if slope is None else centred * slope)
    d = d + s["d_z"].to(real) * 2 / all_tokens * lse[:, None] * p
    if s["d_weights"] is not None:
        dw = torch.where(chosen, s["d_weights"].to(real), 0)
        dot = (dw * weights).sum(1, keepdim=True)
        g = dw
        if s["normalize"]:
            g = weights * (dw - dot)
        elif s["scoring"] == "softmax":
            g = weights * dw
            d = d - p * dot
        else:
            g = weights * dw
        if slope is not None:
            g = g * slope.gather(1, at)
        d = d.scatter_add(1, at, torch.where(chosen, g, 0))
    d = torch.where(keep[:, None], d, 0)
    return {"ids": ids.to(torch.int32), "weights": weights, "counts": counts.to(torch.int32),
            "tokens": tokens.to(torch.int32), "balance": balance, "z": z, "d_logits": d}


def _combine(s, real):
    inverse, dy = s["inverse"], s["dy"].to(real)
    (T, k), (N, D) = inverse.shape, s["y_sorted"].shape
    ok = inverse >= 0
    rows = s["y_sorted"][inverse.clamp(min=0).reshape(-1).long()].to(real).view(T, k, D)
    dw = torch.where(ok, (rows * dy[:, None]).sum(-1), 0)
    dys = torch.zeros((N + 1, D), dtype=real, device=dy.device)
    dys[torch.where(ok, inverse, N).reshape(-1).long()] = (s["weights"].to(real)[..., None] * dy[:, None]).view(T * k, D)
    return dys[:N], dw


def _gather(s, real):
    inverse = s["inverse"]
    T, k = inverse.shape
    rows = s["dxs"][inverse.clamp(min=0).reshape(-1).long()].to(real).view(T, k, -1)
    return torch.where((inverse >= 0)[..., None], rows, 0).sum(1)


def _norm(grads, norm_type):
    if norm_type == math.inf:
        return torch.stack([t.abs().max() for t in grads]).max().double()
    if norm_type == 1:
        return torch.stack([t.float().abs().sum(dtype=torch.float64) for t in grads]).sum()
    return torch.stack([t.float().square().sum(dtype=torch.float64) for t in grads]).sum().sqrt()


def run(state):
    s = state
    if own:
        return _run_own(s)
    if s["op"] == "route":
        r = _route(s, torch.float32)
        r["d_logits"] = r["d_logits"].to(s["logits"].dtype)
        return r
    if s["op"] == "combine":
        dys, dw = _combine(s, torch.float32)
        return {"dys": dys.to(TYPES[s["out"]]), "dw": dw}
    if s["op"] == "gather":
        return {"dx": _gather(s, torch.float32).to(TYPES[s["out"]])}
    norm = _norm(s["grads"], s["norm_type"])
    coef = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    [o.copy_(t.float() * coef) for o, t in zip(s["out"], s["grads"])]
    return {"norm": norm.float(), "grads": s["out_flat"]}


def _run_own(s):
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pallas-moe-kernel_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    if s["op"] == "clip":
        from src.grads import clip_grad_norm
        norm = clip_grad_norm(s["grads"], s["max_norm"], s["norm_type"], out=s["out"])
        return {"norm": norm, "grads": s["out_flat"]}
    from src import router
    if s["op"] == "route":
        how = {"mask": s["mask"], "sequences": s["sequences"], "scoring": s["scoring"], "normalize": s["normalize"]}
        r = router.route_forward_train(s["logits"], s["k"], ids=s["ids"], **how)
        d = router.route_backward(s["logits"], r, d_weights=s["d_weights"], d_balance=s["d_balance"], d_z=s["d_z"], **how)
        return {"ids": r.ids, "weights": r.weights, "counts": r.counts, "tokens": r.tokens, "balance": r.balance_loss,
                "z": r.z_loss, "d_logits": d}
    if s["op"] == "combine":
        dys, dw = router.combine_rows_backward(s["dy"], s["y_sorted"], s["inverse"], s["weights"], s["group_sizes"],
                                               dtype=TYPES[s["out"]])
        return {"dys": dys, "dw": dw}
    return {"dx": router.gather_rows_backward(s["dxs"], s["inverse"], dtype=TYPES[s["out"]])}


# ----------------------------------------------------------------------------- 64 bits
def _exact_route(s):
    """From the definition: the losses and the weighted sum of the weights as one scalar, its gradient by
    differentiation in 64 bits rather than by a formula."""
    E, k, S = s["E"], s["k"], s["sequences"]
    x = s["logits"].double()
    T = x.shape[0]
    keep = torch.isfinite(x).any(1)
    if s["mask"] is not None:
        keep &= s["mask"]
    allowed = torch.isfinite(x) & keep[:, None]
    x = torch.where(allowed, x, 0).requires_grad_()
    low = torch.where(allowed, x, -math.inf)
    low = torch.where(keep[:, None], low, 0)                    # rows that take no part: any finite row
    if s["ids"] is None:
        rank = torch.argsort(low.detach(), dim=1, descending=True, stable=True)[:, :k]
        ids = torch.where(allowed.gather(1, rank), rank, -1)
    else:
        ids = torch.where(keep[:, None], s["ids"].long(), -1)
    chosen = ids >= 0
    lse = torch.logsumexp(low, dim=1)
    if s["scoring"] == "softmax":
        score = torch.exp(low - lse[:, None])
    else:
        score = torch.where(torch.isfinite(low), torch.sigmoid(low), 0)
    weights = torch.where(chosen, score.gather(1, ids.clamp(min=0)), 0)
    if s["normalize"]:
        total = weights.sum(1, keepdim=True)
        weights = weights / torch.where(total > 0, total, 1)
    q = torch.where(keep[:, None], score / score.sum(1, keepdim=True), 0).view(S, T // S, E)
    hot = torch.zeros((T, E + 1), dtype=torch.int32, device=x.device)
    hot.scatter_add_(1, torch.where(chosen, ids, E), torch.ones_like(ids, dtype=torch.int32))
    counts = hot[:, :E].view(S, T // S, E).sum(1)
    tokens = keep.view(S, T // S).sum(1)
    n = tokens.clamp(min=1).double()[:, None]
    per_sequence = (counts.double() * E / (k * n) * (q.sum(1) / n)).sum(1)
    balance = per_sequence.sum() / (tokens > 0).sum().clamp(min=1)
    z = torch.where(keep, lse.square(), 0).sum() / tokens.sum().clamp(min=1)
    loss = balance * s["d_balance"].double() + z * s["d_z"].double()
    if s["d_weights"] is not None:
        loss = loss + (weights * s["d_weights"].double()).sum()
    d, = torch.autograd.grad(loss, x)
    d = torch.where(allowed, d, 0)
    return {"ids": None, "weights": weights.detach(), "counts": None, "tokens": None, "balance": balance.detach(),
            "z": z.detach(), "d_logits": d}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(s)
    if case["op"] == "combine":
        T, k, N = case["T"], case["k"], case["T"] * case["k"]
        token = torch.full((N,), -1, dtype=torch.int64, device=DEV)     # the entry of each row in expert order
        inv = s["inverse"].reshape(-1).long()
        entry = torch.arange(N, device=DEV)
        token[inv[inv >= 0]] = entry[inv >= 0]
        dys = torch.zeros((N, case["D"]), dtype=torch.float64, device=DEV)
        dw = torch.zeros(N, dtype=torch.float64, device=DEV)
        step = 8192
        for a in range(0, N, step):
            i = token[a:a + step]
            live = i >= 0
            i = i.clamp(min=0)
            dy = s["dy"].double()[i // k] * live[:, None]
            dys[a:a + step] = dy * s["weights"].double().reshape(-1)[i, None]
            dw.index_add_(0, i, torch.linalg.vecdot(dy, s["y_sorted"][a:a + step].double()))
        return {"dys": dys, "dw": dw.view(T, k)}
    if case["op"] == "gather":
        inv = s["inverse"].long()
        dx = torch.zeros((case["T"], case["D"]), dtype=torch.float64, device=DEV)
        for j in range(case["k"]):
            at = inv[:, j]
            dx += torch.where((at >= 0)[:, None], s["dxs"][at.clamp(min=0)].double(), 0)
        return {"dx": dx}
    p = s["norm_type"]
    norms = torch.stack([torch.linalg.vector_norm(t.double(), p) for t in s["grads"]])
    norm = torch.linalg.vector_norm(norms, p)
    coef = min(1.0, s["max_norm"] / (float(norm) + 1e-6))
    return {"norm": norm, "grads": torch.cat([t.double() * coef for t in s["grads"]])}


# ----------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "route":
        T, E, k = case["T"], case["E"], case["k"]
        b = 2 * T * E * BYTES[case["type"]]                       # logits in, their gradient out
        b += T * k * (4 + 4) + case["sequences"] * (E + 1) * 4    # ids and weights, counts
        b += T * k * 4 if not case["given"] else 0                # the weights' gradient
        b += T if case["pad"] else 0
        return {"bytes": b, "flops": 20 * T * E}
    if case["op"] == "clip":
        return {"bytes": case["total"] * (BYTES[case["type"]] + BYTES[case["out"]]), "flops": 3 * case["total"]}
    T, k, D = case["T"], case["k"], case["D"]
    rows = T * k
    if case["op"] == "combine":
        b = T * D * BYTES[case["type"]] + rows * D * (4 + BYTES[case["out"]]) + rows * 12
        return {"bytes": b, "flops": 3 * rows * D}
    return {"bytes": rows * D * BYTES[case["type"]] + T * D * BYTES[case["out"]] + rows * 4, "flops": rows * D}
