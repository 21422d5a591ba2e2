"""Measured cases of the norm before a projection, its gradients, the routing to
experts, its gradient, and low-rank adapters beside a projection.

"norm"            r = x + residual (rounded to the residual's type, which the model keeps),
                  y = r / sqrt(mean(r^2) + eps) * (w + offset) in bf16 and, for the FP8
                  products behind it, in e4m3 with a scale per 1x128.
"norm_gradients"  the gradients with respect to r (with what flows into r besides) and w.
"route"           softmax or sigmoid scores, a bias for the choice alone, groups of experts,
                  the k best of the best groups, their weights renormalised and scaled, the
                  shared expert's gate behind them.
"route_gradient"  the weights' gradient carried back to the logits.
"adapters"        y + s_l (x A_l^T) B_l^T with an adapter l for each token, or none.

With `own` false, run() computes them in elementary torch operations, in 32 bits (the scores
that are compared with each other in 64).
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6


def _named(c, name):
    return {**c, "name": name} if name else c


def _norm(T, H, x="bf16", residual=None, codes=True, offset=0.0, name=None):
    return _named({"op": "norm", "T": T, "H": H, "x": x, "residual": residual, "codes": codes, "offset": offset}, name)


def _norm_gradients(T, H, x="bf16", residual=True, offset=0.0, name=None):
    return _named({"op": "norm_gradients", "T": T, "H": H, "x": x, "residual": residual, "offset": offset}, name)


def _route(op, T, E, K, S=0, x="bf16", scoring="softmax", bias=False, groups=1, top_groups=1, group_score="max",
           renormalise=True, scale=1.0, masked=False, name=None):
    return _named({"op": op, "T": T, "E": E, "K": K, "S": S, "x": x, "scoring": scoring, "bias": bias, "groups": groups,
                   "top_groups": top_groups, "group_score": group_score, "renormalise": renormalise, "scale": scale,
                   "masked": masked}, name)


def _adapters(T, L, R, K, N, chunk=1, name=None):
    return _named({"op": "adapters", "T": T, "L": L, "R": R, "K": K, "N": N, "chunk": chunk}, name)


def listed():
    return [
        # one user decoding: the norm before a projection or the experts
        _norm(1, 2048, residual="bf16", name="norm_t1"),
        # a ragged chunk of fp32 activations, no whole number of scale blocks
        _norm(1001, 1111, x="f32", offset=1.0, name="norm_t1001_f32"),
        # a long prefill of a wide model
        _norm(16384, 4096, residual="bf16", name="norm_t16384"),
        # a small training step
        _norm_gradients(333, 2048, name="norm_gradients_t333"),
        # a training step over a long batch
        _norm_gradients(16384, 4096, name="norm_gradients_t16384"),
        # the router of the serving batch, with the shared expert's gate
        _route("route", 64, 256, 8, S=1, name="route_t64"),
        # a long padded batch: sigmoid scores, a balancing bias, four of eight groups
        _route("route", 32768, 256, 8, scoring="sigmoid", bias=True, groups=8, top_groups=4, group_score="top2",
               scale=2.5, masked=True, name="route_t32768"),
        # a training step's router
        _route("route_gradient", 4096, 256, 8, scoring="sigmoid", scale=2.5, name="route_gradient_t4096"),
        # a long padded batch of fp32 logits over more experts, every logit with a gradient
        _route("route_gradient", 32768, 500, 6, x="f32", renormalise=False, masked=True, name="route_gradient_t32768"),
        # a serving batch in which many requests have adapters of their own
        _adapters(64, 32, 16, 2048, 2048, name="adapters_t64"),
        # a ragged chunk of a few requests, no size a whole number of tiles
        _adapters(203, 3, 12, 1111, 1500, chunk=41, name="adapters_t203_ragged"),
        # a full prefill batch of long requests through a large projection
        _adapters(8192, 8, 64, 4096, 8192, chunk=700, name="adapters_t8192"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_route(rng, op):
    while True:
        T, E = _log(rng, 1, 32768), _log(rng, 8, 512)
        if T * E <= 32768 * 500:
            break
    groups, top, score, K = 1, 1, "max", rng.randint(1, min(8, E))
    if rng.random() < 0.5 and E >= 16:
        groups = rng.choice([2, 4, 8])
        E, top = E // groups * groups, rng.randint(1, groups)
        score = rng.choice(["max", "top2"])
        K = rng.randint(1, min(8, E // groups * top))
    x, renormalise = rng.choice(["bf16", "f32"]), rng.random() < 0.7
    if op == "route_gradient" and K == 1:  # (the one weight renormalised is a constant)
        renormalise = False
    return _route(op, T, E, K, S=rng.randint(0, 1), x=x, scoring=rng.choice(["softmax", "sigmoid"]),
                  bias=rng.random() < 0.5, groups=groups, top_groups=top, group_score=score,
                  renormalise=renormalise, scale=rng.choice([1.0, 2.5]), masked=rng.random() < 0.4)


def draw(rng):
    r = rng.random()
    if r < 0.4:
        while True:
            T, H = _log(rng, 1, 16384), _log(rng, 64, 8192)
            if rng.random() < 0.6:
                H = -(-H // 128) * 128
            if T * H <= 16384 * 4096:
                break
        x, offset = rng.choice(["bf16", "bf16", "f32"]), float(rng.randint(0, 1))
        if r < 0.22:
            residual = rng.choice([None, "bf16", "f32"])
            return _norm(T, H, x=x, residual=residual, codes=rng.random() < 0.6, offset=offset)
        return _norm_gradients(T, H, x=x, residual=rng.random() < 0.7, offset=offset)
    if r < 0.7:
        return _draw_route(rng, "route" if r < 0.57 else "route_gradient")
    while True:
        T, L, R, K, N = _log(rng, 1, 8192), _log(rng, 1, 64), _log(rng, 4, 128), _log(rng, 64, 8192), _log(rng, 64, 8192)
        if rng.random() < 0.6:
            R, K, N = -(-R // 16) * 16, -(-K // 64) * 64, -(-N // 64) * 64
        if T * L * R * (K + N) <= 8192 * 512 * 12288:
            break
    return _adapters(T, L, R, K, N, chunk=_log(rng, 1, 1024) if T > 64 else 1)


# ---- inputs -----------------------------------------------------------------

INV_MAX = 0.0022321429569274187  # fp32 1 / 448 (0x3b124925)


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(1000003 * seed + 29)


def _hidden(g, T, H, dtype, std=1.0):
    """N(0, std) with every 61st channel twenty times larger, as hidden states have outlier channels."""
    x = torch.randn((T, H), generator=g, device=DEV) * std
    x[:, 7::61] *= 20.0
    return x.to(dtype)


def _logits(g, case):
    """Router logits [T, E + S], skewed over the experts, and which tokens are no padding. A
    padding token's logits are what an unused row of a batch may hold."""
    T, E, S = case["T"], case["E"], case["S"]
    z = torch.randn((T, E + S), generator=g, device=DEV) * 1.5 + torch.randn(E + S, generator=g, device=DEV)
    z = z.to(TYPES[case["x"]])
    mask = None
    if case["masked"]:
        mask = torch.rand(T, generator=g, device=DEV) < 0.8
        mask[0] = True
        z[~mask] = float("nan")
    return z, mask


def _inputs(case, seed):
    g, op = _generator(seed), case["op"]
    if op in ("norm", "norm_gradients"):
        T, H, dtype = case["T"], case["H"], TYPES[case["x"]]
        s = {"x": _hidden(g, T, H, dtype)}
        s["w"] = (torch.randn(H, generator=g, device=DEV) * 0.1 + 1.0 - case["offset"]).to(torch.bfloat16)
        s["residual"] = None
        if op == "norm" and case["residual"]:
            s["residual"] = _hidden(g, T, H, TYPES[case["residual"]], 2.0)
        if op == "norm_gradients":
            s["dy"] = (torch.randn((T, H), generator=g, device=DEV) * 1e-3).to(dtype)
            if case["residual"]:
                s["residual"] = (torch.randn((T, H), generator=g, device=DEV) * 1e-3).to(dtype)
        return s
    if op in ("route", "route_gradient"):
        z, mask = _logits(g, case)
        E, K, S = case["E"], case["K"], case["S"]
        bias = (torch.rand(E, generator=g, device=DEV) - 0.5) * 0.2 if case["bias"] else None
        s = {"logits": z, "mask": mask, "bias": bias}
        if op == "route_gradient":
            zz = z[:, :E].float() if mask is None else torch.where(mask[:, None], z[:, :E].float(), 0.0)
            ids = torch.topk(zz, K, dim=1).indices
            if S:
                ids = torch.cat([ids, torch.full((case["T"], 1), E, device=DEV)], 1)
            if mask is not None:
                ids = torch.where(mask[:, None], ids, -1)
            s["ids"] = ids.to(torch.int32).contiguous()
            s["dw"] = torch.randn((case["T"], K + S), generator=g, device=DEV) * 1e-3
        return s
    T, L, R, K, N = (case[k] for k in ("T", "L", "R", "K", "N"))
    requests = -(-T // case["chunk"])
    # a tenth of the requests use the projection alone
    who = torch.randint(0, L, (requests,), generator=g, device=DEV)
    who = torch.where(torch.rand(requests, generator=g, device=DEV) < 0.1, -1, who)
    return {"x": _hidden(g, T, K, torch.bfloat16), "y": torch.randn((T, N), generator=g, device=DEV).to(torch.bfloat16),
            "a": (torch.randn((L, R, K), generator=g, device=DEV) / math.sqrt(K)).to(torch.bfloat16),
            "b": (torch.randn((L, N, R), generator=g, device=DEV) / math.sqrt(R)).to(torch.bfloat16),
            "scale": torch.rand(L, generator=g, device=DEV) + 0.5,
            "ids": who.repeat_interleave(case["chunk"])[:T].to(torch.int32).contiguous()}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        package = os.path.join(os.getcwd(), "netra-kernel_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        from netra_moe import adapters, norm, routing

        s["norm"], s["routing"] = norm, routing
        if case["op"] == "adapters":  # weights laid out once, and the batch's plan, which all layers of a step share
            s["adapters"] = adapters.LowRankAdapters(s["a"], s["b"], s["scale"])
            s["plan"] = s["adapters"].plan(s["ids"])
        if case["op"] in ("route", "route_gradient"):
            s["rule"] = {k: case[k] for k in ("scoring", "renormalise", "scale")}
            s["rule"]["shared"] = bool(case["S"])
            if case["op"] == "route":
                s["rule"].update({k: case[k] for k in ("groups", "top_groups", "group_score")})
    return s


# ---- the plain forms ----------------------------------------------------------


def _plain_norm(s):
    case, r = s["case"], s["x"].float()
    T, H = r.shape
    out = {}
    if s["residual"] is not None:
        out["residual"] = (r + s["residual"].float()).to(s["residual"].dtype)
        r = out["residual"].float()
    y = r * torch.rsqrt((r * r).mean(dim=1, keepdim=True) + EPS) * (s["w"].float() + case["offset"])
    out["y"] = y.to(torch.bfloat16)
    if case["codes"]:
        kb = -(-H // 128)
        p = torch.nn.functional.pad(y, (0, kb * 128 - H)).view(T, kb, 128)
        scale = p.abs().amax(dim=2, keepdim=True).clamp_min(1e-10) * INV_MAX
        q = (p * (1.0 / scale)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
        out["codes"], out["scale"] = q.view(T, kb * 128)[:, :H].contiguous(), scale.view(T, kb)
    return out


def _plain_norm_gradients(s):
    r, dy = s["x"].float(), s["dy"].float()
    rstd = torch.rsqrt((r * r).mean(dim=1, keepdim=True) + EPS)
    xh, g = r * rstd, dy * (s["w"].float() + s["case"]["offset"])
    dx = rstd * (g - xh * (g * xh).mean(dim=1, keepdim=True))
    if s["residual"] is not None:
        dx = dx + s["residual"].float()
    return {"dx": dx.to(s["x"].dtype), "dw": (dy * xh).sum(dim=0)}


def _scores(z, scoring):
    if scoring == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-z))
    p = torch.exp(z - z.amax(dim=1, keepdim=True))
    return p / p.sum(dim=1, keepdim=True)


def _slope(z):
    """The sigmoid's derivative."""
    e = torch.exp(-z.abs())
    return e / (1.0 + e).square()


def _plain_route(s):
    """Scores in 64 bits: which of two near ones is larger has one answer."""
    case = s["case"]
    E, K, S, G = (case[k] for k in ("E", "K", "S", "groups"))
    z, mask = s["logits"].double(), s["mask"]
    if mask is not None:
        z = torch.where(mask[:, None], z, 0.0)
    T = z.shape[0]
    score = _scores(z[:, :E], case["scoring"])
    c = score if s["bias"] is None else score + s["bias"].double()
    if G > 1:
        inside = c.view(T, G, E // G)
        two = torch.sort(inside, dim=2, descending=True).values[:, :, :2 if case["group_score"] == "top2" else 1]
        best = torch.sort(two.sum(dim=2), dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        kept = torch.zeros((T, G), dtype=torch.bool, device=z.device).scatter_(1, best, True)
        c = torch.where(kept[:, :, None], inside, -math.inf).view(T, E)
    ids = torch.sort(c, dim=1, descending=True, stable=True).indices[:, :K]
    w = torch.gather(score, 1, ids)
    if case["renormalise"]:
        w = w / w.sum(dim=1, keepdim=True)
    w = w * case["scale"]
    if S:
        ids = torch.cat([ids, torch.full((T, 1), E, device=z.device)], 1)
        w = torch.cat([w, _scores(z[:, E:], "sigmoid")], 1)
    if mask is not None:
        ids, w = torch.where(mask[:, None], ids, -1), torch.where(mask[:, None], w, 0.0)
    return {"ids": ids.to(torch.int32), "weights": w.float()}


def _plain_route_gradient(s):
    case = s["case"]
    E, K, S = (case[k] for k in ("E", "K", "S"))
    z, mask = s["logits"].float(), s["mask"]
    ids, dw = s["ids"][:, :K].long(), s["dw"]
    if mask is not None:
        z, ids = torch.where(mask[:, None], z, 0.0), torch.where(mask[:, None], ids, 0)
    v = dw[:, :K] * case["scale"]
    grad = torch.zeros_like(z)
    chosen = torch.gather(z, 1, ids)
    # differences are taken before they are weighted: near one, 1 - p has few bits left
    across = v[:, :, None] - v[:, None, :]
    if case["scoring"] == "sigmoid":
        score = _scores(chosen, "sigmoid")
        if case["renormalise"]:
            v = (across * score[:, None, :]).sum(dim=2) / score.sum(dim=1, keepdim=True).square()
        grad.scatter_(1, ids, v * _slope(chosen))
    elif case["renormalise"]:
        p = _scores(chosen, "softmax")
        grad.scatter_(1, ids, p * (across * p[:, None, :]).sum(dim=2))
    else:
        whole = _scores(z[:, :E], "softmax")
        others = torch.scatter(whole, 1, ids, 0.0).sum(dim=1, keepdim=True)
        p = torch.gather(whole, 1, ids)
        grad[:, :E] = whole * -(v * p).sum(dim=1, keepdim=True)
        grad.scatter_(1, ids, p * (v * others + (across * p[:, None, :]).sum(dim=2)))
    if S:
        grad[:, E:] = dw[:, K:] * _slope(z[:, E:])
    if mask is not None:
        grad = torch.where(mask[:, None], grad, 0.0)
    return grad.to(s["logits"].dtype)


def _plain_adapters(s):
    L, R, K = s["a"].shape
    N = s["b"].shape[1]
    mine = (s["ids"][:, None] == torch.arange(L, device=s["ids"].device)).float() * s["scale"]
    u = (s["x"].float() @ s["a"].float().view(L * R, K).t()).view(-1, L, R) * mine[:, :, None]
    return (s["y"].float() + u.view(-1, L * R) @ s["b"].float().transpose(1, 2).reshape(L * R, N)).to(torch.bfloat16)


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        if op == "norm":
            r = s["norm"].rms_norm(s["x"], s["w"], residual=s["residual"], eps=EPS, offset=case["offset"],
                                   codes="rows" if case["codes"] else None)
            out = {"y": r.y, "residual": r.residual, "codes": r.codes, "scale": r.scale}
            return {k: v for k, v in out.items() if v is not None and (k != "residual" or s["residual"] is not None)}
        if op == "norm_gradients":
            dx, dw = s["norm"].rms_norm_gradients(s["dy"], s["x"], s["w"], residual_gradient=s["residual"], eps=EPS,
                                                  offset=case["offset"])
            return {"dx": dx, "dw": dw}
        if op == "route":
            r = s["routing"].route(s["logits"], case["K"], selection_bias=s["bias"], mask=s["mask"], **s["rule"])
            return {"ids": r.ids, "weights": r.weights}
        if op == "route_gradient":
            return s["routing"].route_gradient(s["dw"], s["logits"], s["ids"], mask=s["mask"], **s["rule"])
        return s["adapters"].add(s["y"], s["x"], s["plan"])
    if op == "norm":
        return _plain_norm(s)
    if op == "norm_gradients":
        return _plain_norm_gradients(s)
    if op == "route":
        return _plain_route(s)
    if op == "route_gradient":
        return _plain_route_gradient(s)
    return _plain_adapters(s)


def work(case):
    op, T = case["op"], case["T"]
    if op in ("norm", "norm_gradients"):
        H, size = case["H"], TYPES[case["x"]].itemsize
        if op == "norm":
            kept = 2 * TYPES[case["residual"]].itemsize if case["residual"] else 0
            codes = T * (H + 4 * -(-H // 128)) if case["codes"] else 0
            return {"bytes": T * H * (size + kept + 2) + 2 * H + codes, "flops": 6 * T * H}
        return {"bytes": T * H * size * (4 if case["residual"] else 3) + 6 * H, "flops": 10 * T * H}
    if op in ("route", "route_gradient"):
        E, K, S, size = case["E"], case["K"], case["S"], TYPES[case["x"]].itemsize
        routes, mask = 8 * T * (K + S), T if case["masked"] else 0
        if op == "route":
            return {"bytes": T * (E + S) * size + routes + mask + (4 * E if case["bias"] else 0), "flops": 6 * T * E}
        whole = case["scoring"] == "softmax" and not case["renormalise"]
        read = T * ((E if whole else K) + S) * size
        return {"bytes": read + T * (E + S) * size + routes + mask, "flops": (8 * E if whole else 8 * K) * T}
    L, R, K, N = (case[k] for k in ("L", "R", "K", "N"))
    used = min(L, -(-T // case["chunk"]))
    return {"bytes": 2 * T * (K + 2 * N) + 4 * T + used * (2 * R * (K + N) + 4), "flops": 2 * T * R * (K + N)}


# ---- the same in 64 bits ------------------------------------------------------
# Outputs of few bits are given unrounded: codes as the quotient that is rounded to e4m3. The
# residual stream's rounding is a part of the operator.


def exact(case, seed):
    s, op = _inputs(case, seed), case["op"]
    if op == "norm":
        r, out = s["x"].double(), {}
        if s["residual"] is not None:
            out["residual"] = r + s["residual"].double()
            r = out["residual"].float().to(s["residual"].dtype).double()
        H = case["H"]
        y = r / torch.sqrt(r.square().sum(1, keepdim=True) / H + EPS) * (s["w"].double() + case["offset"])
        out["y"] = y
        if case["codes"]:
            scale = torch.stack([y[:, b:b + 128].abs().amax(1) for b in range(0, H, 128)], 1).clamp_min(1e-10) * INV_MAX
            out["codes"], out["scale"] = y / scale.repeat_interleave(128, 1)[:, :H], scale
        return out
    if op == "norm_gradients":
        r = s["x"].double().requires_grad_()
        w = s["w"].double().requires_grad_()
        y = r / torch.sqrt(r.square().sum(1, keepdim=True) / case["H"] + EPS) * (w + case["offset"])
        dx, dw = torch.autograd.grad((y * s["dy"].double()).sum(), (r, w))
        return {"dx": dx if s["residual"] is None else dx + s["residual"].double(), "dw": dw}
    if op in ("route", "route_gradient"):
        E, K, S, G = (case[k] for k in ("E", "K", "S", "groups"))
        live = torch.arange(case["T"], device=DEV) if s["mask"] is None else s["mask"].nonzero().view(-1)
        z = s["logits"][live].double().requires_grad_()
        score = torch.sigmoid(z[:, :E]) if case["scoring"] == "sigmoid" else torch.softmax(z[:, :E], 1)
        if op == "route_gradient":
            ids = s["ids"][live, :K].long()
        else:
            c = score.detach() + (0.0 if s["bias"] is None else s["bias"].double())
            if G > 1:
                each = E // G
                value = c.unflatten(1, (G, each)).topk(2 if case["group_score"] == "top2" else 1, 2).values.sum(2)
                order = torch.argsort(-value, dim=1, stable=True)
                rank = torch.empty_like(order).scatter_(1, order, torch.arange(G, device=DEV).expand_as(order))
                c = c.masked_fill((rank >= case["top_groups"]).repeat_interleave(each, 1), -math.inf)
            ids = torch.argsort(-c, dim=1, stable=True)[:, :K]
        w = score.gather(1, ids)
        w = w * (case["scale"] / w.sum(1, keepdim=True) if case["renormalise"] else case["scale"])
        if S:
            w = torch.cat([w, torch.sigmoid(z[:, E:])], 1)
        if op == "route":
            out = torch.zeros((case["T"], K + S), dtype=torch.float64, device=DEV)
            out[live] = w.detach()
            return {"ids": None, "weights": out}
        out = torch.zeros((case["T"], E + S), dtype=torch.float64, device=DEV)
        out[live] = torch.autograd.grad((w * s["dw"][live].double()).sum(), z)[0]
        return out
    out = s["y"].double()
    for l in range(case["L"]):
        t = (s["ids"] == l).nonzero().view(-1)
        if t.numel():
            out[t] += (s["x"][t].double() @ s["a"][l].double().t()) @ s["b"][l].double().t() * s["scale"][l].double()
    return out
