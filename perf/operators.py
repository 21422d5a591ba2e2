"""Measured cases of the block-FP8 linear layer, its gradients, the per-expert
counts and the router's balance loss.

"linear"    y = x W^T, W e4m3 [N, K] with one fp32 scale per 128x128 block, as a
            block-FP8 checkpoint holds it; x is quantised to e4m3 with a scale per
            1x128 within the call.
            y is bf16.
"gradients" dx = dy W (dy quantised per 1x128; bf16) and dW = dy^T x (of bf16 values,
            fp32).
"counts"    how many routes each expert got.
"balance"   counts, the balance loss coef * sum_e f_e P_e of the router's softmax
            (f_e = E * share of the routes, P_e = mean probability) and its
            gradient with respect to the logits.

With `own` false, run() computes them in elementary torch operations, in 32 bits.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
COEF = 0.01


def _linear(T, N, K, x="bf16", name=None):
    c = {"op": "linear", "T": T, "N": N, "K": K, "x": x}
    return {**c, "name": name} if name else c


def _gradients(T, N, K, x="bf16", name=None):
    c = {"op": "gradients", "T": T, "N": N, "K": K, "x": x}
    return {**c, "name": name} if name else c


def _counts(T, E, K, S, masked=False, name=None):
    c = {"op": "counts", "T": T, "E": E, "K": K, "S": S, "masked": masked}
    return {**c, "name": name} if name else c


def _balance(T, E, K, S, x="bf16", masked=False, name=None):
    c = {"op": "balance", "T": T, "E": E, "K": K, "S": S, "x": x, "masked": masked}
    return {**c, "name": name} if name else c


def listed():
    return [
        # one user decoding: a square projection of the layer's hidden size
        _linear(1, 2048, 2048, name="linear_t1"),
        # a few users, a projection whose rows end inside a scale block
        _linear(13, 576, 2048, name="linear_t13_ragged"),
        # the serving batch, a projection widened to twice the hidden size
        _linear(64, 4096, 2048, name="linear_t64"),
        # a ragged chunk of fp32 activations, no size a multiple of a block
        _linear(1001, 1500, 1111, x="f32", name="linear_t1001_f32"),
        # a full prefill batch through a large layer
        _linear(8192, 8192, 4096, name="linear_t8192"),
        # a small training step of a dense gate/up projection (twice 512 rows)
        _gradients(333, 1024, 2048, name="gradients_t333"),
        # a training step over a full batch
        _gradients(4096, 4096, 2048, name="gradients_t4096"),
        # per-call expert load of the serving batch, shared expert in the last slot
        _counts(64, 256, 8, 1, name="counts_t64"),
        # expert load of a long padded batch
        _counts(50001, 256, 8, 1, masked=True, name="counts_t50001"),
        # the router of the small layer
        _balance(16, 16, 2, 0, name="balance_t16"),
        # a full batch through the layer's router, logits with the shared gate's column
        _balance(4096, 256, 8, 1, name="balance_t4096"),
        # a long padded batch of fp32 logits over more experts
        _balance(32768, 500, 6, 0, x="f32", masked=True, name="balance_t32768"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    r = rng.random()
    if r < 0.65:
        most = 8192 * 8192 * 4096 // (1 if r < 0.4 else 2)
        while True:
            T, N, K = _log(rng, 1, 8192), _log(rng, 64, 8192), _log(rng, 64, 8192)
            if rng.random() < 0.5:
                N, K = -(-N // 128) * 128, -(-K // 128) * 128
            if T * N * K <= most:
                break
        x = "bf16" if rng.random() < 0.75 else "f32"
        if r < 0.4:
            return _linear(T, N, K, x=x)
        return _gradients(T, N, K, x=x)
    E = _log(rng, 8, 512)
    K, S, masked = rng.randint(1, min(8, E)), rng.randint(0, 1), rng.random() < 0.5
    if r < 0.75:
        return _counts(_log(rng, 1, 65536), E, K, S, masked=masked)
    return _balance(_log(rng, 1, 32768), E, K, S, x=rng.choice(["bf16", "f32"]), masked=masked)


# ---- inputs -----------------------------------------------------------------

INV_MAX = 0.0022321429569274187  # fp32 1 / 448 (0x3b124925)


def _blocks(n):
    return -(-n // 128)


def _activations(g, T, K, dtype):
    """N(0, 1) with every 61st channel twenty times larger, as hidden states have outlier channels."""
    x = torch.randn((T, K), generator=g, device=DEV)
    x[:, 7::61] *= 20.0
    return x.to(dtype)


def _checkpoint(g, N, K):
    """e4m3 [N, K] and fp32 scales [ceil(N/128), ceil(K/128)] of N(0, 0.02) weights."""
    nb, kb = _blocks(N), _blocks(K)
    w = torch.zeros((nb * 128, kb * 128), device=DEV)
    w[:N, :K] = torch.randn((N, K), generator=g, device=DEV) * 0.02
    w = w.view(nb, 128, kb, 128)
    scale = w.abs().amax(dim=(1, 3), keepdim=True).clamp_min(1e-10) * INV_MAX
    q = (w * (1.0 / scale)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return q.view(nb * 128, kb * 128)[:N, :K].contiguous(), scale.view(nb, kb)


def _routing(g, case):
    """Router logits [T, E + S] (skewed over the experts), the K best experts of each
    token with the shared expert behind them, and which tokens are no padding. A
    padding token's logits are what an unused row of a batch may hold."""
    T, E, K, S = (case[k] for k in ("T", "E", "K", "S"))
    logits = torch.randn((T, E + S), generator=g, device=DEV) * 1.5 + torch.randn(E + S, generator=g, device=DEV)
    logits = logits.to(TYPES[case.get("x", "bf16")])
    ids = torch.topk(logits[:, :E].float(), K, dim=1).indices
    if S:
        ids = torch.cat([ids, torch.full((T, 1), E, device=DEV)], 1)
    mask = None
    if case["masked"]:
        mask = torch.rand(T, generator=g, device=DEV) < 0.8
        logits[~mask] = float("nan")
    return logits, ids.to(torch.int32).contiguous(), mask


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(1000003 * seed + 17)
    if case["op"] in ("counts", "balance"):
        logits, ids, mask = _routing(g, case)
        return {"logits": logits[:, :case["E"]], "ids": ids, "mask": mask}
    T, N, K = case["T"], case["N"], case["K"]
    s = {"x": _activations(g, T, K, TYPES[case["x"]])}
    s["wq"], s["ws"] = _checkpoint(g, N, K)
    if case["op"] == "gradients":
        s["dy"] = (torch.randn((T, N), generator=g, device=DEV) * 1e-3).to(TYPES[case["x"]])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        package = os.path.join(os.getcwd(), "netra-kernel_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        from netra_moe import balance
        from netra_moe.linear import BlockLinear

        s["balance"] = balance
        if "wq" in s:  # the layer that a program builds once from its checkpoint
            s["layer"] = BlockLinear(s["wq"], s["ws"], gradients=case["op"] == "gradients")
    return s


# ---- the plain forms ----------------------------------------------------------


def _rows_fp8(v):
    """fp32 [t, k] -> the values [t, k] that e4m3 codes and a scale per 1x128 stand for."""
    t, k = v.shape
    kb = _blocks(k)
    p = torch.nn.functional.pad(v, (0, kb * 128 - k)).view(t, kb, 128)
    scale = p.abs().amax(dim=2, keepdim=True).clamp_min(1e-10) * INV_MAX
    q = (p * (1.0 / scale)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return (q.float() * scale).view(t, kb * 128)[:, :k]


def _weight(wq, ws):
    n, k = wq.shape
    return wq.float() * ws.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]


def _plain_counts(ids, mask, E):
    kept = (ids >= 0) & (ids < E)
    if mask is not None:
        kept = kept & mask[:, None]
    to = torch.where(kept, ids, E).view(-1).long()
    return torch.zeros(E + 1, dtype=torch.int32, device=ids.device).index_add_(0, to, torch.ones_like(to, dtype=torch.int32))[:E]


def _plain_balance(logits, ids, mask):
    T, E = logits.shape
    counts = _plain_counts(ids, mask, E)
    valid = torch.ones(T, dtype=torch.bool, device=logits.device) if mask is None else mask
    z = torch.where(valid[:, None], logits.float(), 0.0)
    p = torch.exp(z - z.amax(dim=1, keepdim=True))
    p = p / p.sum(dim=1, keepdim=True)
    p = torch.where(valid[:, None], p, 0.0)
    f = counts.float() * E / counts.sum().clamp_min(1).float()
    s = (p * f).sum(dim=1, keepdim=True)
    scale = COEF / valid.sum().clamp_min(1).float()
    return {"counts": counts, "loss": s.sum() * scale, "dlogits": (p * (f - s) * scale).to(logits.dtype)}


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        if op == "linear":
            return s["layer"].forward(s["x"])
        if op == "gradients":
            dx, dw = s["layer"].backward(s["dy"], s["x"])
            return {"dx": dx, "dw": dw}
        if op == "counts":
            return s["balance"].expert_counts(s["ids"], case["E"], mask=s["mask"])
        r = s["balance"].balance_loss(s["logits"], s["ids"], mask=s["mask"], coefficient=COEF)
        return {"counts": r.counts, "loss": r.loss, "dlogits": r.grad}
    if op == "linear":
        return (_rows_fp8(s["x"].float()) @ _weight(s["wq"], s["ws"]).t()).to(torch.bfloat16)
    if op == "gradients":
        dy, x = s["dy"].float(), s["x"].float()
        dx = (_rows_fp8(dy) @ _weight(s["wq"], s["ws"])).to(torch.bfloat16)
        dw = dy.to(torch.bfloat16).float().t() @ x.to(torch.bfloat16).float()
        return {"dx": dx, "dw": dw}
    if op == "counts":
        return _plain_counts(s["ids"], s["mask"], case["E"])
    return _plain_balance(s["logits"], s["ids"], s["mask"])


def work(case):
    T, K = case["T"], case["K"]
    if case["op"] in ("linear", "gradients"):
        N = case["N"]
        xb = TYPES[case["x"]].itemsize
        weights = N * K + 4 * _blocks(N) * _blocks(K)
        if case["op"] == "linear":
            return {"bytes": xb * T * K + weights + 2 * T * N, "flops": 2 * T * N * K}
        return {"bytes": xb * T * (K + N) + 2 * T * K + weights + 4 * N * K, "flops": 4 * T * N * K}
    E = case["E"]
    routes = 4 * T * (K + case["S"]) + (T if case["masked"] else 0) + 4 * E
    if case["op"] == "counts":
        return {"bytes": routes, "flops": T * K}
    return {"bytes": routes + 2 * TYPES[case["x"]].itemsize * T * E + 4, "flops": 8 * T * E}


# ---- the same in 64 bits ------------------------------------------------------
# The quantisation rule is part of the operator: scale = fp32(max(amax, 1e-10) *
# fp32(1/448)), code = e4m3(fp32(v * fp32(1 / scale))), to nearest, ties to even.
# Everything behind the codes and scales is in 64 bits.


def _e4m3(v):
    """float64 -> the nearest e4m3 value, ties to even, saturating at 448."""
    e = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))).clamp_min(-6.0)
    e = torch.where(torch.exp2(e) > v.abs().clamp_min(2.0 ** -6), e - 1.0, e)
    step = torch.exp2(e - 3.0)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def _quantised(v):
    """Values of v (float64) after quantisation with a scale per 128 of its last dimension."""
    out = torch.empty_like(v)
    for b in range(0, v.shape[-1], 128):
        part = v[..., b:b + 128]
        scale = (part.abs().amax(dim=-1, keepdim=True).clamp_min(float(torch.tensor(1e-10))) * INV_MAX).float().double()
        inv = (1.0 / scale).float().double()
        out[..., b:b + 128] = _e4m3((part * inv).float().double()) * scale
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "counts":
        return None
    if case["op"] == "balance":
        T, E = case["T"], case["E"]
        live = torch.arange(T, device=DEV) if s["mask"] is None else s["mask"].nonzero().view(-1)
        routes = s["ids"][live].view(-1).long()
        counts = torch.bincount(routes[(routes >= 0) & (routes < E)], minlength=E).double()
        f = counts / max(1.0, float(counts.sum())) * E
        p = torch.softmax(s["logits"][live].double(), dim=1)
        s_t = p @ f
        n = max(1, live.numel())
        grad = torch.zeros((T, E), dtype=torch.float64, device=DEV)
        grad[live] = p * (f - s_t[:, None]) * (COEF / n)
        return {"counts": None, "loss": s_t.sum() * (COEF / n), "dlogits": grad}
    w = s["wq"].double()
    for b in range(s["ws"].shape[0]):
        rows = w[128 * b:128 * (b + 1)]
        rows *= s["ws"][b].double().repeat_interleave(128)[:w.shape[1]]
    if case["op"] == "linear":
        return _quantised(s["x"].double()) @ w.t()
    dy, x = s["dy"], s["x"]
    return {"dx": _quantised(dy.double()) @ w,
            "dw": dy.to(torch.bfloat16).double().t().contiguous() @ x.to(torch.bfloat16).double()}
