"""Cases of the dense path around the event memory: a Linear with its epilogue, LayerNorm, and distillation.

Next to its memory lookups a RAVEL language model does dense work: the
projections of every layer (a matrix product with bias, activation and
residual), the norms before them, and the loss on the head's logits.  Each case
here is one call (serving, ``mode = "fwd"``) or one training step
(``mode = "step"``: forward and backward) of one of three operators:

* ``linear``   y = residual + act(x W^T + b);                  d x, d W, d b, d residual
* ``norm``     y = (x - mean) / sqrt(var + eps) * g + b;       d x, d g, d b
* ``distill``  T^2 KL(teacher's top k || student), mean over
               the rows that have a teacher entry;             d logits

``run`` computes them in elementary torch operations in float32, rounded once,
or (``own``) through ``ravel_lm_b200.dense`` / ``.glue`` / ``.distill``.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_EPS = 1e-5


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decoded token through a projection: the call's latency and one read of the weights
        {"name": "linear_token", "op": "linear", "mode": "fwd", "dtype": "bf16", "M": 1, "K": 4096, "N": 4096,
         "act": "none", "bias": True, "residual": True},
        # a batch of decoded tokens through a feed-forward layer's first projection
        {"name": "linear_batch", "op": "linear", "mode": "fwd", "dtype": "bf16", "M": 24, "K": 2048, "N": 8192,
         "act": "silu", "bias": True, "residual": False},
        # the memory layer's read-out of benchmark configuration 5 (8 x 1024 tokens, 768 -> 256), training
        {"name": "linear_readout", "op": "linear", "mode": "step", "dtype": "bf16", "M": 8192, "K": 768, "N": 256,
         "act": "none", "bias": False, "residual": True},
        # a ragged packed batch and widths that are multiples of nothing, float16
        {"name": "linear_odd", "op": "linear", "mode": "step", "dtype": "f16", "M": 1999, "K": 1001, "N": 515,
         "act": "gelu", "bias": True, "residual": True},
        # a large feed-forward layer's first projection, training
        {"name": "linear_large", "op": "linear", "mode": "step", "dtype": "bf16", "M": 16384, "K": 2048, "N": 8192,
         "act": "gelu", "bias": True, "residual": False},
        # the norm before a decoded batch's projection: latency
        {"name": "norm_token", "op": "norm", "mode": "fwd", "dtype": "bf16", "M": 24, "K": 2048, "affine": True},
        # benchmark configuration 5's tokens and width, float32 training
        {"name": "norm_layer", "op": "norm", "mode": "step", "dtype": "f32", "M": 8192, "K": 256, "affine": True},
        # odd rows and width
        {"name": "norm_odd", "op": "norm", "mode": "step", "dtype": "f16", "M": 4097, "K": 1537, "affine": True},
        # benchmark configuration 3's 4 x 32768 tokens at width 1024
        {"name": "norm_large", "op": "norm", "mode": "step", "dtype": "bf16", "M": 131072, "K": 1024, "affine": True},
        # configuration 5's tokens and vocabulary, float32 logits, training
        {"name": "distill_small", "op": "distill", "mode": "step", "dtype": "f32", "M": 8192, "V": 1024, "k": 16,
         "tau": 2.0},
        # evaluation of a ragged batch on an odd vocabulary: the loss alone
        {"name": "distill_odd", "op": "distill", "mode": "fwd", "dtype": "f16", "M": 1021, "V": 32003, "k": 20,
         "tau": 1.0},
        # a large vocabulary, training
        {"name": "distill_large", "op": "distill", "mode": "step", "dtype": "bf16", "M": 8192, "V": 65536, "k": 64,
         "tau": 2.0},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A width: mostly a multiple of 64, one in four of nothing."""
    n = _spread(rng, lo, hi)
    return n if rng.random() < 0.25 else max(lo, min(hi, (n + 32) // 64 * 64))


def draw(rng):
    op = rng.choice(["linear", "norm", "distill"])
    mode = rng.choice(["fwd", "step", "step"])
    if op == "linear":
        while True:
            M, K, N = _spread(rng, 1, 16384), _width(rng, 64, 8192), _width(rng, 64, 8192)
            if M * K * N <= 16384 * 2048 * 8192 // 2:
                break
        return {"op": op, "mode": mode, "dtype": rng.choice(["bf16", "bf16", "f16"]), "M": M, "K": K, "N": N,
                "act": rng.choice(["none", "relu", "gelu", "silu"]), "bias": rng.random() < 0.7,
                "residual": rng.random() < 0.5}
    if op == "norm":
        while True:
            M, K = _spread(rng, 1, 131072), _width(rng, 64, 16384)
            if M * K <= 131072 * 1024 // 2:
                break
        return {"op": op, "mode": mode, "dtype": rng.choice(["f32", "bf16", "f16"]), "M": M, "K": K,
                "affine": rng.random() < 0.9}
    while True:
        M, V = _spread(rng, 1, 16384), _width(rng, 256, 131072)
        if M * V <= 8192 * 65536 // 2:
            break
    return {"op": op, "mode": mode, "dtype": rng.choice(["f32", "bf16", "f16"]), "M": M, "V": V,
            "k": _spread(rng, 1, 64), "tau": rng.choice([1.0, 1.5, 2.0, 4.0])}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    step = case["mode"] == "step"

    def normal(*shape, scale=1.0, shift=0.0, grad=step):
        t = torch.randn(*shape, generator=g, device="cuda")
        return t.mul_(scale).add_(shift).to(dt).requires_grad_(grad)

    s = dict(case)
    M = case["M"]
    if case["op"] == "linear":
        K, N = case["K"], case["N"]
        s["x"] = normal(M, K)
        s["w"] = normal(N, K, scale=K ** -0.5)
        s["b"] = normal(N, scale=0.2) if case["bias"] else None
        s["r"] = normal(M, N) if case["residual"] else None
        s["gy"] = normal(M, N, grad=False) if step else None
    elif case["op"] == "norm":
        K = case["K"]
        s["x"] = normal(M, K, scale=1.5, shift=0.3)
        s["w"] = normal(K, scale=0.1, shift=1.0) if case["affine"] else None
        s["b"] = normal(K, scale=0.1) if case["affine"] else None
        s["gy"] = normal(M, K, grad=False) if step else None
    else:
        V, k = case["V"], case["k"]
        s["x"] = normal(M, V, scale=2.0)
        # k distinct ids per row (an odd step around the vocabulary); one row in eight has fewer
        # entries and one in 64 none at all (padding tokens)
        start = torch.randint(0, V, (M, 1), generator=g, device="cuda")
        hop = torch.randint(1, max(2, V // max(k, 1)), (M, 1), generator=g, device="cuda")
        ids = (start + hop * torch.arange(k, device="cuda")) % V
        kept = torch.randint(1, k + 1, (M,), generator=g, device="cuda")
        row = torch.arange(M, device="cuda")
        n = torch.where(row % 8 == 3, kept, torch.full_like(kept, k))
        n = torch.where(row % 64 == 11, torch.zeros_like(n), n)
        s["ids"] = torch.where(torch.arange(k, device="cuda") < n[:, None], ids, torch.full_like(ids, -1))
        t = torch.randn(M, k, generator=g, device="cuda") * 2.0 + 4.0
        s["t"] = torch.sort(t, dim=1, descending=True)[0].to(dt)
    return s


# ------------------------------------------------------------------ one pass
def _act(z, act):
    if act == "relu":
        return z.clamp_min(0.0)
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        sg = 1.0 / (1.0 + torch.exp(-z))
        return sg * (1.0 + z * (1.0 - sg))
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    return torch.ones_like(z)


def _plain_linear(s):
    dt = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].float()
    y = _act(z, s["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    out = {"y": y.to(dt)}
    if s["mode"] == "step":
        gy = s["gy"].float()
        dz = gy * _act_grad(z, s["act"]) if s["act"] != "none" else gy
        out["dx"] = (dz @ w).to(dt)
        out["dw"] = (dz.t() @ x).to(dt)
        if s["b"] is not None:
            out["db"] = dz.sum(0).to(dt)
        if s["r"] is not None:
            out["dr"] = s["gy"]
    return out


def _plain_norm(s):
    dt = s["x"].dtype
    x = s["x"].float()
    xc = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((xc * xc).mean(1, keepdim=True) + _EPS)
    xh = xc * rstd
    y = xh * s["w"].float() + s["b"].float() if s["affine"] else xh
    out = {"y": y.to(dt)}
    if s["mode"] == "step":
        gy = s["gy"].float()
        gw = gy * s["w"].float() if s["affine"] else gy
        dx = rstd * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
        out["dx"] = dx.to(dt)
        if s["affine"]:
            out["dw"] = (gy * xh).sum(0).to(dt)
            out["db"] = gy.sum(0).to(dt)
    return out


def _plain_distill(s):
    tau = s["tau"]
    x = s["x"].float() / tau
    ids, live = s["ids"].clamp_min(0), s["ids"] >= 0
    t = torch.where(live, s["t"].float() / tau, torch.full_like(s["t"], float("-inf"), dtype=torch.float32))
    full = live.any(1)
    tm = torch.where(full, t.max(1)[0], torch.zeros_like(t[:, 0]))
    e = torch.exp(t - tm[:, None])
    z = torch.where(full, e.sum(1), torch.ones_like(tm))
    p = e / z[:, None]
    logp = torch.where(live, t - (tm + torch.log(z))[:, None], torch.zeros_like(t))
    m = x.max(1, keepdim=True)[0]
    ex = torch.exp(x - m)
    tot = ex.sum(1, keepdim=True)
    logq = x.gather(1, ids) - (m + torch.log(tot))
    loss = torch.where(full, tau * tau * (p * (logp - torch.where(live, logq, torch.zeros_like(logq)))).sum(1),
                       torch.zeros_like(tm))
    count = full.sum().clamp_min(1)
    out = {"loss": loss.sum() / count}
    if s["mode"] == "step":
        q = ex / tot
        q.scatter_add_(1, ids, -p)
        out["dx"] = (q * (full[:, None] * (tau / count))).to(s["x"].dtype)
    return out


def _own_linear(s):
    from ravel_lm_b200.dense import fused_linear
    y = fused_linear(s["x"], s["w"], s["b"], activation=s["act"], residual=s["r"])
    if s["mode"] != "step":
        return {"y": y}
    names = [n for n in ("x", "w", "b", "r") if s[n] is not None]
    grads = torch.autograd.grad(y, [s[n] for n in names], s["gy"])
    return {"y": y, **{"d" + n: v for n, v in zip(names, grads)}}


def _own_norm(s):
    from ravel_lm_b200.glue import layer_norm
    y = layer_norm(s["x"], s["w"], s["b"], _EPS)
    if s["mode"] != "step":
        return {"y": y}
    names = [n for n in ("x", "w", "b") if s[n] is not None]
    grads = torch.autograd.grad(y, [s[n] for n in names], s["gy"])
    return {"y": y, **{"d" + n: v for n, v in zip(names, grads)}}


def _own_distill(s):
    from ravel_lm_b200.distill import distill_topk_loss
    loss = distill_topk_loss(s["x"], s["ids"], s["t"], temperature=s["tau"])
    if s["mode"] != "step":
        return {"loss": loss}
    return {"loss": loss, "dx": torch.autograd.grad(loss, [s["x"]])[0]}


def run(state):
    if own:
        return {"linear": _own_linear, "norm": _own_norm, "distill": _own_distill}[state["op"]](state)
    with torch.no_grad():
        return {"linear": _plain_linear, "norm": _plain_norm, "distill": _plain_distill}[state["op"]](state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    e, M, step = _BYTES[case["dtype"]], case["M"], case["mode"] == "step"
    if case["op"] == "linear":
        K, N, b, r = case["K"], case["N"], int(case["bias"]), int(case["residual"])
        n = M * K + N * K + b * N + r * M * N + M * N                      # x, W, b, residual in; y out
        if step:
            n += M * N + M * K + N * K + b * N                             # grad in; d x, d W, d b out (d residual is the grad)
        return {"bytes": n * e, "flops": 2.0 * M * N * K * (3 if step else 1)}
    if case["op"] == "norm":
        K, a = case["K"], int(case["affine"])
        n = 2 * M * K + 2 * a * K
        if step:
            n += 2 * M * K + 2 * a * K                                     # x is counted once for both directions
        return {"bytes": n * e, "flops": M * K * (16.0 if step else 8.0)}
    V, k = case["V"], case["k"]
    n = M * V * e * (2 if step else 1) + M * k * (8 + e) + 4               # logits in (and their gradient out), ids, teacher
    return {"bytes": n, "flops": M * V * (8.0 if step else 4.0)}


# ------------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    step = case["mode"] == "step"
    with torch.no_grad():
        x = s["x"].detach().double()
        if case["op"] == "linear":
            w = s["w"].detach().double()
            z = torch.mm(x, w.T)
            if case["bias"]:
                z += s["b"].detach().double()
            cdf = torch.special.ndtr(z) if case["act"] == "gelu" else torch.sigmoid(z)
            f = {"none": lambda: z, "relu": lambda: torch.relu(z), "silu": lambda: z * cdf, "gelu": lambda: z * cdf}
            y = f[case["act"]]()
            if case["residual"]:
                y = y + s["r"].detach().double()
            out = {"y": y}
            if step:
                dz = s["gy"].double()
                if case["act"] == "relu":
                    dz = torch.where(z > 0, dz, torch.zeros_like(dz))
                elif case["act"] == "silu":
                    dz = dz * (cdf + z * cdf * (1 - cdf))
                elif case["act"] == "gelu":
                    dz = dz * (cdf + z * torch.exp(-z * z / 2) * (2 * math.pi) ** -0.5)
                out["dx"] = torch.mm(dz, w)
                out["dw"] = torch.mm(dz.T, x)
                if case["bias"]:
                    out["db"] = dz.sum(dim=0)
                if case["residual"]:
                    out["dr"] = s["gy"].double()
            return out
        if case["op"] == "norm":
            K = case["K"]
            mean = x.sum(1, keepdim=True) / K
            var = ((x - mean) ** 2).sum(1, keepdim=True) / K
            inv = (var + _EPS) ** -0.5
            xh = (x - mean) * inv
            w = s["w"].detach().double() if case["affine"] else torch.ones(K, dtype=torch.float64, device=x.device)
            b = s["b"].detach().double() if case["affine"] else torch.zeros(K, dtype=torch.float64, device=x.device)
            out = {"y": torch.addcmul(b, xh, w)}
            if step:
                gy = s["gy"].double()
                a = gy * w
                # the Jacobian of (x - mean) * inv applied to a
                c1 = a.sum(1, keepdim=True) / K
                c2 = (a * xh).sum(1, keepdim=True) / K
                out["dx"] = (a - c1 - xh * c2) * inv
                if case["affine"]:
                    out["dw"] = torch.einsum("mk,mk->k", gy, xh)
                    out["db"] = torch.einsum("mk->k", gy)
            return out
        tau, ids = case["tau"], s["ids"]
        M, V = x.shape
        live = ids >= 0
        full = live.any(dim=1)
        n = max(1, int(full.sum()))
        t = (s["t"].double() / tau).masked_fill(~live, float("-inf")).masked_fill(~full[:, None], 0.0)
        logp = torch.log_softmax(t, dim=1)
        p = torch.exp(logp) * full[:, None]
        x.div_(tau)
        lse = torch.logsumexp(x, dim=1)
        entropy = torch.special.xlogy(p, p).sum(1)
        cross = (p * (lse[:, None] - torch.gather(x, 1, ids.clamp(min=0)))).sum(1)
        out = {"loss": ((entropy + cross) * full).sum() * (tau * tau / n)}
        if step:
            d = x.sub_(lse[:, None]).exp_()
            d.scatter_add_(1, ids.clamp(min=0), -p)
            out["dx"] = d.mul_((full * (tau / n))[:, None])
        return out
