"""Cases of the vocabulary's two ends and of the optimizer step.

A RAVEL training step looks its token ids up in an embedding, ends in a loss over the vocabulary, and then updates
every parameter.  Each case here is one call (``mode = "fwd"``) or one training step (``mode = "step"``) of one of
three operators:

* ``embed``  y_i = scale W[id_i];                             d W_v = scale sum_{id_i = v} g_i
* ``ce``     z = x W^T;  -log softmax(z)[target], mean over
             the rows that have one, or each row's;           d x, d W
* ``adamw``  clipping by the global norm, then for every
             tensor  m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,
             p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)

``run`` computes them in elementary torch operations in float32, rounded once, or (``own``) through
``ravel_lm_b200.vocab`` / ``.optim``.

The optimizer's states are float32 or 8 bits.  8-bit states share a power of two per block of 256 elements of a
tensor, the least that the block's largest value fits under with 1.875 times it; below that the first moment has a sign, 4 bits of exponent and 3 of
mantissa, the second moment (never negative) 5 and 3.  They are rounded stochastically, so that changes smaller than
a step count on average; the random bits are a hash of the element's index, the tensor's place in the list and the step.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_HYPER = {"lr": 1e-3, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01}
_STEP0 = 100   # steps taken before a case's first
_CLIP = 1.0
_BLOCK = 256   # elements that share a power of two


# ------------------------------------------------------------------ cases
def listed():
    return [
        # log-likelihoods of a batch of continuations' next tokens: the call's latency and one read of the head
        {"name": "ce_score", "op": "ce", "mode": "fwd", "dtype": "bf16", "M": 24, "K": 2048, "V": 32000,
         "reduction": "none"},
        # benchmark configuration 5's tokens, width and vocabulary, training
        {"name": "ce_config5", "op": "ce", "mode": "step", "dtype": "bf16", "M": 8192, "K": 256, "V": 1024,
         "reduction": "mean"},
        # a ragged packed batch, a width and a vocabulary that are multiples of nothing, float16
        {"name": "ce_odd", "op": "ce", "mode": "step", "dtype": "f16", "M": 1021, "K": 515, "V": 32003,
         "reduction": "mean"},
        # a large vocabulary, training
        {"name": "ce_large", "op": "ce", "mode": "step", "dtype": "bf16", "M": 8192, "K": 1024, "V": 65536,
         "reduction": "mean"},
        # a decoded batch's tokens: latency
        {"name": "embed_token", "op": "embed", "mode": "fwd", "dtype": "bf16", "M": 24, "K": 2048, "V": 65536,
         "scale": 1.0},
        # benchmark configuration 5's tokens, width and vocabulary in float32, training
        {"name": "embed_config5", "op": "embed", "mode": "step", "dtype": "f32", "M": 8192, "K": 256, "V": 1024,
         "scale": 16.0},
        # odd tokens, width and vocabulary
        {"name": "embed_odd", "op": "embed", "mode": "step", "dtype": "f16", "M": 4097, "K": 257, "V": 32003,
         "scale": 1.0},
        # benchmark configuration 3's 4 x 32768 tokens at width 1024
        {"name": "embed_large", "op": "embed", "mode": "step", "dtype": "bf16", "M": 131072, "K": 1024, "V": 65536,
         "scale": 32.0},
        # a small model in float32: 2 layers of width 256, 21 tensors, launches and small tensors
        {"name": "adamw_small", "op": "adamw", "mode": "step", "dtype": "f32", "bits": 32, "layers": 2, "d": 256,
         "V": 1024, "clip": True},
        # widths that are multiples of nothing, 8-bit states
        {"name": "adamw_odd", "op": "adamw", "mode": "step", "dtype": "f16", "bits": 8, "layers": 3, "d": 515,
         "V": 32003, "clip": True},
        # 118 million bfloat16 parameters with float32 masters and states
        {"name": "adamw_large", "op": "adamw", "mode": "step", "dtype": "bf16", "bits": 32, "layers": 8, "d": 1024,
         "V": 32768, "clip": False},
        # the same with 8-bit states
        {"name": "adamw_large8", "op": "adamw", "mode": "step", "dtype": "bf16", "bits": 8, "layers": 8, "d": 1024,
         "V": 32768, "clip": False},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A width: mostly a multiple of 64, one in four of nothing."""
    n = _spread(rng, lo, hi)
    return n if rng.random() < 0.25 else max(lo, min(hi, (n + 32) // 64 * 64))


def draw(rng):
    op = rng.choice(["ce", "embed", "adamw"])
    if op == "ce":
        while True:
            M, K, V = _spread(rng, 1, 16384), _width(rng, 64, 4096), _width(rng, 256, 131072)
            if M * V <= 8192 * 65536 // 2 and M * V * K <= 8192 * 65536 * 1024 // 2 and V * K <= 65536 * 1024:
                break
        mode = rng.choice(["fwd", "step", "step"])
        return {"op": op, "mode": mode, "dtype": rng.choice(["bf16", "bf16", "f16"]), "M": M, "K": K, "V": V,
                "reduction": rng.choice(["mean", "mean", "sum", "none"])}
    if op == "embed":
        while True:
            M, K, V = _spread(rng, 1, 131072), _width(rng, 64, 4096), _width(rng, 256, 131072)
            if M * K <= 131072 * 1024 // 2 and V * K <= 65536 * 1024:
                break
        return {"op": op, "mode": rng.choice(["fwd", "step", "step"]), "dtype": rng.choice(["f32", "bf16", "f16"]),
                "M": M, "K": K, "V": V, "scale": rng.choice([1.0, 16.0, 22.5])}
    while True:
        layers, d, V = rng.randint(1, 12), _width(rng, 64, 2048), _width(rng, 256, 65536)
        if V * d + layers * 10 * d * d <= 60_000_000:
            break
    return {"op": op, "mode": "step", "dtype": rng.choice(["f32", "bf16", "f16"]), "bits": rng.choice([32, 8]),
            "layers": layers, "d": d, "V": V, "clip": rng.random() < 0.5}


# ------------------------------------------------------------------ inputs
def _shapes(case):
    """The tensors of a small language model: embedding, then norms, projections and feed-forward of every layer."""
    d = case["d"]
    layer = [(d,), (d,), (d, d), (d,), (d, d), (d,), (4 * d, d), (4 * d,), (d, 4 * d)]
    return [(case["V"], d)] + layer * case["layers"] + [(d,), (d,)]


def _spans(case):
    """(start, length) of every tensor in flat buffers, each starting at a multiple of a block."""
    spans, at = [], 0
    for shape in _shapes(case):
        n = math.prod(shape)
        spans.append((at, n))
        at += (n + _BLOCK - 1) // _BLOCK * _BLOCK
    return spans, at


def _zipf(n, count, g):
    """Token ids of a Zipf distribution over n, the frequent ones anywhere in the vocabulary."""
    cdf = torch.arange(1, n + 1, dtype=torch.float64, device="cuda").pow(-1.05).cumsum(0)
    u = torch.rand(count, generator=g, dtype=torch.float64, device="cuda") * cdf[-1]
    return torch.randperm(n, generator=g, device="cuda")[torch.searchsorted(cdf, u).clamp_max(n - 1)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    step = case["mode"] == "step"

    def normal(*shape, scale=1.0, grad=step):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).to(dt).requires_grad_(grad)

    s = dict(case)
    if case["op"] == "adamw":
        spans, total = _spans(case)
        live = torch.zeros(total, device="cuda")
        for a, n in spans:
            live[a:a + n] = 1.0

        def flat(scale):
            return torch.randn(total, generator=g, device="cuda").mul_(live).mul_(scale)

        # gradients of very different sizes, as layers and frequent and rare tokens have them
        size = torch.exp(flat(1.5)).mul_(1e-4).mul_(live)
        s["g"] = flat(1.0).mul_(size).to(dt)
        m = flat(0.3).mul_(size)
        v = torch.exp(flat(0.3)).mul_(size).mul_(size)
        master = flat(0.02)
        s["p"] = master.to(dt)
        s["master"] = None if dt == torch.float32 else master.add_(flat(1e-5))
        s["step"] = torch.full((1,), _STEP0, dtype=torch.int64, device="cuda")
        if case["bits"] == 32:
            s["m"], s["v"], s["me"], s["ve"] = m, v, None, None
        else:
            r = torch.randint(0, 1 << 32, (total,), generator=g, device="cuda")
            s["m"], s["me"] = _quantise(m, r & 0xFFFF, 15)
            s["v"], s["ve"] = _quantise(v, r >> 16, 31)
        if dt != torch.float32:  # a master rounds to its parameter
            s["p"] = s["master"].to(dt)
        s["shapes"], s["spans"] = _shapes(case), spans

        def views(t):
            return None if t is None else [t[a:a + n].view(sh) for (a, n), sh in zip(spans, s["shapes"])]

        def blocks(t):
            return None if t is None else [t[a // _BLOCK:(a + n + _BLOCK - 1) // _BLOCK] for a, n in spans]

        s["params"], s["grads"], s["masters"] = views(s["p"]), views(s["g"]), views(s["master"])
        s["ms"], s["vs"], s["mes"], s["ves"] = views(s["m"]), views(s["v"]), blocks(s["me"]), blocks(s["ve"])
        return s
    M, K, V = case["M"], case["K"], case["V"]
    if case["op"] == "embed":
        s["ids"] = _zipf(V, M, g)
        s["w"] = normal(V, K, scale=K ** -0.5)
        s["gy"] = normal(M, K, grad=False) if step else None
        return s
    s["x"] = normal(M, K)
    s["w"] = normal(V, K, scale=2.0 * K ** -0.5)
    t = _zipf(V, M, g)
    # one row in 32 has no target (padding of a packed batch)
    s["t"] = torch.where(torch.arange(M, device="cuda") % 32 == 5, torch.full_like(t, -100), t)
    s["up"] = torch.rand(M, generator=g, device="cuda") if step and case["reduction"] == "none" else None
    return s


# ------------------------------------------------------------------ one pass
def _hash(i):
    """32 well-mixed bits of 32 (two multiplications between shifted exclusive ors)."""
    i = ((i ^ (i >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    i = ((i ^ (i >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return i ^ (i >> 16)


def _pow2(e):
    """2^e for whole -126 <= e <= 127, as float32."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantise(x, r, bias):
    """8-bit codes and block exponents of float32 values (whole blocks), r: 16 random bits an element."""
    b = x.view(-1, _BLOCK)
    top = b.abs().amax(1)
    e = torch.where(top == 0, -126, torch.frexp(top)[1] - 1).clamp_min(-126)
    e = e + (top > _pow2(e) * 1.875)
    # the block's largest value becomes at most 1.875; scaling by a power of two, in two steps that cannot overflow
    h = e >> 1
    y = (b.abs() * _pow2(-h)[:, None] * _pow2(h - e)[:, None]).view(-1)
    bits = (y.view(torch.int32).to(torch.int64) + (r << 4) + 8) >> 20
    normal = bits - ((127 - bias) << 3)
    tiny = torch.floor(y * 2.0 ** (bias + 2) + (r.float() + 0.5) * 2.0 ** -16).to(torch.int64)
    code = torch.where(y < 2.0 ** (1 - bias), tiny, normal)
    sign = (x < 0).to(torch.int64) << 7 if bias == 15 else 0
    return (code | sign).to(torch.uint8), e.to(torch.int8)


def _values(code, e, bias):
    """What 8-bit codes and block exponents stand for, in float32."""
    c = code.to(torch.int32)
    a = c & 0x7F if bias == 15 else c
    y = torch.where(a < 8, a.float() * 2.0 ** (-bias - 2), ((a + ((127 - bias) << 3)) << 20).view(torch.float32))
    y = (y.view(-1, _BLOCK) * _pow2(e)[:, None]).view(-1)
    return torch.where(c > 127, -y, y) if bias == 15 else y


def _plain_adamw(s):
    b1, b2 = _HYPER["betas"]
    lr, dt = _HYPER["lr"], s["p"].dtype
    t = s["step"].add_(1).double()
    c1 = (lr / (1.0 - b1 ** t)).float()
    c2 = (1.0 / torch.sqrt(1.0 - b2 ** t)).float()
    g = s["g"].float()
    out = {"step": s["step"]}
    if s["clip"]:
        norm = torch.sqrt((g.double() * g.double()).sum())
        out["norm"] = norm.float()
        g = g * torch.clamp(_CLIP / (norm + 1e-6), max=1.0).float()
    eight = s["bits"] == 8
    m = _values(s["m"], s["me"], 15) if eight else s["m"]
    v = _values(s["v"], s["ve"], 31) if eight else s["v"]
    p = s["p"] if s["master"] is None else s["master"]
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + (g * g) * (1.0 - b2)
    p = p * (1.0 - lr * _HYPER["weight_decay"]) - (m / (torch.sqrt(v) * c2 + _HYPER["eps"])) * c1
    if s["master"] is not None:
        s["master"].copy_(p)
        out["master"] = s["master"]
    s["p"].copy_(p.to(dt))
    out["p"] = s["p"]
    if not eight:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return {**out, "m": s["m"], "v": s["v"]}
    # each tensor's elements count from 0; a tensor's place and the step key the hash
    n = torch.tensor([(n + _BLOCK - 1) // _BLOCK * _BLOCK for _, n in s["spans"]], device="cuda")
    first = torch.tensor([a for a, _ in s["spans"]], device="cuda").repeat_interleave(n)
    place = torch.arange(len(n), device="cuda").repeat_interleave(n)
    i = torch.arange(p.numel(), device="cuda") - first
    r = _hash(i ^ _hash((s["step"] * 0x9E3779B1 + place) & 0xFFFFFFFF))
    for name, x, bits, bias in (("m", m, r & 0xFFFF, 15), ("v", v, r >> 16, 31)):
        code, e = _quantise(x, bits, bias)
        s[name].copy_(code)
        s[name + "e"].copy_(e)
        out[name] = _values(code, e, bias).to(torch.bfloat16)  # 4 significant bits: exact
    return out


def _plain_ce(s):
    x, w = s["x"].float(), s["w"].float()
    live = s["t"] >= 0
    t = s["t"].clamp_min(0)[:, None]
    z = x @ w.t()
    m = z.max(1, keepdim=True)[0]
    e = torch.exp(z - m)
    tot = e.sum(1, keepdim=True)
    loss = torch.where(live, (m + torch.log(tot) - z.gather(1, t))[:, 0], torch.zeros_like(tot[:, 0]))
    count = live.sum().clamp_min(1) if s["reduction"] == "mean" else 1
    out = {"loss": loss if s["reduction"] == "none" else loss.sum() / count}
    if s["mode"] == "step":
        u = live.float() / count if s["up"] is None else live * s["up"]
        dz = e / tot
        dz.scatter_add_(1, t, torch.full_like(t, -1.0, dtype=torch.float32))
        dz = dz * u[:, None]
        out["dx"] = (dz @ w).to(s["x"].dtype)
        out["dw"] = (dz.t() @ x).to(s["x"].dtype)
    return out


def _plain_embed(s):
    out = {"y": (s["w"][s["ids"]].float() * s["scale"]).to(s["w"].dtype)}
    if s["mode"] == "step":
        d = torch.zeros(s["w"].shape, dtype=torch.float64, device="cuda")  # a frequent token's sum is long
        d.index_add_(0, s["ids"], s["gy"].double())
        out["dw"] = (d * s["scale"]).to(s["w"].dtype)
    return out


def _own_adamw(s):
    from ravel_lm_b200.optim import adamw_step, state_values
    norm = adamw_step(s["params"], s["grads"], s["ms"], s["vs"], s["step"], masters=s["masters"],
                      exp_avg_exponents=s["mes"], exp_avg_sq_exponents=s["ves"],
                      max_norm=_CLIP if s["clip"] else None, **_HYPER)
    out = {"step": s["step"], "p": s["p"]}
    if s["clip"]:
        out["norm"] = norm
    if s["master"] is not None:
        out["master"] = s["master"]
    if s["bits"] == 32:
        return {**out, "m": s["m"], "v": s["v"]}
    return {**out, "m": state_values(s["m"], s["me"], signed=True, dtype=torch.bfloat16),
            "v": state_values(s["v"], s["ve"], signed=False, dtype=torch.bfloat16)}


def _own_ce(s):
    from ravel_lm_b200.vocab import linear_cross_entropy
    loss = linear_cross_entropy(s["x"], s["w"], s["t"], reduction=s["reduction"])
    if s["mode"] != "step":
        return {"loss": loss}
    dx, dw = torch.autograd.grad(loss, [s["x"], s["w"]], s["up"])
    return {"loss": loss, "dx": dx, "dw": dw}


def _own_embed(s):
    from ravel_lm_b200.vocab import token_embedding
    y = token_embedding(s["ids"], s["w"], scale=s["scale"])
    if s["mode"] != "step":
        return {"y": y}
    return {"y": y, "dw": torch.autograd.grad(y, [s["w"]], s["gy"])[0]}


def run(state):
    if own:
        return {"ce": _own_ce, "embed": _own_embed, "adamw": _own_adamw}[state["op"]](state)
    with torch.no_grad():
        return {"ce": _plain_ce, "embed": _plain_embed, "adamw": _plain_adamw}[state["op"]](state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    e, step = _BYTES[case["dtype"]], case["mode"] == "step"
    if case["op"] == "adamw":
        n = sum(math.prod(sh) for sh in _shapes(case))
        b = e + e + (4 if e == 4 else 8)                                   # gradient in; parameter out; p or master in, out
        b += 16 if case["bits"] == 32 else 4 + 4.0 / _BLOCK                # states in and out
        if case["bits"] == 8:
            b += 4                                                         # the values they stand for, out
        return {"bytes": n * b, "flops": n * 14.0}
    M, K, V = case["M"], case["K"], case["V"]
    if case["op"] == "embed":
        rows = min(M, V)                                                   # distinct rows at most
        n = rows * K * e + M * K * e + M * 8
        if step:
            n += M * K * e + V * K * e
        return {"bytes": n, "flops": M * K * (2.0 if step else 1.0)}
    n = (M * K + V * K) * e * (2 if step else 1) + M * 8 + 4
    return {"bytes": n, "flops": 2.0 * M * K * V * (3 if step else 1)}


# ------------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    step = case["mode"] == "step"
    with torch.no_grad():
        if case["op"] == "adamw":
            b1, b2 = _HYPER["betas"]
            t = _STEP0 + 1
            g = s["g"].double()
            norm = torch.linalg.vector_norm(g)
            if case["clip"]:
                g = g * min(1.0, _CLIP / (float(norm) + 1e-6))
            eight = case["bits"] == 8
            m = (_values(s["m"], s["me"], 15) if eight else s["m"]).double().lerp_(g, 1.0 - b1)
            v = (_values(s["v"], s["ve"], 31) if eight else s["v"]).double().mul_(b2).addcmul_(g, g, value=1.0 - b2)
            p = (s["p"] if s["master"] is None else s["master"]).double()
            p = p.mul_(1.0 - _HYPER["lr"] * _HYPER["weight_decay"])
            p = p.addcdiv_(m / (1.0 - b1 ** t), (v / (1.0 - b2 ** t)).sqrt_().add_(_HYPER["eps"]),
                           value=-_HYPER["lr"])
            # 8-bit states: which neighbour a value goes to is the random bits' choice
            out = {"step": None, "p": p, "m": None if eight else m, "v": None if eight else v}
            if case["clip"]:
                out["norm"] = norm
            if s["master"] is not None:
                out["master"] = p
            return out
        w = s["w"].detach().double()
        if case["op"] == "embed":
            out = {"y": torch.index_select(w, 0, s["ids"]).mul_(case["scale"])}
            if step:
                # sums of sorted runs as differences of running sums
                order = torch.argsort(s["ids"], stable=True)
                run_sum = torch.cumsum(s["gy"].double()[order], 0)
                ids, n = torch.unique_consecutive(s["ids"][order], return_counts=True)
                ends = run_sum[torch.cumsum(n, 0) - 1]
                d = torch.zeros_like(w)
                d[ids] = torch.diff(ends, dim=0, prepend=torch.zeros_like(ends[:1]))
                out["dw"] = d.mul_(case["scale"])
            return out
        x = s["x"].detach().double()
        rows = torch.nonzero(s["t"] >= 0)[:, 0]
        t = s["t"][rows]
        logp = torch.log_softmax(torch.mm(x[rows], w.T), dim=1)
        nll = -logp[torch.arange(rows.numel(), device="cuda"), t]
        scale = 1.0 / max(1, rows.numel()) if case["reduction"] == "mean" else 1.0
        if case["reduction"] == "none":
            out = {"loss": torch.zeros(case["M"], dtype=torch.float64, device="cuda").index_copy_(0, rows, nll)}
        else:
            out = {"loss": nll.sum() * scale}
        if step:
            p = logp.exp_()
            p[torch.arange(rows.numel(), device="cuda"), t] -= 1.0
            p.mul_(scale if s["up"] is None else s["up"].double()[rows][:, None])
            out["dx"] = torch.zeros_like(x).index_copy_(0, rows, torch.mm(p, w))
            out["dw"] = torch.mm(p.T, x[rows])
        return out
