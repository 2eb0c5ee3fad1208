"""``layer_norm`` against the formula in 64 bits.

Tolerances, with e = 2^-24 (float32 roundoff), u the output type's roundoff
(2^-24, 2^-8, 2^-11) and d = K / 32 + 64 (no sum has a longer chain of additions:
32 lanes or more share a row):

* the mean is off by at most d e mean|x|, the variance relatively by 2 d e and by
  the square of the mean's error, so with r = 1 / sqrt(var + eps)
  |d xh| <= r (d e mean|x| + 2 e |x|) + (d + 16) e |xh|;
* y adds |g| |d xh|, two float32 roundings and its own rounding u |y|;
* dx = r (a - m1 - xh m2): the means' sums are off by d e of their magnitudes, m2 also
  by mean(|a| |d xh|);
* dg and db: M + 64 additions at most in a chain, plus |dy| |d xh|.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -140, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
E = 2.0 ** -24
EPS = 1e-5


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import ravel_lm_b200._lib as L
    L.load()
    yield
    torch.cuda.synchronize()
    assert L.device_error(torch.cuda.current_stream().cuda_stream) == 0


def make(M, K, dtype, seed, affine=True, shift=0.4):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(M, K, generator=g, device="cuda") * 1.7 + shift).to(dtype).requires_grad_(True)
    w = (1 + 0.2 * torch.randn(K, generator=g, device="cuda")).to(dtype).requires_grad_(True) if affine else None
    b = (0.2 * torch.randn(K, generator=g, device="cuda")).to(dtype).requires_grad_(True) if affine else None
    gy = torch.randn(M, K, generator=g, device="cuda").to(dtype)
    return x, w, b, gy


def within(got, want, tol, what):
    if got.numel() == 0:
        return
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} beyond tolerance, worst "
                           f"{float((err / tol)[bad].max()):.3g} times")


def check(x, w, b, gy, y, grads, eps=EPS):
    u, tiny = U[x.dtype], TINY[x.dtype]
    x64 = x.detach().double().reshape(-1, x.shape[-1])
    M, K = x64.shape
    d = K / 32 + 64
    g64 = w.detach().double() if w is not None else torch.ones(K, dtype=torch.float64, device="cuda")
    b64 = b.detach().double() if b is not None else torch.zeros(K, dtype=torch.float64, device="cuda")
    mean = x64.mean(1, keepdim=True)
    r = 1 / torch.sqrt(((x64 - mean) ** 2).mean(1, keepdim=True) + eps)
    xh = (x64 - mean) * r
    off = d * E * x64.abs().mean(1, keepdim=True)
    dxh = r * (off + 2 * E * x64.abs()) + ((d + 16) * E + (off * r) ** 2) * xh.abs()
    want = xh * g64 + b64
    within(y.reshape(M, K), want, g64.abs() * dxh + 2 * E * (want.abs() + b64.abs()) + u * want.abs() + tiny, "y")
    if not grads:
        return
    gy64 = gy.double().reshape(M, K)
    a = gy64 * g64
    m1, m2 = a.mean(1, keepdim=True), (a * xh).mean(1, keepdim=True)
    if "dx" in grads:
        e1 = d * E * a.abs().mean(1, keepdim=True)
        e2 = d * E * (a * xh).abs().mean(1, keepdim=True) + (a.abs() * dxh).mean(1, keepdim=True)
        want = r * (a - m1 - xh * m2)
        tol = r * (e1 + xh.abs() * e2 + m2.abs() * dxh + 4 * E * (a.abs() + m1.abs() + (xh * m2).abs()))
        within(grads["dx"].reshape(M, K), want, tol + ((d + 16) * E + u) * want.abs() + tiny, "dx")
    if "dw" in grads:
        want = (gy64 * xh).sum(0)
        tol = (gy64.abs() * dxh).sum(0) + (M + 64) * E * (gy64 * xh).abs().sum(0) + u * want.abs() + tiny
        within(grads["dw"], want, tol, "dw")
    if "db" in grads:
        want = gy64.sum(0)
        within(grads["db"], want, (M + 64) * E * gy64.abs().sum(0) + u * want.abs() + tiny, "db")


def step(x, w, b, gy, eps=EPS):
    from ravel_lm_b200.glue import layer_norm
    y = layer_norm(x, w, b, eps)
    leaves = {n: t for n, t in (("dx", x), ("dw", w), ("db", b)) if t is not None}
    return y, dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), gy)))


# one element, every way a row is shared (1, 4 and 16 warps, vectors and single elements), the wide kernels,
# few and many rows
SHAPES = [(1, 1), (3, 2), (5, 7), (2, 31), (9, 32), (4, 255), (7, 256), (1, 1024), (65, 1000), (30, 1537), (3, 4096),
          (17, 2055), (2, 8191), (5, 8200), (3, 16384), (2, 40001), (3, 65536), (2000, 96), (3001, 256), (1500, 515),
          (1300, 1024), (2500, 2048), (1201, 2049)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", SHAPES)
def test_step(M, K, dtype):
    x, w, b, gy = make(M, K, dtype, seed=M + K, affine=(M + K) % 5 != 0)
    y, g = step(x, w, b, gy)
    check(x, w, b, gy, y, g)
    from ravel_lm_b200.glue import layer_norm
    with torch.no_grad():  # the forward alone gives the same bits, and so does a second step
        assert torch.equal(layer_norm(x, w, b, EPS), y)
    y2, g2 = step(x, w, b, gy)
    assert torch.equal(y, y2) and all(torch.equal(g[n], g2[n]) for n in g)


def test_weight_or_bias_alone():
    from ravel_lm_b200.glue import layer_norm
    x, w, b, gy = make(50, 64, torch.float32, seed=1)
    for ww, bb in ((w, None), (None, b)):
        y, g = step(x, ww, bb, gy)
        check(x, ww, bb, gy, y, g)
    for pick, leaf in (("dx", x), ("dw", w), ("db", b)):  # one gradient at a time, the others frozen
        ts = {"dx": x.detach(), "dw": w.detach(), "db": b.detach(), pick: leaf}
        y = layer_norm(ts["dx"], ts["dw"], ts["db"], EPS)
        check(x, w, b, gy, y, {pick: torch.autograd.grad(y, leaf, gy)[0]})


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_mean_far_from_zero(dtype):
    """The variance is summed around the mean: a row offset of 500 deviations costs no more than the offset's
    own rounding in the input."""
    x, w, b, gy = make(40, 768 if dtype != torch.float32 else 772, dtype, seed=2, shift=850.0)
    y, g = step(x, w, b, gy)
    check(x, w, b, gy, y, g)


def test_strides_broadcasts_and_leading_dimensions():
    from ravel_lm_b200.glue import layer_norm
    g = torch.Generator(device="cuda").manual_seed(3)
    big = torch.randn(5, 40, 300, generator=g, device="cuda").half()
    for x in (big[:, :, :256], big[:, ::3, 8:200], big[:, :, 5:205], big.transpose(0, 1)[..., :96],
              big[:1].expand(4, 40, 300), big[0].t()):
        K = x.shape[-1]
        w = torch.randn(2 * K, generator=g, device="cuda").half()[::2].requires_grad_(True)
        b = torch.randn(K + 1, generator=g, device="cuda").half()[1:].requires_grad_(True)
        xs = x.detach().clone().requires_grad_(True)
        y = layer_norm(x, w, b, EPS)
        assert torch.equal(y, layer_norm(xs, w, b, EPS))
        ys = layer_norm(xs, w, b, EPS)
        for gy in (torch.randn(K, generator=g, device="cuda").half().expand_as(ys),
                   torch.randn(ys.shape[::-1], generator=g, device="cuda").half().permute(*range(ys.dim())[::-1])):
            got = dict(zip(("dx", "dw", "db"), torch.autograd.grad(ys, [xs, w, b], gy, retain_graph=True)))
            check(xs, w, b, gy, y, got)


def test_empty_constant_and_non_finite_rows():
    from ravel_lm_b200.glue import layer_norm
    w = torch.ones(64, device="cuda", requires_grad=True)
    b = torch.zeros(64, device="cuda", requires_grad=True)
    x = torch.empty(0, 64, device="cuda", requires_grad=True)
    y = layer_norm(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], torch.empty(0, 64, device="cuda"))
    assert y.shape == (0, 64) and gx.shape == (0, 64) and not gw.any() and not gb.any()
    x, w, b, gy = make(6, 64, torch.float32, seed=4)
    with torch.no_grad():
        x[1] = 3.0                       # zero variance: y = b
        x[2, 7] = float("inf")
        x[3, 0] = float("nan")
    y, g = step(x, w, b, gy)
    assert torch.equal(y[1], b)
    assert torch.isnan(y[2]).all() and torch.isnan(y[3]).all()
    keep = [0, 1, 4, 5]
    check(x.detach()[keep], w, b, gy[keep], y[keep], {"dx": g["dx"][keep]})


def test_gradient_against_differences():
    x, w, b, gy = make(6, 40, torch.float32, seed=5)
    _, g = step(x, w, b, gy)
    base = [t.detach().double() for t in (x, w, b)]

    def f(x_, w_, b_):
        xc = x_ - x_.mean(1, keepdim=True)
        return ((xc / torch.sqrt((xc * xc).mean(1, keepdim=True) + EPS) * w_ + b_) * gy.double()).sum()
    h = 1e-6
    for i, n in enumerate(("dx", "dw", "db")):
        v = torch.randn(base[i].shape, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda").double()
        up, dn = list(base), list(base)
        up[i], dn[i] = base[i] + h * v, base[i] - h * v
        want = float((f(*up) - f(*dn)) / (2 * h))
        got = float((g[n].double() * v).sum())
        # float32 gradients of magnitude ~1: their sums of 240 products are good to 1e-4 at the worst
        assert abs(got - want) <= 1e-4 * max(1.0, float((g[n].double() * v).abs().sum())), (n, got, want)


def test_another_stream_and_graph_replay():
    from ravel_lm_b200.glue import layer_norm
    x, w, b, gy = make(300, 200, torch.bfloat16, seed=6)
    y, g = step(x, w, b, gy)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        y2, g2 = step(x, w, b, gy)
    s.synchronize()
    assert torch.equal(y, y2) and all(torch.equal(g[n], g2[n]) for n in g)
    graph = torch.cuda.CUDAGraph()
    xs = x.detach().clone()
    with torch.cuda.graph(graph):
        out = layer_norm(xs, w.detach(), b.detach(), EPS)
    xs.copy_(torch.randn(300, 200, device="cuda"))
    graph.replay()
    assert torch.equal(out, layer_norm(xs, w.detach(), b.detach(), EPS))


def test_offsets_past_32_bits():
    from ravel_lm_b200.glue import layer_norm
    M, K = (1 << 31) // 1024 + 300, 1024
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    tail = torch.randn(200, K, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda").bfloat16()
    x[-200:] = tail
    w, b = torch.full((K,), 2.0, device="cuda").bfloat16(), torch.ones(K, device="cuda").bfloat16()
    x.requires_grad_(True)
    y = layer_norm(x, w, b, EPS)
    assert bool((y[:-200] == 1).all())
    gx, = torch.autograd.grad(y, x, y.detach())
    check(tail, w, b, y.detach()[-200:], y[-200:], {"dx": gx[-200:]})


def test_refusals():
    from ravel_lm_b200.glue import layer_norm
    x, w, b, _ = make(4, 8, torch.float32, seed=8)
    with pytest.raises(ValueError, match="weight and bias"):
        layer_norm(x, w[:4], b)
    with pytest.raises(ValueError, match="weight and bias"):
        layer_norm(x, w, b[None])
    with pytest.raises(ValueError, match="K >= 1"):
        layer_norm(x[:, :0])
    with pytest.raises(TypeError, match="one dtype"):
        layer_norm(x, w.half(), b)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        layer_norm(x.double())
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        layer_norm(x.cpu())
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        layer_norm(x, w.cpu())
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(layer_norm(x, w, b).sum(), x, create_graph=True)
