"""``fused_linear`` against the formula in 64 bits.

Tolerances follow from the arithmetic.  With u the unit roundoff of the 16-bit
type (2^-8 bfloat16, 2^-11 float16) and S = sum_k |a_k b_k| of an element:

* the product accumulates in float32: error <= (K + 8) 2^-23 S, S the sum of
  the magnitudes (the accumulator may truncate, hence 2^-23);
* an activation is Lipschitz (|act'| <= 1.13) and evaluated to a few float32
  units of its argument: twice the product's bound covers it;
* the output is rounded once: u |y| (and the type's smallest subnormal);
* z is kept in 16 bits for the backward: it moves act' by <= L u |z|, L = max |act''|
  (0.8 gelu, 0.5 silu, 0 otherwise; act' itself <= 1.13), and dz is rounded:
  |d dz| <= u |dz| + L u |z dy|, which enters the gradient products linearly;
* a bias gradient sums unrounded dz: M 2^-23 sum |dz| + the L u |z dy| terms.

The gradients are also held against central differences of the 64-bit formula.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
LIP = {"none": 0.0, "relu": 0.0, "gelu": 0.8, "silu": 0.5}
ACTS = ["none", "relu", "gelu", "silu"]


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import ravel_lm_b200._lib as L
    L.load()
    yield
    torch.cuda.synchronize()
    assert L.device_error(torch.cuda.current_stream().cuda_stream) == 0


def act64(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z / math.sqrt(2.0)))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def act64_grad(z, act):
    if act == "relu":
        return (z > 0).double()
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z / math.sqrt(2.0))) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        s = torch.sigmoid(z)
        return s + z * s * (1 - s)
    return torch.ones_like(z)


def make(M, K, N, dtype, seed, bias=True, residual=True, grad=False):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def t(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype).requires_grad_(grad)
    x, w = t(M, K), t(N, K, scale=max(K, 1) ** -0.5)
    return x, w, (t(N, scale=0.3) if bias else None), (t(M, N) if residual else None)


def within(got, want, tol, what):
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)} != {tuple(want.shape)}"
    if got.numel() == 0:
        return
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    if bad.any():
        i = int(torch.argmax(torch.where(bad, err - tol, torch.zeros_like(err)).flatten()))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} beyond tolerance; worst {got.flatten()[i]} "
                             f"for {want.flatten()[i]}, tolerance {tol.flatten()[i]}")


def check(x, w, b, r, act, y, grads=None, gy=None):
    """y (and grads: dict of dx, dw, db, dr) against the 64-bit formula with the tolerances above."""
    dt = x.dtype
    u, tiny = U[dt], TINY[dt]
    x64, w64 = x.detach().double().reshape(math.prod(x.shape[:-1]), x.shape[-1]), w.detach().double()
    M, K = x64.shape
    N = w64.shape[0]
    z = x64 @ w64.t()
    S = x64.abs() @ w64.abs().t()
    if b is not None:
        z = z + b.detach().double()
        S = S + b.detach().double().abs()
    want = act64(z, act)
    acc = 2 * (K + 8) * 2.0 ** -23 * S
    if r is not None:
        want = want + r.detach().double().reshape(M, N)
    within(y.reshape(M, N), want, acc + u * want.abs() + tiny, "y")
    if grads is None:
        return
    gy64 = gy.double().reshape(M, N)
    d = act64_grad(z, act)
    if act == "relu":  # elements whose sign the accumulation leaves open count either way
        open_ = (z.abs() <= acc).double()
    else:
        open_ = torch.zeros_like(z)
    dz = gy64 * d
    slip = (LIP[act] * (u * z.abs() + acc) + 2.0 ** -20 + open_) * gy64.abs() + tiny
    edz = u * dz.abs() + slip
    if "dx" in grads:
        want = dz @ w64
        tol = edz @ w64.abs() * (1 + u) + (N + 8) * 2.0 ** -23 * (dz.abs() @ w64.abs()) + u * want.abs() + tiny
        within(grads["dx"].reshape(M, K), want, tol, "dx")
    if "dw" in grads:
        want = dz.t() @ x64
        tol = edz.t() @ x64.abs() * (1 + u) + (M + 8) * 2.0 ** -23 * (dz.abs().t() @ x64.abs()) + u * want.abs() + tiny
        within(grads["dw"], want, tol, "dw")
    if "db" in grads:
        want = dz.sum(0)
        tol = slip.sum(0) + (M + 8) * 2.0 ** -23 * dz.abs().sum(0) + u * want.abs() + tiny
        within(grads["db"], want, tol, "db")
    if "dr" in grads:
        assert torch.equal(grads["dr"].reshape(M, N), gy.reshape(M, N)), "d residual is the output's gradient"


def step(x, w, b, r, act, gy):
    from ravel_lm_b200.dense import fused_linear
    y = fused_linear(x, w, b, activation=act, residual=r)
    leaves = {n: t for n, t in (("dx", x), ("dw", w), ("db", b), ("dr", r)) if t is not None}
    return y, dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), gy)))


# small and odd sizes, tile edges, and widths that need the padded copies (the launch shapes: test_gpu_dense_shapes.py)
SHAPES = [(1, 64, 128), (1, 4096, 256), (2, 512, 1000), (7, 8, 8), (24, 2048, 512), (33, 100, 60), (127, 65, 129),
          (128, 1024, 128), (129, 1000, 257), (300, 333, 515), (512, 256, 768), (1000, 128, 2056), (2049, 64, 511),
          (4096, 192, 1024), (3000, 520, 2304)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_forward(M, K, N, dtype):
    from ravel_lm_b200.dense import fused_linear
    act = ACTS[(M + N) % 4]
    x, w, b, r = make(M, K, N, dtype, seed=M + 7 * N, bias=(M + K) % 3 != 0, residual=(K + N) % 2 == 0)
    check(x, w, b, r, act, fused_linear(x, w, b, activation=act, residual=r))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("M,K,N", [(5, 192, 96), (260, 130, 300), (1024, 256, 512)])
def test_step_every_epilogue(M, K, N, bias, residual, act):
    for dtype in (torch.bfloat16, torch.float16):
        x, w, b, r = make(M, K, N, dtype, seed=M, bias=bias, residual=residual, grad=True)
        gy = torch.randn(M, N, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
        y, g = step(x, w, b, r, act, gy)
        check(x, w, b, r, act, y, g, gy)


@pytest.mark.parametrize("M,K,N", SHAPES + [(8192, 768, 256), (6000, 1024, 2048)])
def test_step_every_shape(M, K, N):
    act = ACTS[(M + K + N) % 4]
    x, w, b, r = make(M, K, N, torch.bfloat16, seed=M + N, residual=M % 2 == 0, grad=True)
    gy = torch.randn(M, N, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(torch.bfloat16)
    y, g = step(x, w, b, r, act, gy)
    check(x, w, b, r, act, y, g, gy)
    # the same inputs give the same bits
    y2, g2 = step(x, w, b, r, act, gy)
    assert torch.equal(y, y2) and all(torch.equal(g[n], g2[n]) for n in g)


@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_gradient_against_differences(act):
    """<grad, direction> = the central difference of <y, gy> along the direction (64-bit formula), to the
    gradient's own rounding: each gradient element is good to 3 u of its magnitude sum."""
    M, K, N, h = 40, 72, 136, 1e-4
    x, w, b, r = make(M, K, N, torch.float16, seed=3, grad=True)
    gy = torch.randn(M, N, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").half()
    _, g = step(x, w, b, r, act, gy)

    def f(x_, w_, b_):
        return ((act64(x_ @ w_.t() + b_, act)) * gy.double()).sum()
    base = [t.detach().double() for t in (x, w, b)]
    S = [gy.double().abs() @ base[1].abs(), gy.double().abs().t() @ base[0].abs(), gy.double().abs().sum(0)]
    for i, n in enumerate(("dx", "dw", "db")):
        v = torch.randn(base[i].shape, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda").double()
        up, dn = list(base), list(base)
        up[i], dn[i] = base[i] + h * v, base[i] - h * v
        want = float((f(*up) - f(*dn)) / (2 * h))
        got = float((g[n].double() * v).sum())
        tol = 3 * U[torch.float16] * float(((S[i] * 1.13) * v.abs()).sum()) + 1e-6
        assert abs(got - want) <= tol, f"{n}: {got} vs {want} (tolerance {tol})"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K,N", [(256, 4096, 2048), (40, 8192, 4100), (1500, 1000, 515)])
def test_relu_signs_of_sums_near_zero(M, K, N, dtype):
    """The derivative is the exact sum's sign unless that lies within float32's own rounding of a sum of K terms in
    lanes of K / 32 (K / 32 + 16 additions of partial sums no larger than a few times the sum's spread of 1)."""
    x, w, b, _ = make(M, K, N, dtype, seed=K, residual=False, grad=True)
    ones = torch.ones(M, N, device="cuda", dtype=dtype)  # the bias gradient counts a column's open elements
    from ravel_lm_b200.dense import fused_linear
    z = x.detach().double() @ w.detach().double().t() + b.detach().double()
    db = torch.autograd.grad(fused_linear(x, w, b, activation="relu"), b, ones)[0]
    sure = z.abs() > (K / 32 + 16) * 2.0 ** -24 * 4
    low = ((z > 0) & sure).sum(0).double()
    high = low + (~sure).sum(0)
    # counts up to M are rounded to the type
    u = U[dtype]
    assert bool(((db.double() >= low * (1 - u)) & (db.double() <= high * (1 + u))).all())
    part = torch.arange(0, M, max(1, M // 8), device="cuda")  # and rows one at a time, where counts are 0 or 1
    for i in part.tolist():
        xi = x.detach()[i:i + 1].expand(2, K).contiguous().requires_grad_(True)
        gy = torch.zeros(2, N, device="cuda", dtype=dtype)
        gy[0] = 1
        di = torch.autograd.grad(fused_linear(xi, w, b, activation="relu"), b, gy)[0].double()
        wrong = (di != (z[i] > 0).double()) & sure[i]
        assert not wrong.any(), (i, z[i][wrong])


def test_strides_views_and_leading_dimensions():
    from ravel_lm_b200.dense import fused_linear
    g = torch.Generator(device="cuda").manual_seed(5)
    big = torch.randn(6, 50, 400, generator=g, device="cuda").bfloat16()
    W = torch.randn(90, 300, generator=g, device="cuda").bfloat16() * 0.1
    for x in (big[:, :, :96], big[:, ::2, 8:104], big[:, :, 3:99], big.transpose(0, 1)[:, :, 16:112],
              big[:1, :1, :96].expand(3, 5, 96), big[0].t()[:96].t()):
        for w in (W[:, :96], W[:, 5:101], W[::2, 16:112], W.t()[:90, :96]):
            if w.shape[1] != x.shape[-1]:
                continue
            xs, ws = x.detach().clone().requires_grad_(True), w.detach().clone().requires_grad_(True)
            r = torch.randn(*x.shape[:-1], w.shape[0], generator=g, device="cuda").bfloat16()
            y = fused_linear(x, w, activation="silu", residual=r.transpose(0, -1).contiguous().transpose(0, -1))
            check(xs, ws, None, r, "silu", y)
            # the layout of the inputs does not change the bits
            assert torch.equal(y, fused_linear(xs, ws, activation="silu", residual=r))
            # a gradient that is a broadcast or a transposed view
            ye = fused_linear(xs, ws, activation="silu", residual=r)
            gy = torch.randn(w.shape[0], generator=g, device="cuda").bfloat16().expand_as(ye)
            got = torch.autograd.grad(ye, [xs, ws], gy)
            check(xs, ws, None, r, "silu", y, {"dx": got[0], "dw": got[1]}, gy)


def test_a_bias_and_a_weight_shared_by_two_calls():
    from ravel_lm_b200.dense import fused_linear
    x, w, b, _ = make(70, 64, 64, torch.bfloat16, seed=6, residual=False, grad=True)
    gy = torch.randn(70, 64, device="cuda").bfloat16()
    y1 = fused_linear(x, w, b, activation="relu")
    y2 = fused_linear(y1, w, b)
    one = torch.autograd.grad(y2, [w, b], gy, retain_graph=True)
    mid = torch.autograd.grad(y2, [y1], gy, retain_graph=True)[0]
    x1, w1, b1 = (t.detach().clone().requires_grad_(True) for t in (y1, w, b))
    part2 = torch.autograd.grad(fused_linear(x1, w1, b1), [w1, b1], gy)
    part1 = torch.autograd.grad(y1, [w, b], mid)
    for a, p, q in zip(one, part1, part2):
        assert torch.equal(a, p + q)


def test_empty_and_single():
    from ravel_lm_b200.dense import fused_linear
    for M, K, N in ((0, 16, 24), (5, 0, 24), (5, 16, 0), (0, 0, 0), (1, 1, 1), (1, 1, 9), (3, 2, 1)):
        x, w, b, r = make(M, K, N, torch.bfloat16, seed=8, grad=True)
        gy = torch.randn(M, N, device="cuda").bfloat16()
        y, g = step(x, w, b, r, "gelu", gy)
        check(x, w, b, r, "gelu", y, g, gy)
    one = fused_linear(torch.ones(16, device="cuda").half(), torch.ones(24, 16, device="cuda").half())
    assert one.shape == (24,) and bool((one == 16).all())


def test_only_the_gradients_that_are_asked_for():
    from ravel_lm_b200.dense import fused_linear
    x, w, b, r = make(64, 96, 80, torch.bfloat16, seed=9)
    gy = torch.randn(64, 80, device="cuda").bfloat16()
    for pick in ("dx", "dw", "db", "dr"):
        ts = {"dx": x, "dw": w, "db": b, "dr": r}
        leaf = ts[pick].clone().requires_grad_(True)
        ts[pick] = leaf
        y = fused_linear(ts["dx"], ts["dw"], ts["db"], activation="gelu", residual=ts["dr"])
        check(ts["dx"], ts["dw"], ts["db"], ts["dr"], "gelu", y, {pick: torch.autograd.grad(y, leaf, gy)[0]}, gy)
    xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = fused_linear(xs, ws, b)
    only = torch.autograd.grad(y, xs, gy, retain_graph=True)[0]
    assert torch.equal(only, torch.autograd.grad(y, [xs, ws], gy)[0])


def test_infinities_and_nan_stay_in_their_rows():
    from ravel_lm_b200.dense import fused_linear
    x, w, b, _ = make(40, 64, 64, torch.bfloat16, seed=10, residual=False)
    x[3, 5] = float("inf")
    x[7, 0] = float("nan")
    for act in ACTS:
        y = fused_linear(x, w, b, activation=act)
        assert torch.isnan(y[7]).all()
        assert not torch.isfinite(y[3].float()).all()
        keep = [i for i in range(40) if i not in (3, 7)]
        check(x[keep], w, b, None, act, y[keep])


def test_another_stream_and_graph_replay():
    from ravel_lm_b200.dense import fused_linear
    x, w, b, r = make(200, 100, 120, torch.bfloat16, seed=11)  # K = 100: padded copies are workspaces
    want = fused_linear(x, w, b, activation="gelu", residual=r)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = fused_linear(x, w, b, activation="gelu", residual=r)
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fused_linear(x, w, b, activation="gelu", residual=r)
    x.copy_(torch.randn(200, 100, device="cuda"))
    graph.replay()
    assert torch.equal(out, fused_linear(x, w, b, activation="gelu", residual=r))


def test_offsets_past_32_bits():
    from ravel_lm_b200.dense import fused_linear
    M, K, N = 40000, 64, 65536  # 2.6e9 outputs
    x, w, b, _ = make(M, K, N, torch.bfloat16, seed=13, residual=False)
    y = fused_linear(x, w, b, activation="silu")
    for rows in (slice(0, 128), slice(M // 2, M // 2 + 128), slice(M - 128, M)):
        check(x[rows], w, b, None, "silu", y[rows])


def test_refusals():
    from ravel_lm_b200.dense import fused_linear
    x, w, b, r = make(4, 8, 16, torch.bfloat16, seed=12)
    with pytest.raises(ValueError, match="activation"):
        fused_linear(x, w, b, activation="tanh")
    with pytest.raises(ValueError, match="weight"):
        fused_linear(x, w[:, :4], b)
    with pytest.raises(ValueError, match="bias"):
        fused_linear(x, w, b[:3])
    with pytest.raises(ValueError, match="residual"):
        fused_linear(x, w, b, residual=r[:2])
    with pytest.raises(TypeError, match="one dtype"):
        fused_linear(x, w.half(), b)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        fused_linear(x.float(), w.float())
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        fused_linear(x.cpu(), w.cpu())
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        fused_linear(x, w, b.cpu())
    xs = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(fused_linear(xs, w, b).sum(), xs, create_graph=True)
