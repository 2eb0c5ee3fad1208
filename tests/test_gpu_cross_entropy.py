"""``linear_cross_entropy`` against the formula in 64 bits.

Tolerances.  A logit is a tensor-core sum of K products, which may drop up to 2^-23 of
the sum's running size (at most A = max over the row of sum |x w|) in each of its K / 8 steps and
a few more: dz = (K / 8 + 16) 2^-23 A.  With e = 2^-24, exponents in base 2 are off by
4 e |z| more, ex2 and lg2 by 2^-21, and a row's sum by (V / 32 + 64) e.  Hence a loss is off by

    dl = 2 dz + 8 e max |z| + 2^-20 + (V / 32 + 64) e,

a probability by that much of itself.  d z enters the gradients' products rounded to 16 bits (u = eps / 2 of
the type), once more in the three-product form (where f x is rounded), so that

    |d x error| <= (2 u + 2 dl + (V / 8 + 16) 2^-23) (|d z| |W|) + u |d x|

elementwise, with |d z| times the row's upstream gradient, d W likewise with K's place taken by the rows.  float16
keeps d z times 2^15: what is below its smallest number, 2^-25 2^-15 of the largest upstream gradient, adds up over V.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
DTYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import ravel_lm_b200._lib as L
    L.load()
    yield
    torch.cuda.synchronize()
    assert L.device_error(torch.cuda.current_stream().cuda_stream) == 0


def ce(*a, **k):
    from ravel_lm_b200.vocab import linear_cross_entropy
    return linear_cross_entropy(*a, **k)


def make(M, K, V, dt, seed, scale=2.0, ignored=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(M, K, generator=g, device="cuda").to(dt)
    w = (torch.randn(V, K, generator=g, device="cuda") * scale * K ** -0.5).to(dt)
    t = torch.randint(0, V, (M,), generator=g, device="cuda")
    if ignored and M > 2:
        t[M // 2] = -100
        t[::7] = -100
    return x, w, t


def within(got, want, tol, what):
    d = (got.double() - want).abs()
    bad = ~((d <= tol) | (got.double() == want))
    if bool(bad.any()):
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} beyond tolerance, worst "
                             f"{float((d / tol)[bad].max()):.3g} times")


def reference(x, w, t, ignore=-100):
    """Losses, softmax - onehot of the rows with a target (else 0), and how far a loss may be off."""
    x, w = x.detach().double(), w.detach().double()
    V, K = w.shape
    live = (t >= 0) & (t < V) & (t != ignore)
    x = torch.where(live[:, None], x, torch.zeros_like(x))
    z = x @ w.T
    lp = torch.log_softmax(z, 1)
    safe = torch.where(live, t, torch.zeros_like(t))[:, None]
    loss = torch.where(live, -lp.gather(1, safe)[:, 0], torch.zeros_like(lp[:, 0]))
    A = (x.abs() @ w.abs().T).amax(1)
    dz = (K / 8 + 16) * 2.0 ** -23 * A
    dl = 2 * dz + 8 * E * z.abs().amax(1) + 2.0 ** -20 + (V / 32 + 64) * E
    d = lp.exp_()
    d.scatter_add_(1, safe, torch.full_like(safe, -1.0, dtype=torch.float64))
    d.mul_(live[:, None])
    return loss, d, dl * live, live


def check(x, w, t, reduction="mean", up=None, ignore=-100):
    dt = x.dtype
    u = torch.finfo(dt).eps / 2
    M, K = x.shape
    V = w.shape[0]
    xl, wl = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = ce(xl, wl, t, reduction=reduction, ignore_index=ignore)
    assert loss.dtype == torch.float32
    want, d, dl, live = reference(x, w, t, ignore)
    n = max(1, int(live.sum()))
    tol = dl + 4 * E * want.abs()
    if reduction == "none":
        within(loss.detach(), want, tol, "losses")
        f = torch.ones(M, dtype=torch.float64, device="cuda") if up is None else up.double()
        f = torch.where(live, f, torch.zeros_like(f))
        got = torch.autograd.grad(loss, [xl, wl], torch.ones_like(loss) if up is None else up)
    else:
        div = n if reduction == "mean" else 1
        within(loss.detach(), want.sum() / div, (tol.sum() + (M / 32 + 64) * E * want.sum()) / div + 1e-30, "loss")
        f = torch.full((M,), (1.0 if up is None else float(up)) / div, dtype=torch.float64, device="cuda")
        got = torch.autograd.grad(loss, [xl, wl], up)
    alone = ce(x.detach(), w.detach(), t, reduction=reduction, ignore_index=ignore)  # without the gradients' products
    if reduction == "none":
        within(alone, want, tol, "losses alone")
    else:
        within(alone, want.sum() / div, (tol.sum() + (M / 32 + 64) * E * want.sum()) / div + 1e-30, "loss alone")
    d = d * f[:, None]
    xa = torch.where(live[:, None], x.detach().double(), torch.zeros_like(x, dtype=torch.float64))
    wa = w.detach().double()
    low = float(f.abs().max()) * 2.0 ** -40 if dt == torch.float16 and M else 0.0
    rel = 2 * u + 2 * dl[:, None]
    want_x, want_w = d @ wa, d.T @ xa
    # 2 dl bounds a probability's error relative to itself, the target's 1 - p_t likewise
    tx = (d.abs() * (rel + (V / 8 + 16) * 2.0 ** -23)) @ wa.abs() + low * wa.abs().sum(0) + (u + 4 * E) * want_x.abs()
    tw = (d.abs() * (rel + (M / 8 + 16) * 2.0 ** -23)).T @ xa.abs() + low * xa.abs().sum(0) + (u + 4 * E) * want_w.abs()
    # an error of p_t is one of 1 - p_t
    pt = torch.where(live, torch.exp(-want), torch.zeros_like(want)) * dl * f.abs()
    tx += pt[:, None] * wa[torch.where(live, t, torch.zeros_like(t))].abs()
    tw.index_add_(0, torch.where(live, t, torch.zeros_like(t)), pt[:, None] * xa.abs())
    within(got[0], want_x, tx + TINY[dt], "d x")
    within(got[1], want_w, tw + TINY[dt], "d weight")
    assert not got[0][~live].any()
    return loss, got


# one of everything; rows around the tiles of 128 and 256; odd widths and vocabularies; both launch shapes
SHAPES = [(1, 1, 1), (1, 8, 2), (2, 3, 5), (3, 5, 33), (24, 200, 320), (127, 64, 300), (128, 72, 257), (129, 16, 1000),
          (255, 33, 4097), (256, 128, 256), (257, 40, 1031), (1000, 96, 515), (40, 1032, 6000), (2000, 24, 64),
          (600, 520, 9000)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,K,V", SHAPES)
def test_sizes(dt, M, K, V):
    check(*make(M, K, V, dt, seed=M + V))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_reductions_and_upstream_gradients(dt, reduction):
    x, w, t = make(300, 64, 700, dt, seed=1)
    if reduction == "none":
        g = torch.Generator(device="cuda").manual_seed(2)
        up = torch.randn(300, generator=g, device="cuda")
        up[5], up[8] = 0.0, 1e-4
        check(x, w, t, reduction, up)
        check(x, w, t, reduction)
        check(x, w, t, reduction, up * 1e6 if dt == torch.bfloat16 else up * 1e-3)
        check(x, w, t, reduction, torch.zeros_like(up))
        up[t == -100] = float("nan")  # where a row has no target, anything may stand
        check(x, w, t, reduction, torch.nan_to_num(up, nan=float("inf")))
    else:
        for v in (1.0, -2.5, 0.0, 65536.0 if reduction == "mean" else 3.0):
            check(x, w, t, reduction, torch.tensor(v, device="cuda"))


@pytest.mark.parametrize("dt,M,K,V", [(torch.bfloat16, 5000, 128, 65536), (torch.bfloat16, 1300, 1100, 32003),
                                      (torch.float16, 4500, 32, 65536), (torch.bfloat16, 300, 1600, 70001)])
def test_pieces_and_three_products(dt, M, K, V):
    """Past 3e10 = M K V bfloat16 takes three products; past 512 MB of d z the rows go in pieces."""
    check(*make(M, K, V, dt, seed=K))


def test_three_products_of_rows_far_from_their_targets():
    """Losses past 55, whose exp(z - z_t) bfloat16 or float32 could not hold: in some rows of a piece, and in all."""
    x, w, t = make(1400, 512, 48000, torch.bfloat16, seed=3)
    big = x.clone()
    big[100:110] *= 40
    check(big, w, t)
    check(x * 12, w, t)


def test_confident_rows():
    """1 - p_t far below one step of 1: the target's gradient must not come from a difference."""
    M, K, V = 200, 256, 900
    x, w, t = make(M, K, V, torch.bfloat16, seed=4, scale=0.5, ignored=False)
    w[t[:100]] = x[:100] * 0.08  # z_t about 20
    loss, (dx, dw) = check(x, w, t, "sum")


@pytest.mark.parametrize("dt", DTYPES)
def test_common_offsets_and_large_logits(dt):
    """An offset of every logit changes nothing; logits of several hundred."""
    x, w, t = make(140, 64, 500, dt, seed=5)
    x[:, -1] = 8.0
    w[:, -1] = 60.0
    check(x, w, t)
    check(x * 4, w * 4, t)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,K,V", [(300, 40, 200), (1300, 1100, 32003)])
def test_rows_without_a_target(dt, M, K, V):
    x, w, t = make(M, K, V, dt, seed=6)
    l0, g0 = check(x, w, t)
    x[t == -100] = float("nan")
    x[7] = float("inf")  # every seventh row has no target
    xl, wl = x.requires_grad_(True), w.clone().requires_grad_(True)
    loss = ce(xl, wl, t)
    dx, dw = torch.autograd.grad(loss, [xl, wl])
    assert torch.equal(loss, l0) and torch.equal(dx, g0[0]) and torch.equal(dw, g0[1])
    with torch.no_grad():
        assert torch.equal(ce(x, w, t), ce(torch.nan_to_num(x.detach(), 0.0, 0.0, 0.0), w, t))
    none = torch.full_like(t, -100)
    for red in ("mean", "sum"):
        loss = ce(xl, wl, none, reduction=red)
        dx, dw = torch.autograd.grad(loss, [xl, wl])
        assert float(loss.detach()) == 0.0 and not dx.any() and not dw.any()
    # an ignored index inside the vocabulary
    check(torch.nan_to_num(x.detach(), 0.0, 0.0, 0.0), w, t.clamp_min(0), ignore=0)


def test_no_rows():
    w = torch.randn(50, 16, device="cuda").bfloat16().requires_grad_(True)
    x = torch.zeros(0, 16, device="cuda").bfloat16().requires_grad_(True)
    t = torch.zeros(0, dtype=torch.int64, device="cuda")
    loss = ce(x, w, t)
    dx, dw = torch.autograd.grad(loss, [x, w])
    assert float(loss.detach()) == 0.0 and dx.shape == (0, 16) and dw.shape == (50, 16) and not dw.any()
    assert ce(x, w, t, reduction="none").shape == (0,)


@pytest.mark.parametrize("grads", [False, True])
def test_a_target_outside_the_vocabulary_is_reported_and_ignored(grads):
    import ravel_lm_b200._lib as L
    st = torch.cuda.current_stream().cuda_stream
    x, w, t = make(200, 32, 90, torch.bfloat16, seed=7)
    bad = t.clone()
    bad[3], bad[9], bad[150] = 90, -1, 1 << 40
    clean = t.clone()
    clean[[3, 9, 150]] = -100
    x.requires_grad_(grads)
    a = ce(x, w, bad)
    assert L.device_error(st) == L.RAVEL_DEVERR_INDEX
    L.clear_device_error(st)
    b = ce(x, w, clean)
    assert torch.equal(a, b) and L.device_error(st) == 0
    if grads:
        assert torch.equal(torch.autograd.grad(a, x)[0], torch.autograd.grad(b, x)[0])


def test_strides_alignment_dimensions_and_target_types():
    x, w, t = make(6 * 31, 72, 130, torch.bfloat16, seed=8)
    l0, (dx0, dw0) = check(x, w, t)
    xw, ww = torch.randn(6 * 31, 90, device="cuda").bfloat16(), torch.randn(130, 90, device="cuda").bfloat16()
    for off in (0, 1, 8):
        xw[:, off:off + 72], ww[:, off:off + 72] = x, w
        xl, wl = xw[:, off:off + 72].detach().requires_grad_(True), ww[:, off:off + 72].detach().requires_grad_(True)
        loss = ce(xl, wl, t.int())
        dx, dw = torch.autograd.grad(loss, [xl, wl])
        assert torch.equal(loss, l0) and torch.equal(dx, dx0) and torch.equal(dw, dw0)
        with torch.no_grad():
            assert torch.equal(ce(xl, wl, t.int()), ce(x, w, t))
    x3 = x.view(6, 31, 72).transpose(0, 1).contiguous().transpose(0, 1).requires_grad_(True)
    loss = ce(x3, w, t.view(6, 31).t().contiguous().t())
    assert torch.equal(loss, l0) and torch.equal(torch.autograd.grad(loss, x3)[0].reshape(-1, 72), dx0)
    assert ce(x3, w, t.view(6, 31), reduction="none").shape == (6, 31)
    one = ce(x[1], w, t[1])  # no leading dimension
    assert one.shape == () and torch.allclose(one, ce(x[1:2], w, t[1:2]))


def test_one_gradient_only_and_a_second_backward():
    x, w, t = make(300, 48, 400, torch.bfloat16, seed=9)
    _, (dx0, dw0) = check(x, w, t)
    for reduction in ("mean", "none"):
        up = torch.ones(300, device="cuda") if reduction == "none" else None
        xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss = ce(xl, wl, t, reduction=reduction)
        g1 = torch.autograd.grad(loss, [xl, wl], up, retain_graph=True)
        g1[0].zero_()
        g2 = torch.autograd.grad(loss, [xl, wl], up, retain_graph=True)
        gx, = torch.autograd.grad(loss, xl, up, retain_graph=True)
        gw, = torch.autograd.grad(loss, wl, up)
        assert torch.equal(g2[0], gx) and torch.equal(g2[1], gw) and gx.any()
        gx1, = torch.autograd.grad(ce(xl, w, t, reduction=reduction), xl, up)
        gw1, = torch.autograd.grad(ce(x, wl, t, reduction=reduction), wl, up)
        assert torch.equal(gx1, gx) and torch.equal(gw1, gw)
    wl = w.clone().requires_grad_(True)
    loss = ce(x, wl, t, reduction="none").sum()
    with torch.no_grad():
        wl += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_gradient_against_differences():
    """The loss's own derivative along random directions, by central differences in 64 bits."""
    x, w, t = make(64, 40, 150, torch.bfloat16, seed=10)
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(ce(xl, wl, t), [xl, wl])

    def loss(a, b):
        return torch.nn.functional.cross_entropy(a @ b.T, t, ignore_index=-100)
    g = torch.Generator(device="cuda").manual_seed(11)
    for _ in range(3):
        ax = torch.randn(64, 40, generator=g, device="cuda", dtype=torch.float64)
        aw = torch.randn(150, 40, generator=g, device="cuda", dtype=torch.float64)
        h = 1e-5
        num = (loss(x.double() + h * ax, w.double() + h * aw) - loss(x.double() - h * ax, w.double() - h * aw)) / (2 * h)
        got = (dx.double() * ax).sum() + (dw.double() * aw).sum()
        # roundings of 2^-9 of each element at most twice over, in random directions
        scale = 2.0 ** -8 * ((dx.double() * ax).norm() + (dw.double() * aw).norm()) * 4
        assert abs(float(num - got)) <= float(scale) + 1e-8, (float(num), float(got))


@pytest.mark.parametrize("M,K,V", [(200, 64, 1000), (1100, 1200, 24001)])
def test_the_same_bits_every_time_on_any_stream_and_replayed(M, K, V):
    x, w, t = make(M, K, V, torch.bfloat16, seed=12)
    x.requires_grad_(True)
    w.requires_grad_(True)
    l0 = ce(x, w, t)
    g0 = torch.autograd.grad(l0, [x, w])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:  # two calls at once
        with torch.cuda.stream(s):
            loss = ce(x, w, t)
            got.append((loss, torch.autograd.grad(loss, [x, w])))
    torch.cuda.synchronize()
    for loss, g in got:
        assert torch.equal(loss, l0) and all(torch.equal(a, b) for a, b in zip(g, g0))
    del loss, got
    xg, wg = x.detach().clone().requires_grad_(True), w.detach().clone().requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lg = ce(xg, wg, t)
        gg = torch.autograd.grad(lg, [xg, wg])
    x2, w2, t2 = make(M, K, V, torch.bfloat16, seed=13)
    with torch.no_grad():
        xg.copy_(x2)
        wg.copy_(w2)
    t.copy_(t2)
    for _ in range(2):
        graph.replay()
    x2.requires_grad_(True)
    w2.requires_grad_(True)
    l2 = ce(x2, w2, t2)
    g2 = torch.autograd.grad(l2, [x2, w2])
    assert torch.equal(lg, l2) and all(torch.equal(a, b) for a, b in zip(gg, g2))


def test_offsets_past_32_bits():
    V, K, M = 70000, 32768, 130  # 2.3e9 elements of weight and of its gradient
    g = torch.Generator(device="cuda").manual_seed(16)
    w = torch.zeros(V, K, dtype=torch.bfloat16, device="cuda")
    w[-3:] = (torch.randn(3, K, generator=g, device="cuda") * 0.01).bfloat16()
    x = torch.randn(M, K, generator=g, device="cuda").bfloat16()
    t = torch.randint(0, V, (M,), generator=g, device="cuda")
    t[:40], t[40:60] = V - 1, 5
    w.requires_grad_(True)
    loss = ce(x, w, t, reduction="sum")
    dw, = torch.autograd.grad(loss, w)
    z = x.double() @ w.detach()[-3:].double().T  # every other logit is 0
    s = (V - 3) + z.exp().sum(1)
    zt = torch.where((t >= V - 3)[:, None] & (torch.arange(V - 3, V, device="cuda") == t[:, None]), z, 0.0 * z).sum(1)
    assert abs(float(loss.detach()) - float((s.log() - zt).sum())) <= 1e-5 * float(loss.detach())
    for v in (0, 5, 6, V // 2, V - 4, V - 3, V - 1):
        p = (z[:, v - (V - 3)].exp() if v >= V - 3 else torch.ones_like(s)) / s
        d = p - (t == v).double()
        want, top = d @ x.double(), d.abs() @ x.double().abs()
        within(dw[v], want, 2.0 ** -7 * top + 2.0 ** -8 * want.abs() + 1e-30, f"d weight[{v}]")


def test_rows_past_32_bits():
    M, K, V = 70000, 32768, 6
    g = torch.Generator(device="cuda").manual_seed(17)
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    x[-200:] = torch.randn(200, K, generator=g, device="cuda").bfloat16()
    w = (torch.randn(V, K, generator=g, device="cuda") * K ** -0.5).bfloat16()
    t = torch.randint(0, V, (M,), generator=g, device="cuda")
    x.requires_grad_(True)
    loss = ce(x, w, t, reduction="none")
    want, d, dl, _ = reference(x[-200:], w, t[-200:])
    within(loss[-200:].detach(), want, dl + 4 * E * want.abs(), "losses")
    assert torch.allclose(loss[:1000].detach(), torch.full((1000,), math.log(V), device="cuda"))
    up = torch.zeros(M, device="cuda")
    up[-200:] = 1.0
    dx, = torch.autograd.grad(loss, x, up)
    wx = d @ w.double()
    within(dx[-200:], wx, (d.abs() * (2.0 ** -7 + 2 * dl[:, None])) @ w.double().abs() + 2.0 ** -8 * wx.abs() + 1e-30, "d x")
    assert not dx[:1000].any() and not dx[-1000:-200].any()


def test_non_finite_inputs_show():
    x, w, t = make(20, 16, 40, torch.bfloat16, seed=14, ignored=False)
    x[3, 2] = float("nan")
    loss = ce(x, w, t, reduction="none")
    assert math.isnan(float(loss[3])) and torch.isfinite(torch.cat([loss[:3], loss[4:]])).all()


def test_second_derivatives_and_tangents_are_refused():
    x, w, t = make(5, 16, 9, torch.bfloat16, seed=15)
    x.requires_grad_(True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(ce(x, w, t), x, create_graph=True)
    import torch.autograd.forward_ad as fwad
    with fwad.dual_level():
        dual = fwad.make_dual(x.detach(), torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            ce(dual, w, t)


def test_gradients_of_single_losses_without_rows():
    w = torch.randn(50, 16, device="cuda").bfloat16().requires_grad_(True)
    x = torch.zeros(0, 16, device="cuda").bfloat16().requires_grad_(True)
    t = torch.zeros(0, dtype=torch.int64, device="cuda")
    for _ in range(3):
        dirt = torch.full((1 << 20,), float("nan"), device="cuda")  # what the allocator hands out next
        del dirt
        loss = ce(x, w, t, reduction="none")
        dx, dw = torch.autograd.grad(loss, [x, w], torch.zeros(0, device="cuda"))
        assert dx.shape == (0, 16) and dw.shape == (50, 16) and not dw.any()


@pytest.mark.parametrize("dt,reduction,M,K,V", [
    (torch.bfloat16, "sum", 200, 256, 900), (torch.float16, "sum", 200, 256, 900), (torch.bfloat16, "none", 100, 256, 900),
    (torch.bfloat16, "sum", 1400, 512, 48000)])  # the last: the three-product form
def test_gradients_of_confident_rows_are_as_exact_as_others(dt, reduction, M, K, V):
    """Targets with 1 - p_t of 1e-4 to 1e-7, every row of its own token: relative to |d z|, of which the target's part
    is 1 - p_t, so that a difference 1 - p_t taken in float32 (off by 2^-24 of 1) would show.

    A logit's error moves 1 - p_t by p_t dl and hence by dl of itself (d log(1 - p_t) / d z_t = -p_t), another
    column's probability likewise: 2 dl of |d z| holds both, and no term of p_t is added.
    """
    u = torch.finfo(dt).eps / 2
    x, w, _ = make(M, K, V, dt, seed=18, scale=0.5, ignored=False)
    t = torch.arange(M, device="cuda") * (V // M) + 1
    # z_t = |x|^2 c, about log V + 9 to log V + 16; the other rows' logits with W_t are about N(0, c^2 K), small against it
    c = torch.linspace(math.log(V) + 9, math.log(V) + 16, M, device="cuda") / K
    w[t] = (x.float() * c[:, None]).to(dt)
    want, d, dl, _ = reference(x, w, t)
    rest = -torch.expm1(-want)  # 1 - p_t
    assert float(rest.max()) < 3e-3 and float(rest.median()) < 1e-5 and float(rest.min()) < 1e-6
    # from the other columns' probabilities, as a float64 difference at 1 - p_t = 1e-7 has 1e-9 of itself
    d.scatter_(1, t[:, None], 0.0)
    d.scatter_(1, t[:, None], -d.sum(1, keepdim=True))
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    got = torch.autograd.grad(ce(xl, wl, t, reduction=reduction), [xl, wl],
                              torch.ones(M, device="cuda") if reduction == "none" else None)
    xa, wa = x.double(), w.double()
    rel = 2 * u + 2 * dl[:, None]
    low = 2.0 ** -40 if dt == torch.float16 else 0.0
    want_x, want_w = d @ wa, d.T @ xa
    tx = (d.abs() * (rel + (V / 8 + 16) * 2.0 ** -23)) @ wa.abs() + low * wa.abs().sum(0) + (u + 4 * E) * want_x.abs()
    tw = (d.abs() * (rel + (M / 8 + 16) * 2.0 ** -23)).T @ xa.abs() + low * xa.abs().sum(0) + (u + 4 * E) * want_w.abs()
    within(got[0], want_x, tx + TINY[dt], "d x")
    within(got[1], want_w, tw + TINY[dt], "d weight")
    # and the bounds tell: gradients without the target's term lie beyond them in most elements
    without = d.clone()
    without.scatter_(1, t[:, None], 0.0)
    assert float(((without @ wa - want_x).abs() > tx + TINY[dt]).double().mean()) > 0.5
    assert float(((without.T @ xa - want_w).abs() > tw + TINY[dt])[t].double().mean()) > 0.5


@pytest.mark.parametrize("dt,K", [(torch.float16, 16), (torch.bfloat16, 16), (torch.bfloat16, 40)])
def test_a_last_piece_of_one_row(dt, K):
    """1024 rows a piece, four and a row; the last case takes three products."""
    check(*make(4097, K, 210000, dt, seed=19))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_row_whose_upstream_gradient_is_no_number_leaves_the_others(dt, bad):
    x, w, t = make(200, 64, 300, dt, seed=24, ignored=False)
    x.requires_grad_(True)
    loss = ce(x, w, t, reduction="none")
    up = torch.linspace(-1.0, 2.0, 200, device="cuda")
    up[3] = 0.0
    want, = torch.autograd.grad(loss, x, up, retain_graph=True)
    up[3] = bad
    got, = torch.autograd.grad(loss, x, up)
    rest = torch.arange(200, device="cuda") != 3
    assert torch.equal(got[rest], want[rest]) and torch.isfinite(want).all() and not torch.isfinite(got[3]).any()
