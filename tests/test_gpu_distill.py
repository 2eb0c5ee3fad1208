"""``distill_topk_loss`` against the formula in 64 bits.

Tolerances, with e = 2^-24 and exponents in base 2: a logit enters as
x = s log2(e) / T, whose constant and product are each rounded, so an exponent
x - max x is off by at most 4 e X, X = max |x| over the row's finite logits; ex2 and
lg2 are good to 2^-21; a sum's chain has at most V / 32 + 64 additions.  Hence

* q is relatively good to  dq = 4 e X + 2^-20 + (V / 32 + 64) e,
* p to the same with the teacher's magnitude and k: dp,
* the gradient c (q - P) to |c| (q dq + P dp) and its rounding u,
* a row's loss T^2 sum p (log p - log q) to T^2 (sum p |log p - log q| dp + dq + dp),

and the reduced loss to the sum of those (and its own R additions, by a tree of 1024).
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}
E = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import ravel_lm_b200._lib as L
    L.load()
    yield
    torch.cuda.synchronize()
    assert L.device_error(torch.cuda.current_stream().cuda_stream) == 0


def make(R, V, k, dtype, seed, tdtype=None, ragged=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = (torch.randn(R, V, generator=g, device="cuda") * 2).to(dtype).requires_grad_(True)
    ids = torch.randint(0, V, (R, k), generator=g, device="cuda")  # repeats among them
    t = (torch.randn(R, k, generator=g, device="cuda") * 2 + 3).to(tdtype or dtype)
    if ragged and k:
        n = torch.randint(0, k + 1, (R, 1), generator=g, device="cuda")
        ids = torch.where(torch.arange(k, device="cuda") < n, ids, torch.full_like(ids, -1))
        if R > 2:
            ids[R // 2] = -1
    return s, ids, t


def reference(s, ids, t, T, weight=1.0):
    """Rows' losses, d (sum of the rows' losses), live rows; and their tolerances."""
    u, tiny = U[s.dtype], TINY[s.dtype]
    s64, t64 = s.detach().double() / T, t.double() / T
    R, V = s64.shape
    k = ids.shape[1]
    live = (ids >= 0) & (ids < V) & (t64 != -math.inf)
    rows = live.any(1)
    safe = ids.clamp(0, V - 1)
    tt = torch.where(live, t64, torch.full_like(t64, -math.inf))
    lp = torch.where(live & rows[:, None], torch.log_softmax(tt, 1), torch.zeros_like(tt)) if k else tt
    p = torch.where(live, torch.exp(lp), torch.zeros_like(lp))
    lse = torch.logsumexp(s64, 1, keepdim=True)
    lq = s64 - lse
    q = torch.exp(lq)
    P = torch.zeros_like(q).scatter_add_(1, safe, p) if k else torch.zeros_like(q)
    diff = torch.where(p > 0, lp - lq.gather(1, safe), torch.zeros_like(p)) if k else p
    loss = weight * T * T * (p * diff).sum(1)
    grad = weight * T * (q - P)
    X = torch.where(torch.isfinite(s64) & (q > 0), s64.abs(), torch.zeros_like(s64)).amax(1, keepdim=True) * 1.4427
    Y = torch.where(live, t64.abs(), torch.zeros_like(t64)).amax(1, keepdim=True) * 1.4427 if k else X
    dq = 4 * E * X + 2.0 ** -20 + (V / 32 + 64) * E
    dp = 4 * E * Y + 2.0 ** -20 + (k / 32 + 64) * E
    tol_loss = abs(weight) * T * T * ((p * diff.abs()).sum(1) * dp[:, 0] + dq[:, 0] + dp[:, 0])
    tol_grad = abs(weight) * T * (q * dq + P * dp) + u * grad.abs()
    zero = ~rows
    loss, grad = loss.masked_fill(zero, 0.0), grad.masked_fill(zero[:, None], 0.0)
    tol_loss, tol_grad = tol_loss.masked_fill(zero, 0.0), tol_grad.masked_fill(zero[:, None], 0.0)
    return loss, grad, rows, tol_loss, tol_grad, tiny


def within(got, want, tol, what):
    if got.numel() == 0:
        return
    ok = ((got.double() - want).abs() <= tol) | ((want == got.double()) & torch.isinf(want))
    assert bool(ok.all()), (f"{what}: {int((~ok).sum())} of {ok.numel()} beyond tolerance, worst "
                            f"{float(((got.double() - want).abs() / tol)[~ok].max()):.3g} times")


def check(s, ids, t, T, reduction, weight=1.0, up=None):
    """Loss and gradient for a reduction and an upstream gradient (1 unless given)."""
    from ravel_lm_b200.distill import distill_topk_loss
    loss = distill_topk_loss(s, ids, t, temperature=T, reduction=reduction, weight=weight)
    R = s.reshape(-1, s.shape[-1]).shape[0]
    s2, i2, t2 = s.reshape(R, -1), ids.reshape(R, ids.shape[-1]), t.reshape(R, t.shape[-1])
    want, grad, rows, tl, tg, tiny = reference(s2, i2, t2, T, weight)
    n = max(1, int(rows.sum()))
    if reduction == "none":
        within(loss.reshape(-1), want, tl, "losses")
        up = torch.ones_like(loss) if up is None else up
        got, = torch.autograd.grad(loss, s, up)
        f = up.double().reshape(R, 1)
    else:
        div = n if reduction == "mean" else 1
        within(loss, want.sum() / div, (tl.sum() + (R / 1024 + 64) * E * want.abs().sum()) / div + 1e-30, "loss")
        got, = torch.autograd.grad(loss, s, up)
        f = (1.0 if up is None else float(up)) / div
    f = f * torch.ones(1, 1, dtype=torch.float64, device="cuda")
    within(got.reshape(R, -1), grad * f, tg * f.abs() + 8 * E * (grad * f).abs() + tiny, "d logits")
    dead = ~rows
    assert not got.reshape(R, -1)[dead].any(), "rows without an entry have no gradient"
    return loss, got


# a vocabulary of one, one row, odd rows (heads and tails of single elements), each block size
SHAPES = [(1, 1, 1), (4, 2, 3), (7, 5, 5), (3, 33, 8), (20, 1000, 16), (130, 1025, 20), (5, 4096, 64), (300, 2051, 7),
          (9, 32003, 33), (200, 20001, 20), (4, 65536, 100), (2, 131075, 4)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,k", SHAPES)
def test_step(R, V, k, dtype):
    s, ids, t = make(R, V, k, dtype, seed=R + V)
    loss, g = check(s, ids, t, 2.0, "mean")
    loss2, g2 = check(s, ids, t, 2.0, "mean")
    assert torch.equal(loss, loss2) and torch.equal(g, g2)
    with torch.no_grad():
        from ravel_lm_b200.distill import distill_topk_loss
        assert torch.equal(distill_topk_loss(s, ids, t, temperature=2.0), loss.detach())


# training steps of longer rows, around the lengths where the kernel's way changes; rows that start off 16 bytes;
# repeated ids, every row dead
@pytest.mark.parametrize("dtype,R,V,k", [
    (torch.bfloat16, 700, 8192, 5), (torch.bfloat16, 301, 16887, 128), (torch.bfloat16, 160, 16896, 64),
    (torch.bfloat16, 333, 32003, 31), (torch.bfloat16, 90, 65536, 64), (torch.bfloat16, 40, 131001, 33),
    (torch.bfloat16, 20, 140000, 129), (torch.float32, 650, 4096, 1), (torch.float32, 300, 8443, 16),
    (torch.float32, 200, 16001, 40), (torch.float32, 75, 50304, 100), (torch.float32, 9, 67500, 7),
    (torch.float32, 3, 70000, 7)])
def test_long_rows(dtype, R, V, k):
    s, ids, t = make(R, V, k, dtype, seed=R + k)
    for reduction, weight in (("mean", 1.0), ("sum", -0.5)):
        loss, g = check(s, ids, t, 1.5, reduction, weight)
        loss2, g2 = check(s, ids, t, 1.5, reduction, weight)
        assert torch.equal(loss, loss2) and torch.equal(g, g2)
    repeated = ids.clone()
    repeated[:, : k // 2] = repeated[:, k // 2 : k // 2 * 2]
    check(s, repeated, t, 1.0, "mean")
    check(s, torch.full_like(ids, -1), t, 1.0, "mean")


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_reductions_temperatures_weights_and_upstream_gradients(dtype, reduction):
    for T, weight, up in ((1.0, 1.0, None), (0.5, 0.3, 1.0), (4.0, 1.0, 2.5), (2.0, -1.0, 0.0)):
        s, ids, t = make(37, 1003, 12, dtype, seed=int(10 * T))
        if up is not None:
            up = torch.tensor(up, device="cuda")
            if reduction == "none":
                up = up * torch.randn(37, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
        check(s, ids, t, T, reduction, weight, up)


def test_types_of_ids_and_teacher():
    for dtype in DTYPES:
        for tdtype in DTYPES:
            s, ids, t = make(19, 515, 9, dtype, seed=3, tdtype=tdtype)
            a = check(s, ids, t, 1.5, "mean")
            b = check(s, ids.int(), t, 1.5, "mean")
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_a_second_backward_and_a_gradient_changed_in_place():
    from ravel_lm_b200.distill import distill_topk_loss
    s, ids, t = make(40, 777, 10, torch.float32, seed=4)
    loss = distill_topk_loss(s, ids, t, temperature=2.0)
    g1, = torch.autograd.grad(loss, s, retain_graph=True)
    want = g1.clone()
    g1.zero_()  # the caller may do what it likes with the gradient it was given
    g2, = torch.autograd.grad(loss, s, retain_graph=True)
    assert torch.equal(g2, want)
    g3, = torch.autograd.grad(loss, s, torch.tensor(2.0, device="cuda"), retain_graph=True)
    assert torch.equal(g3, 2 * want)
    assert torch.equal(g2, want)
    # as one term of a sum, scaled
    s2 = s.detach().clone().requires_grad_(True)
    (0.5 * distill_topk_loss(s2, ids, t, temperature=2.0) + (s2 * 0).sum()).backward()
    assert torch.allclose(s2.grad, 0.5 * want, rtol=1e-5, atol=1e-9)
    with torch.no_grad():
        s2 += 1
    loss = distill_topk_loss(s2, ids, t)
    with torch.no_grad():
        s2 += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss, s2)


def test_repeated_ids_add_up():
    s = torch.randn(3, 100, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).requires_grad_(True)
    ids = torch.tensor([[7, 7, 7, 7], [1, 2, 1, 2], [99, -1, 99, 0]], device="cuda")
    t = torch.tensor([[1.0, 2.0, 3.0, 4.0]] * 3, device="cuda")
    check(s, ids, t, 1.0, "sum")


def test_no_entries_and_no_rows():
    from ravel_lm_b200.distill import distill_topk_loss
    for k in (0, 3):
        s = torch.randn(5, 64, device="cuda", requires_grad=True)
        ids = torch.full((5, k), -1, device="cuda")
        for reduction in ("mean", "sum"):
            loss = distill_topk_loss(s, ids, torch.zeros(5, k, device="cuda"), reduction=reduction)
            g, = torch.autograd.grad(loss, s)
            assert float(loss) == 0.0 and not g.any()
    s = torch.empty(0, 64, device="cuda", requires_grad=True)
    ids, t = torch.empty(0, 3, dtype=torch.int64, device="cuda"), torch.empty(0, 3, device="cuda")
    for reduction in ("mean", "sum", "none"):
        loss = distill_topk_loss(s, ids, t, reduction=reduction)
        assert float(loss.sum()) == 0.0
        assert torch.autograd.grad(loss.sum(), s)[0].shape == (0, 64)


def test_masked_and_non_finite_values():
    """Logits of -inf (a masked vocabulary) and of the type's lowest value get no gradient; a teacher logit of -inf is
    no entry; a dead row's values do not matter; NaN and +inf stay in their rows."""
    from ravel_lm_b200.distill import distill_topk_loss
    for dtype in DTYPES:
        s, ids, t = make(12, 300, 6, dtype, seed=6, ragged=False)
        ids = ids % 200
        with torch.no_grad():
            s[0:4, 200:] = float("-inf")
            s[4:6, 200:] = torch.finfo(dtype).min
            t[1, :3] = float("-inf")
            t[2] = float("-inf")           # a row without entries
            ids[3] = -1
            s[3] = float("nan")            # ... whose logits do not matter
        loss, g = check(s, ids, t, 1.0, "mean")
        assert torch.isfinite(loss)
        assert not g[0:6, 200:].any()
        assert not g[2].any() and not g[3].any()
        with torch.no_grad():
            s[7, 5] = float("nan")
            s[8, 5] = float("inf")
            s[9] = float("-inf")
            s[10, ids[10, 0]] = float("-inf")
        losses = distill_topk_loss(s, ids, t, reduction="none")
        g, = torch.autograd.grad(losses, s, torch.ones_like(losses))
        assert torch.isnan(losses[7:10]).all() and torch.isnan(g[7]).all() and torch.isnan(g[9]).all()
        assert float(losses[10]) == math.inf and torch.isfinite(g[10]).all()
        want, grad, _, tl, tg, tiny = reference(s, ids, t, 1.0)
        keep = [0, 1, 2, 3, 4, 5, 6, 11]
        within(losses[keep], want[keep].nan_to_num(0.0), tl[keep].nan_to_num(0.0) + 1e-30, "losses")
        within(g[10], grad[10], tg[10] + tiny, "d logits of a row whose entry is masked")


def test_an_id_past_the_vocabulary_is_reported_and_not_used():
    import ravel_lm_b200._lib as L
    from ravel_lm_b200.distill import distill_topk_loss
    s, ids, t = make(6, 50, 4, torch.float32, seed=7, ragged=False)
    ids2 = ids.clone()
    ids2[2, 1] = 50
    ids2[4] = 2 ** 33 + 1
    st = torch.cuda.current_stream().cuda_stream
    loss = distill_topk_loss(s, ids2, t, reduction="none")
    assert L.device_error(st) == L.RAVEL_DEVERR_INDEX
    L.clear_device_error(st)
    ids[2, 1], ids[4] = -1, -1
    assert torch.equal(loss, distill_topk_loss(s, ids, t, reduction="none"))
    assert L.device_error(st) == 0


def test_strides_and_leading_dimensions():
    from ravel_lm_b200.distill import distill_topk_loss
    g = torch.Generator(device="cuda").manual_seed(8)
    big = torch.randn(4, 10, 1100, generator=g, device="cuda").bfloat16()
    for s in (big[..., :1024], big[..., 3:1030], big[:, ::2, 5:], big.transpose(0, 1)[..., :900],
              big[:1].expand(3, 10, 1100), big[0, 0], big.permute(2, 0, 1)[:60]):
        V = s.shape[-1]
        ids = torch.randint(0, V, (*s.shape[:-1], 10), generator=g, device="cuda")[..., ::2]
        t = torch.randn(*s.shape[:-1], 5, generator=g, device="cuda").bfloat16()
        s1, s2 = s.detach().requires_grad_(True), s.detach().clone().requires_grad_(True)
        l1, g1 = check(s1, ids, t, 1.0, "mean")
        l2, g2 = check(s2, ids, t, 1.0, "mean")
        assert g1.shape == s.shape
        within(l1, l2.double(), 1e-5 * l2.abs().double(), "loss of a view and of its copy")


def test_gradient_against_differences():
    s, ids, t = make(5, 60, 6, torch.float32, seed=9)
    T, h = 1.7, 1e-6
    _, g = check(s, ids, t, T, "sum")
    v = torch.randn(5, 60, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").double()

    class Shift:  # the reference's loss at s + h v, in 64 bits
        def __init__(self, x):
            self.x, self.dtype = x, torch.float32

        def detach(self):
            return self.x
    up = reference(Shift(s.detach().double() + h * v), ids, t, T)[0].sum()
    dn = reference(Shift(s.detach().double() - h * v), ids, t, T)[0].sum()
    want, got = float(up - dn) / (2 * h), float((g.double() * v).sum())
    assert abs(got - want) <= 1e-5 * float((g.double() * v).abs().sum()) + 1e-7


def test_another_stream_and_graph_replay():
    from ravel_lm_b200.distill import distill_topk_loss
    s, ids, t = make(64, 1031, 8, torch.bfloat16, seed=10)
    loss, g = check(s, ids, t, 2.0, "mean")
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        l2 = distill_topk_loss(s, ids, t, temperature=2.0)
        g2, = torch.autograd.grad(l2, s)
    st.synchronize()
    assert torch.equal(loss, l2) and torch.equal(g, g2)
    graph = torch.cuda.CUDAGraph()
    x = s.detach().clone().requires_grad_(True)
    with torch.cuda.graph(graph):
        lg = distill_topk_loss(x, ids, t, temperature=2.0)
        gg, = torch.autograd.grad(lg, x)
    new = torch.randn(64, 1031, device="cuda").bfloat16()
    with torch.no_grad():
        x.copy_(new)
    for _ in range(2):  # replays do not depend on what an earlier one left
        graph.replay()
    want_l = distill_topk_loss(x, ids, t, temperature=2.0)
    assert torch.equal(lg, want_l) and torch.equal(gg, torch.autograd.grad(want_l, x)[0])


def test_offsets_past_32_bits():
    from ravel_lm_b200.distill import distill_topk_loss
    R, V = 33000, 65537
    s = torch.zeros(R, V, dtype=torch.bfloat16, device="cuda")
    tail, ids_t, t_t = make(50, V, 6, torch.bfloat16, seed=11)
    with torch.no_grad():
        s[-50:] = tail
    s.requires_grad_(True)
    ids = torch.full((R, 6), -1, device="cuda")
    ids[-50:] = ids_t
    t = torch.zeros(R, 6, dtype=torch.bfloat16, device="cuda")
    t[-50:] = t_t
    loss = distill_topk_loss(s, ids, t, temperature=2.0)
    g, = torch.autograd.grad(loss, s)
    ls = distill_topk_loss(tail, ids_t, t_t, temperature=2.0)
    gs, = torch.autograd.grad(ls, tail)
    assert abs(float(loss) - float(ls)) <= 1e-5 * abs(float(ls))
    # the two tensors' rows start at other alignments: the sums' order differs, the rounding to 16 bits mostly not
    within(g[-50:], gs.double(), 2.0 ** -7 * gs.double().abs() + 2.0 ** -126, "d logits")
    assert not g[:-50].any()


def test_refusals():
    from ravel_lm_b200.distill import distill_topk_loss
    s, ids, t = make(4, 16, 3, torch.float32, seed=12, ragged=False)
    with pytest.raises(ValueError, match="reduction"):
        distill_topk_loss(s, ids, t, reduction="max")
    with pytest.raises(ValueError, match="teacher_ids and teacher_logits"):
        distill_topk_loss(s, ids[:2], t)
    with pytest.raises(ValueError, match="teacher_ids and teacher_logits"):
        distill_topk_loss(s, ids[0], t[0])
    with pytest.raises(ValueError, match="V >= 1"):
        distill_topk_loss(s[:, :0], ids, t)
    for T in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            distill_topk_loss(s, ids, t, temperature=T)
    with pytest.raises(ValueError, match="must not require a gradient"):
        distill_topk_loss(s, ids, t.requires_grad_(True))
    t = t.detach()
    with pytest.raises(TypeError, match="int32 or int64"):
        distill_topk_loss(s, ids.float(), t)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        distill_topk_loss(s.double(), ids, t)
    with pytest.raises(ValueError, match="unsupported|range"):
        distill_topk_loss(s, ids.repeat(1, 2000), t.repeat(1, 2000))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        distill_topk_loss(s.cpu(), ids.cpu(), t.cpu())
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        distill_topk_loss(s, ids.cpu(), t)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(distill_topk_loss(s, ids, t), s, create_graph=True)
