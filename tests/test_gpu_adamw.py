"""``adamw_step`` and ``AdamW`` against the formula in 64 bits.

Tolerances, with e = 2^-24: a state is a sum of two products, each operation rounded (and the clipping
factor and the constants once): 4 e (|b m| + |(1 - b) g|), 6 e likewise for v.  The update
lr m^ / (sqrt(v^) + eps) has some ten roundings and two approximations of 2^-22; where m is a difference of larger terms
its own error counts: lr / (1 - b1^t) (4 e (|b1 m| + |(1 - b1) g|)) / (sqrt(v^) + eps) more.  A parameter adds its own rounding, e |p|.
A 16-bit parameter is its master rounded once.  8-bit states are compared with the two codes around the
64-bit value.
"""
from __future__ import annotations

import copy
import math
import pickle

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
HYPER = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import ravel_lm_b200._lib as L
    L.load()
    yield
    torch.cuda.synchronize()
    assert L.device_error(torch.cuda.current_stream().cuda_stream) == 0


def step(*a, **k):
    from ravel_lm_b200.optim import adamw_step
    return adamw_step(*a, **k)


def values(code, exponents, signed):
    """What codes stand for, in 64 bits, from the format's definition."""
    c = code.reshape(-1).double()
    ex = exponents.double().repeat_interleave(256)[:c.numel()]
    neg = signed & (c >= 128)
    a = torch.where(neg, c - 128, c)
    field, man, bias = torch.floor(a / 8), torch.remainder(a, 8), 15 if signed else 31
    y = torch.where(field > 0, (1 + man / 8) * torch.exp2(field - bias), man * 2.0 ** (-bias - 2))
    return (torch.where(neg, -y, y) * torch.exp2(ex)).view(code.shape)


class Case:
    """Lists of tensors of the given sizes; states as after some steps."""

    def __init__(self, sizes, dtype, bits, seed=0, offset=0, g_scale=1e-2):
        gen = torch.Generator(device="cuda").manual_seed(seed)

        def rand(n, scale=1.0):
            return torch.randn(n + offset, generator=gen, device="cuda")[offset:] * scale

        def place(t, dt):  # a view that begins `offset` elements into its storage
            out = torch.zeros(t.numel() + offset, dtype=dt, device="cuda")[offset:]
            return out.copy_(t)
        self.dtype, self.bits = dtype, bits
        half = dtype != torch.float32
        p = [rand(n, 0.5) for n in sizes]
        self.g = [place(rand(n) * torch.exp(rand(n)) * g_scale, dtype) for n in sizes]
        self.masters = [place(q, torch.float32) for q in p] if half else None
        self.p = [place(q, dtype) for q in p]
        self.step = torch.full((1,), 10, dtype=torch.int64, device="cuda")
        self.me = self.ve = None
        if bits == 32:
            self.m = [place(rand(n, 0.3 * g_scale), torch.float32) for n in sizes]
            self.v = [place((rand(n, g_scale) ** 2), torch.float32) for n in sizes]
        else:
            def codes(n, low, high):
                return place(torch.randint(low, high, (n,), generator=gen, device="cuda"), torch.uint8)
            e = round(math.log2(g_scale))
            self.m = [codes(n, 0, 256) for n in sizes]
            self.v = [codes(n, 100, 256) for n in sizes]
            self.me = [torch.full(((n + 255) // 256,), e - 2, dtype=torch.int8, device="cuda") for n in sizes]
            self.ve = [torch.full(((n + 255) // 256,), 2 * e, dtype=torch.int8, device="cuda") for n in sizes]

    def clone(self):
        return copy.deepcopy(self)

    def run(self, **k):
        return step(self.p, self.g, self.m, self.v, self.step, masters=self.masters, exp_avg_exponents=self.me,
                    exp_avg_sq_exponents=self.ve, **{**HYPER, **k})

    def state(self, i):
        if self.bits == 32:
            return self.m[i].double(), self.v[i].double()
        return values(self.m[i], self.me[i], True), values(self.v[i], self.ve[i], False)


def around(x, exponents, signed, n):
    """The spacing of codes around each value: the grid below 2^exponent."""
    bias = 15 if signed else 31
    ex = exponents.double().repeat_interleave(256)[:n]
    y = x.abs() * torch.exp2(-ex)
    return torch.exp2(torch.floor(torch.log2(y.clamp_min(2.0 ** (1 - bias)))) - 3 + ex)


def check(case, max_norm=None, **k):
    before = case.clone()
    hyper = {**HYPER, **k}
    norm = case.run(max_norm=max_norm, **k)
    b1, b2 = hyper["betas"]
    lr, t = float(hyper["lr"]), int(before.step) + 1
    assert int(case.step) == t
    clip = 1.0
    if max_norm is not None:
        want = math.sqrt(sum(float((g.double() ** 2).sum()) for g in before.g))
        assert abs(float(norm) - want) <= 2 * E * want
        clip = min(1.0, max_norm / (want + 1e-6))
    else:
        assert norm is None
    for i in range(len(case.p)):
        g = before.g[i].double() * clip
        m0, v0 = before.state(i)
        m, v = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g * g
        tm = 4 * E * ((b1 * m0).abs() + ((1 - b1) * g).abs()) + 2.0 ** -149
        tv = 6 * E * v + 2.0 ** -149
        d = torch.sqrt(v / (1 - b2 ** t)) + hyper["eps"]
        p0 = (before.p if before.masters is None else before.masters)[i].double()
        upd = lr * (m / (1 - b1 ** t)) / d
        p = p0 * (1 - lr * hyper["weight_decay"]) - upd
        tol = 2 * E * p0.abs() + E * p.abs() + (16 * E + 2.0 ** -21) * upd.abs() + lr / (1 - b1 ** t) * tm / d
        got = (case.p if case.masters is None else case.masters)[i]
        assert bool(((got.double() - p).abs() <= tol).all()), i
        if case.masters is not None:
            assert torch.equal(case.p[i], case.masters[i].to(case.dtype))
        gm, gv = case.state(i)
        if case.bits == 32:
            assert bool(((gm - m).abs() <= tm).all()) and bool(((gv - v).abs() <= tv).all()), i
        elif m.numel():
            n = m.numel()
            assert bool(((gm - m).abs() <= around(m, case.me[i], True, n) * (1 + 1e-6) + tm).all()), i
            assert bool(((gv - v).abs() <= around(v, case.ve[i], False, n) * (1 + 1e-6) + tv).all()), i
            for x, ex in ((m, case.me[i]), (v, case.ve[i])):  # the least power of two that holds a block
                top = torch.nn.functional.pad(x.abs(), (0, -n % 256)).view(-1, 256).amax(1)
                hi = 1.875 * torch.exp2(ex.double())
                live = top > 2.0 ** -120
                assert bool((top <= hi * (1 + 1e-6))[live].all()) and bool((top > hi / 2 * (1 - 1e-6))[live].all())
    return case


SIZES = [[1], [255, 256, 257], [0, 5, 0], [2047, 2048, 2049, 1], [100000, 7, 4096], [64] * 50]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes", SIZES)
def test_sizes(dtype, bits, sizes):
    check(Case(sizes, dtype, bits, seed=len(sizes)))
    check(Case(sizes, dtype, bits, seed=1), max_norm=0.5)
    check(Case(sizes, dtype, bits, seed=2), max_norm=1e6)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_off_16_bytes_and_many_of_them(dtype, bits):
    for off in (1, 3):
        check(Case([1000, 513, 9], dtype, bits, offset=off), max_norm=1.0)
    sizes = [(i * 37) % 300 + 1 for i in range(1000)]  # more than one launch's
    a = check(Case(sizes, dtype, bits, seed=3), max_norm=0.3)
    b = Case(sizes, dtype, bits, seed=3)
    b.run(max_norm=0.3)
    for x, y in zip(a.p + a.m + a.v, b.p + b.m + b.v):  # the same bits every time
        assert torch.equal(x, y)


def test_hyper_parameters_and_lr_on_the_device():
    for k in (dict(lr=0.0), dict(weight_decay=0.0), dict(betas=(0.0, 0.0)), dict(eps=0.0), dict(eps=1e-3),
              dict(betas=(0.95, 0.9999))):
        check(Case([3000], torch.float32, 32, seed=4), **k)
    a, b = Case([3000], torch.bfloat16, 8, seed=5), Case([3000], torch.bfloat16, 8, seed=5)
    lr = torch.tensor(0.0625, device="cuda")
    a.run(lr=0.0625)
    b.run(lr=lr)
    assert torch.equal(a.p[0], b.p[0]) and torch.equal(a.m[0], b.m[0])
    lr.fill_(0.0)
    keep = b.masters[0].clone()
    b.run(lr=lr)
    assert torch.equal(b.masters[0], keep)


def test_gradients_of_every_size():
    """The norm of gradients whose squares leave float32; the smallest and the largest gradients."""
    for scale in (1e-30, 1e25, 1e-18):
        c = Case([5000], torch.float32, 32, seed=6, g_scale=1e-2)
        c.g[0].mul_(scale)
        want = float(c.g[0].double().norm())
        got = c.run(max_norm=1.0)
        assert abs(float(got) - want) <= 2 * E * want
    check(Case([3000], torch.float32, 8, seed=7, g_scale=2.0 ** -40))
    check(Case([3000], torch.float32, 8, seed=7, g_scale=2.0 ** 30))


def test_stochastic_rounding_keeps_small_changes():
    """v moves by 1% of the distance to g^2 a step, far less than a grid step of 1/8: on average it still arrives."""
    n = 1 << 16
    p, g = torch.zeros(n, device="cuda"), torch.full((n,), 0.01, device="cuda")
    m, v = (torch.zeros(n, dtype=torch.uint8, device="cuda") for _ in range(2))
    me, ve = (torch.full((n // 256,), -126, dtype=torch.int8, device="cuda") for _ in range(2))
    t = torch.zeros(1, dtype=torch.int64, device="cuda")
    for _ in range(300):
        step([p], [g], [m], [v], t, exp_avg_exponents=[me], exp_avg_sq_exponents=[ve], **HYPER)
    gv, gm = values(v, ve, False), values(m, me, True)
    want = 1e-4 * (1 - 0.99 ** 300)
    # each step's rounding has at most a quarter of a squared grid step (v / 8) variance; they decay by 0.99 a step
    sd = 0.5 / 8 * 1e-4 / math.sqrt(1 - 0.99 ** 2) / math.sqrt(n)
    assert abs(float(gv.mean()) - want) <= 5 * sd + 1e-9
    assert abs(float(gm.mean()) - 0.01 * (1 - 0.9 ** 300)) <= 5 * (0.5 / 8 * 0.01 / math.sqrt(1 - 0.81) / math.sqrt(n))


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_non_finite_gradients(bad):
    c = Case([1000], torch.float32, 32, seed=8)
    c.g[0][300] = bad
    before = c.clone()
    c.run()
    assert not torch.isfinite(c.m[0][300]) and torch.isfinite(c.m[0]).sum() == 999
    keep = torch.arange(1000, device="cuda") != 300
    before.g[0][300] = 0.0
    before.run()
    assert torch.equal(c.p[0][keep], before.p[0][keep])
    e = Case([1000], torch.float32, 8, seed=8)
    e.g[0][300] = bad
    e.run()
    assert e.me[0].tolist()[1] == -128 and (e.me[0] == -128).sum() == 1 and (e.ve[0] == -128).sum() == 1
    from ravel_lm_b200.optim import state_values
    assert torch.isnan(state_values(e.m[0], e.me[0], signed=True)).sum() == 256
    e.run()
    assert torch.isnan(e.p[0][256:512]).all() and torch.isfinite(e.p[0][:256]).all()
    n = Case([1000], torch.float32, 32, seed=9)
    n.g[0][5] = bad
    assert not math.isfinite(float(n.run(max_norm=1.0)))


@pytest.mark.parametrize("n", [1, 255, 4096, 5001])
def test_state_values(n):
    from ravel_lm_b200.optim import state_values
    g = torch.Generator(device="cuda").manual_seed(n)
    for off in (0, 1):
        code = torch.randint(0, 256, (n + off,), generator=g, device="cuda").to(torch.uint8)[off:]
        ex = torch.randint(-100, 100, ((n + 255) // 256,), generator=g, device="cuda").to(torch.int8)
        for signed in (True, False):
            want = values(code, ex, signed)
            assert torch.equal(state_values(code, ex, signed=signed).double(), want.float().double())
            ok = (want == 0) | (want.abs() > 2.0 ** -120)  # bfloat16 holds 4 significant bits
            assert torch.equal(state_values(code, ex, signed=signed, dtype=torch.bfloat16).double()[ok], want[ok])


def test_global_norm_of_mixed_types():
    from ravel_lm_b200.optim import global_norm
    ts = [torch.randn(1000, 3, device="cuda"), torch.randn(77, device="cuda").bfloat16(), torch.randn(5, device="cuda").half(),
          torch.randn(40, 50, device="cuda").t(), torch.zeros(0, device="cuda")]
    want = math.sqrt(sum(float((t.double() ** 2).sum()) for t in ts))
    got = global_norm(ts)
    assert got.dtype == torch.float64 and got.shape == () and abs(float(got) - want) <= 1e-14 * want
    assert float(global_norm([torch.zeros(0, device="cuda")])) == 0.0
    a, b = Case([500], torch.float32, 32), Case([500], torch.float32, 32)
    n = global_norm(a.g)
    assert torch.equal(a.run(max_norm=0.1, norm=n), b.run(max_norm=0.1)) and torch.equal(a.p[0], b.p[0])


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count_on(bits):
    a, b = Case([5000, 33], torch.bfloat16, bits, seed=10), Case([5000, 33], torch.bfloat16, bits, seed=10)
    lr = torch.tensor(0.01, device="cuda")
    a.run(lr=lr, max_norm=0.5)
    b.run(lr=lr, max_norm=0.5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = a.run(lr=lr, max_norm=0.5)
    for i in range(3):
        lr.fill_(0.01 * (i + 1))
        for x, y in zip(a.g, b.g):
            x.normal_(std=0.01)
            y.copy_(x)
        graph.replay()
        want = b.run(lr=lr, max_norm=0.5)
        assert torch.equal(norm, want)
    assert int(a.step) == int(b.step) == 14
    for x, y in zip(a.p + a.masters + a.m + a.v, b.p + b.masters + b.m + b.v):
        assert torch.equal(x, y)


@pytest.mark.parametrize("bits", [32, 8])
def test_offsets_past_32_bits(bits):
    n, k = (1 << 31) + 1000, 5000
    big = Case([k], torch.bfloat16, bits, seed=12)
    small = Case([k], torch.bfloat16, bits, seed=12)
    tail = (n - k) // 256 * 256  # a block's start, so that the small case has the same blocks
    cut = n - tail

    def grow(t, dt):
        out = torch.zeros(n, dtype=dt, device="cuda")
        out[tail:] = torch.nn.functional.pad(t, (0, cut - k)) if cut > k else t[:cut]
        return out
    for c in (big.p, big.g, big.masters, big.m, big.v):
        c[0] = grow(c[0], c[0].dtype)
    for c in (small.p, small.g, small.masters, small.m, small.v):
        c[0] = torch.nn.functional.pad(c[0], (0, cut - k))
    if bits == 8:
        for name in ("me", "ve"):
            e = torch.full(((n + 255) // 256,), -126, dtype=torch.int8, device="cuda")
            se = torch.full(((cut + 255) // 256,), -126, dtype=torch.int8, device="cuda")
            se[:(k + 255) // 256] = getattr(small, name)[0]
            e[tail // 256:] = se
            setattr(big, name, [e])
            setattr(small, name, [se.clone()])
    big.run(max_norm=0.5)
    small.run(max_norm=0.5)
    assert torch.equal(big.masters[0][tail:], small.masters[0]) and torch.equal(big.p[0][tail:], small.p[0])
    assert not big.masters[0][:1 << 20].any() and not big.m[0][tail - (1 << 20):tail].any()
    if bits == 32:
        assert torch.equal(big.m[0][tail:], small.m[0]) and torch.equal(big.v[0][tail:], small.v[0])
    else:  # other random bits: the codes around the same values
        m, v = values(big.m[0][tail:], big.me[0][tail // 256:], True), values(small.m[0], small.me[0], True)
        assert bool(((m - v).abs() <= around(torch.maximum(m.abs(), v.abs()), small.me[0], True, cut)).all())


def test_another_stream_and_gradients_laid_out_otherwise():
    a, b = Case([64 * 48], torch.float32, 32, seed=11), Case([64 * 48], torch.float32, 32, seed=11)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        a.run()
    st.synchronize()
    b.p = [b.p[0].view(64, 48)]
    b.g = [b.g[0].view(64, 48).t().contiguous().t()]
    version = b.p[0]._version
    b.run()
    assert torch.equal(a.p[0], b.p[0].view(-1)) and b.p[0]._version > version


# ------------------------------------------------------------------ the optimizer
def model(seed, dtype=torch.float32):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(40, 65), torch.nn.Tanh(), torch.nn.Linear(65, 7)).cuda().to(dtype)


def grads(m, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    for p in m.parameters():
        p.grad = torch.randn(p.shape, generator=g, device="cuda").to(p.dtype) * 0.1


def test_optimizer_against_torch():
    from ravel_lm_b200.optim import AdamW
    a, b = model(0), model(0)
    groups = lambda m: [{"params": m[0].parameters(), "lr": 1e-3}, {"params": m[2].parameters(), "weight_decay": 0.3}]  # noqa: E731
    oa = AdamW(groups(a), lr=5e-3, betas=(0.8, 0.95), max_norm=1.0)
    ob = torch.optim.AdamW(groups(b), lr=5e-3, betas=(0.8, 0.95))
    for i in range(6):
        grads(a, i)
        grads(b, i)
        for m in (a, b):
            if i == 2:
                m[2].bias.grad = None  # a parameter without a gradient counts no step
            if i < 2:
                m[0].weight.grad = None  # and one may come later
        want = torch.nn.utils.clip_grad_norm_(b.parameters(), 1.0)
        oa.step()
        ob.step()
        assert abs(float(oa.grad_norm) - float(want)) <= 1e-6 * float(want)
        oa.param_groups[0]["lr"] = ob.param_groups[0]["lr"] = 1e-3 * (i + 1)
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.allclose(p, q, rtol=1e-5, atol=1e-6)
    assert [int(oa.state[p]["step"]) for p in a.parameters()] == [4, 6, 6, 5]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_copy_and_pickle_go_on_as_the_original(dtype, bits):
    from ravel_lm_b200.optim import AdamW

    def fresh(m):
        return AdamW(m.parameters(), lr=1e-2, state_bits=bits, max_norm=2.0)
    a = model(1, dtype)
    oa = fresh(a)
    for i in range(3):
        grads(a, i)
        if i == 1:
            a[0].bias.grad = None
        oa.step()
    b = copy.deepcopy(a)
    ob = fresh(b)
    ob.load_state_dict(oa.state_dict())
    c, oc = copy.deepcopy((a, oa))
    d, od = pickle.loads(pickle.dumps((a, oa)))
    for i in range(3, 5):
        for m, o in ((a, oa), (b, ob), (c, oc), (d, od)):
            grads(m, i)
            o.step()
    for m, o in ((b, ob), (c, oc), (d, od)):
        for p, q in zip(a.parameters(), m.parameters()):
            assert torch.equal(p, q)
            for k, v in oa.state[p].items():
                assert torch.equal(v, o.state[q][k]) and v.dtype == o.state[q][k].dtype, k
    if dtype == torch.bfloat16:
        st = oa.state[a[0].weight]
        assert st["master"].dtype == torch.float32 and torch.equal(st["master"].bfloat16(), a[0].weight)
        with torch.no_grad():
            a[0].weight.fill_(1.0)
        oa.reset_masters()
        assert torch.equal(st["master"], torch.ones_like(st["master"]))
    with pytest.raises(ValueError, match="state_bits"):
        AdamW(model(1, dtype).parameters(), state_bits=40 - bits).load_state_dict(oa.state_dict())


def test_optimizer_closure_no_gradients_and_capture():
    from ravel_lm_b200.optim import AdamW
    m = model(2)
    o = AdamW(m.parameters(), lr=torch.tensor(1e-3, device="cuda"), max_norm=1.0)
    o.step()  # nothing to do
    x = torch.randn(9, 40, device="cuda")

    def closure():
        o.zero_grad()
        loss = m(x).square().mean()
        loss.backward()
        return loss
    l0 = float(o.step(closure).detach())
    assert float(closure().detach()) < l0
    twin = copy.deepcopy((m, o))
    for p, q in zip(m.parameters(), twin[0].parameters()):
        q.grad = p.grad.clone()  # a copy of a parameter has no gradient
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        o.step()
    for _ in range(2):
        graph.replay()
        twin[1].step()
    torch.cuda.synchronize()
    for p, q in zip(m.parameters(), twin[0].parameters()):
        assert torch.equal(p, q)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [1e-20, 1e-40, 1e-50, 0.0])
def test_gradients_whose_squares_are_subnormal(bits, eps):
    """A first step from states of zero moves by lr g / (|g| + eps), whatever the size of g and eps; no gradient, no step.

    v = (1 - b2) g^2 lies on the grid of subnormal numbers, off by at most 2^-149 (g^2 and the sum, half of a
    smallest number each): at most 0.4% of v for |g| >= 2e-20, and half of it in the root; lr g / |g| has the usual rest.
    """
    n = 3000
    gen = torch.Generator(device="cuda").manual_seed(20)
    size = torch.exp(torch.empty(n, device="cuda").uniform_(math.log(2e-20), math.log(1e-17), generator=gen))
    g = size * torch.where(torch.rand(n, generator=gen, device="cuda") < 0.5, -1.0, 1.0)
    if eps > 0.0:
        g[::7] = 0.0
    p = torch.zeros(n, device="cuda")
    blocks = (n + 255) // 256
    m, v = (torch.zeros(n, dtype=torch.float32 if bits == 32 else torch.uint8, device="cuda") for _ in range(2))
    ex = {}
    if bits == 8:
        ex = {k: [torch.full((blocks,), -126, dtype=torch.int8, device="cuda")]
              for k in ("exp_avg_exponents", "exp_avg_sq_exponents")}
    t = torch.zeros(1, dtype=torch.int64, device="cuda")
    hyper = dict(lr=1e-2, betas=(0.9, 0.999), eps=eps, weight_decay=0.0)
    step([p], [g], [m], [v], t, **ex, **hyper)
    gd = g.double()
    want = torch.where(gd == 0, 0.0, -1e-2 * gd / (gd.abs() + eps))
    tol = want.abs() * (2.0 ** -149 / (1e-3 * gd * gd).clamp_min(1e-300) + 2.0 ** -20)
    tol[gd == 0] = 0.0
    assert bool(((p.double() - want).abs() <= tol).all()), float((p.double() - want).abs().max())
    for _ in range(3):
        step([p], [g], [m], [v], t, **ex, **hyper)
    assert not p[g == 0].any() and bool(torch.isfinite(p).all())


@pytest.mark.parametrize("eps", [0.0, 1e-8])
def test_a_second_moment_of_nan_shows(eps):
    c = Case([600], torch.float32, 32, seed=21)
    c.v[0][300] = float("nan")
    c.run(eps=eps)
    assert torch.isnan(c.p[0]).nonzero().flatten().tolist() == [300]
    e = Case([600], torch.float32, 8, seed=21)
    e.ve[0][1] = -128  # a block that stands for NaN
    e.run(eps=eps)
    assert torch.isnan(e.p[0]).nonzero().flatten().tolist() == list(range(256, 512))


@pytest.mark.parametrize("r", [1e-5, 1e-6])
def test_blocks_with_a_wide_range_take_steps_of_lr(r):
    """Half of each block has gradients r times the other half's.  A small element's second moment must not be rounded to 0
    while its first moment is not, which would divide the one by eps.

    With b1 = 0.9, b2 = 0.999 Cauchy's inequality gives |m| <= 7.3 sqrt(v) in exact arithmetic, a block's largest values
    among them.  m's smallest step is 2^-17 2^e <= 2^-17 1.07 max |m|, v's smallest value 2^-33 2^e >= 2^-33 max v / 1.875,
    so that one step of m over the root of v's smallest value is at most 7.3 * 1.07 * 1.37 / sqrt(2) = 7.6; with the value
    that was rounded (7.3) and the new gradient's part (0.1 / sqrt(0.001) = 3.2) no step passes 18.1 lr, or 20.4 with the
    values' own roundings of 1/8 (bias correction: sqrt(1 - b2^t) / (1 - b1^t) <= 1).
    """
    from ravel_lm_b200.optim import AdamW, state_values
    n = 64 * 256
    gen = torch.Generator(device="cuda").manual_seed(22)
    small = torch.arange(n, device="cuda") % 256 >= 128
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    opt = AdamW([p], lr=1.0, betas=(0.9, 0.999), weight_decay=0.0, state_bits=8)
    worst = torch.zeros((), device="cuda")
    for _ in range(100):
        p.grad = torch.randn(n, generator=gen, device="cuda") * torch.where(small, r, 1.0)
        p.data.zero_()
        opt.step()
        worst = torch.maximum(worst, p.detach().abs().max())
    assert float(worst) <= 20.4
    st = opt.state[p]
    assert bool((st["exp_avg_sq"] > 0).all())
    assert bool((state_values(st["exp_avg_sq"], st["exp_avg_sq_exponents"], signed=False) > 0).all())


@pytest.mark.parametrize("n,off", [(1000, 0), (1000, 1), (4096, 0)])
def test_positive_second_moments(n, off):
    """Exactly 0 keeps code 0, a positive value has code 1 at least; all else is as without the option."""
    def go(**k):
        c = Case([n], torch.float32, 8, seed=23, offset=off)
        c.g[0].zero_()
        c.g[0][::3] = 1e-2
        c.g[0][1::3] = 1e-11
        c.m[0].zero_(), c.v[0].zero_()
        c.run(**k)
        return c
    a, b = go(), go(positive_exp_avg_sq=True)
    none = torch.arange(n, device="cuda") % 3 == 2
    assert not b.v[0][none].any() and bool((b.v[0][~none] > 0).all()) and not a.v[0][1::3].any()
    assert torch.equal(b.v[0], torch.where(none, a.v[0], a.v[0].clamp_min(1))) and torch.equal(a.ve[0], b.ve[0])
    assert torch.equal(a.m[0], b.m[0]) and torch.equal(a.me[0], b.me[0]) and torch.equal(a.p[0], b.p[0])
    with pytest.raises(ValueError, match="8-bit states only"):
        Case([n], torch.float32, 32).run(positive_exp_avg_sq=True)


def test_a_capture_refuses_what_a_replay_would_repeat():
    """States made, or a step count copied, inside a capture would start again in every replay."""
    from ravel_lm_b200.optim import AdamW
    m = model(4)
    o = AdamW(m.parameters(), lr=1e-2, max_norm=1.0)
    grads(m, 0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before a capture"):
        with torch.cuda.graph(graph):
            o.step()
    assert not any(o.state.values())
    o.step()
    gone = m[2].bias.grad
    m[2].bias.grad = None  # has counted a step, and has no gradient now
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before a capture"):
        with torch.cuda.graph(graph):
            o.step()
    o.step()  # as the message says
    twin = copy.deepcopy((m, o))
    for p, q in zip(m.parameters(), twin[0].parameters()):
        q.grad = None if p.grad is None else p.grad.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o.step()
    for _ in range(3):
        graph.replay()
        twin[1].step()
    torch.cuda.synchronize()
    assert gone is not None and [int(o.state[p]["step"]) for p in m.parameters()] == [5, 5, 5, 1]
    for p, q in zip(m.parameters(), twin[0].parameters()):
        assert torch.equal(p, q)
