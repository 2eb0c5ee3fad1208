"""``token_embedding`` against the formula in 64 bits.

Tolerances, with e = 2^-24 and u half a step of the type (eps / 2): an output is a product
rounded to float32 and once more to the type, |y| (u + e); a token's gradient adds n
rows in float32, at most (n + 2) e sum |g| scale in all, and is rounded once.  Subnormal results of a
16-bit type are off by half its smallest number at most.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
E = 2.0 ** -24
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import ravel_lm_b200._lib as L
    L.load()
    yield
    torch.cuda.synchronize()
    assert L.device_error(torch.cuda.current_stream().cuda_stream) == 0


def embed(*a, **k):
    from ravel_lm_b200.vocab import token_embedding
    return token_embedding(*a, **k)


def within(got, want, tol, what):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} beyond tolerance"


def check(ids, w, gy, scale=1.0, pad=None):
    """Output and gradient of a call with ids in the vocabulary."""
    dt, V, K = w.dtype, *w.shape
    u = torch.finfo(dt).eps / 2
    w = w.detach().requires_grad_(True)
    y = embed(ids, w, scale=scale, padding_idx=pad)
    assert y.shape == (*ids.shape, K) and y.dtype == dt
    want = w.detach().double()[ids.long()] * scale
    within(y.detach(), want, want.abs() * (u + E) + TINY[dt], "y")
    dw, = torch.autograd.grad(y, w, gy)
    assert dw.shape == w.shape and dw.dtype == dt
    flat, g = ids.reshape(-1).long(), gy.reshape(-1, K).double()
    if pad is not None:
        flat, g = flat[flat != pad % V], g[flat != pad % V]
    s = torch.zeros(V, K, dtype=torch.float64, device="cuda").index_add_(0, flat, g)
    a = torch.zeros(V, K, dtype=torch.float64, device="cuda").index_add_(0, flat, g.abs())
    n = torch.bincount(flat, minlength=V).double()[:, None]
    within(dw, s * scale, abs(scale) * (n + 2) * E * a + (s * scale).abs() * (u + E) + TINY[dt], "d weight")
    return y, dw


def make(N, V, K, dt, seed, zipf=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if zipf:
        cdf = torch.arange(1, V + 1, dtype=torch.float64, device="cuda").pow(-1.1).cumsum(0)
        ids = torch.searchsorted(cdf, torch.rand(N, generator=g, dtype=torch.float64, device="cuda") * cdf[-1])
        ids = ids.clamp_max(V - 1)
    else:
        ids = torch.randint(0, V, (N,), generator=g, device="cuda")
    w = torch.randn(V, K, generator=g, device="cuda").to(dt)
    return ids, w, torch.randn(N, K, generator=g, device="cuda").to(dt)


# one of everything; up to 512 ids in one launch, then ranges of sums that end inside, at and behind tokens; odd widths;
# several digits of ids (2^10 and 2^20 are the borders of one and two passes); several steps a tile (past 131072 ids)
SHAPES = [(1, 1, 1), (1, 7, 8), (2, 2, 3), (15, 1, 4), (16, 3, 5), (17, 300, 64), (64, 512, 33), (65, 513, 40),
          (512, 1025, 40), (513, 1024, 8), (1000, 5, 256), (2048, 1000, 100), (2049, 1025, 1), (4097, 32003, 24),
          (9000, 40, 520), (300, 262145, 8), (300, 1300000, 4), (2000, 1050000, 4), (300001, 700, 4), (20000, 65536, 16)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,V,K", SHAPES)
def test_sizes(dt, N, V, K):
    check(*make(N, V, K, dt, seed=N + K), scale=1.0 if K % 2 else 22.5)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,V,K", [(512, 3, 520), (500, 40, 17), (5000, 50, 128), (40000, 1000, 96), (70000, 30000, 33)])
def test_frequent_tokens(dt, N, V, K):
    check(*make(N, V, K, dt, seed=7, zipf=True), scale=-3.0)
    ids, w, gy = make(N, V, K, dt, seed=8)
    check(torch.full_like(ids, V - 1), w, gy)  # a single token


@pytest.mark.parametrize("ids_dtype", [torch.int32, torch.int64])
def test_leading_dimensions_strides_and_alignment(ids_dtype):
    ids, w, gy = make(6 * 50, 90, 72, torch.bfloat16, seed=1)
    ids = ids.to(ids_dtype)
    y0, d0 = check(ids, w, gy)
    y, d = check(ids.view(6, 50), w, gy.view(6, 50, 72))
    assert torch.equal(y.reshape(-1, 72), y0) and torch.equal(d, d0)
    # strided rows, rows that start off 16 bytes, ids and gradients laid out otherwise
    wide = torch.randn(90, 100, device="cuda").bfloat16()
    for off in (0, 1, 8):
        wide[:, off:off + 72] = w
        v = wide[:, off:off + 72]
        leaf = v.detach().requires_grad_(True)
        y2 = embed(ids.view(6, 50), leaf)
        assert torch.equal(y2.reshape(-1, 72), y0)
        gt = gy.view(6, 50, 72).transpose(0, 1).contiguous().transpose(0, 1)
        assert torch.equal(torch.autograd.grad(y2, leaf, gt)[0], d0)
    tr = ids.view(6, 50).t().contiguous().t()
    assert torch.equal(embed(tr, w).reshape(-1, 72), y0)
    # a broadcast gradient
    leaf = w.clone().requires_grad_(True)
    d, = torch.autograd.grad(embed(ids, leaf).sum(), leaf)
    check_n = torch.bincount(ids.long(), minlength=90).bfloat16()
    assert torch.equal(d, check_n[:, None].expand(90, 72))


@pytest.mark.parametrize("N", [400, 3000])  # in one launch, and sorted
def test_padding_id_and_no_ids(N):
    ids, w, gy = make(N, 60, 40, torch.float32, seed=2)
    _, d = check(ids, w, gy, pad=11)
    assert not d[11].any() and d[12].any()
    _, d2 = check(ids, w, gy, pad=11 - 60)
    assert torch.equal(d, d2)
    # what stands at padding positions does not matter
    bad = gy.clone()
    bad[ids == 11] = float("nan")
    leaf = w.clone().requires_grad_(True)
    d3, = torch.autograd.grad(embed(ids, leaf, padding_idx=11), leaf, bad)
    assert torch.equal(d3, d)
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    leaf = w.clone().requires_grad_(True)
    y = embed(none, leaf)
    assert y.shape == (0, 40) and not torch.autograd.grad(y.sum(), leaf)[0].any()
    empty = torch.zeros(60, 0, device="cuda", requires_grad=True)
    assert embed(ids, empty).shape == (N, 0)


@pytest.mark.parametrize("N", [500, 1500])
def test_ids_outside_the_vocabulary_are_reported_and_not_used(N):
    import ravel_lm_b200._lib as L
    ids, w, gy = make(N, 60, 40, torch.bfloat16, seed=3)
    ids[3], ids[77], ids[400] = 60, -1, 1 << 40
    ok = (ids >= 0) & (ids < 60)
    leaf = w.clone().requires_grad_(True)
    y = embed(ids, leaf)
    d, = torch.autograd.grad(y, leaf, gy)
    st = torch.cuda.current_stream().cuda_stream
    assert L.device_error(st) == L.RAVEL_DEVERR_INDEX
    L.clear_device_error(st)
    assert not y[~ok].any() and torch.equal(y[ok], w[ids[ok]])
    leaf2 = w.clone().requires_grad_(True)
    d2, = torch.autograd.grad(embed(ids[ok], leaf2), leaf2, gy[ok])
    assert torch.allclose(d.float(), d2.float(), rtol=2 ** -7, atol=1e-6)  # other ranges: another order of sums
    assert L.device_error(st) == 0


@pytest.mark.parametrize("N", [512, 30000])
def test_the_same_bits_every_time_on_any_stream_and_replayed(N):
    ids, w, gy = make(N, 2000, 64, torch.float32, seed=4, zipf=True)
    y, d = check(ids, w, gy)
    leaf = w.clone().requires_grad_(True)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        y2 = embed(ids, leaf)
        d2, = torch.autograd.grad(y2, leaf, gy)
    st.synchronize()
    assert torch.equal(y, y2) and torch.equal(d, d2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y3 = embed(ids, leaf, scale=2.0)
        d3, = torch.autograd.grad(y3, leaf, gy)
    ids2, _, gy2 = make(N, 2000, 64, torch.float32, seed=5)
    ids.copy_(ids2)
    gy.copy_(gy2)
    for _ in range(2):
        graph.replay()
    leaf2 = w.clone().requires_grad_(True)
    y4 = embed(ids, leaf2, scale=2.0)
    assert torch.equal(y3, y4) and torch.equal(d3, torch.autograd.grad(y4, leaf2, gy)[0])


def test_offsets_past_32_bits():
    V, K = 70000, 32768  # 2.3e9 elements
    w = torch.zeros(V, K, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(6)
    w[-3:] = torch.randn(3, K, generator=g, device="cuda").bfloat16()
    ids = torch.tensor([V - 1, 0, V - 3, V - 1], device="cuda")
    w.requires_grad_(True)
    y = embed(ids, w)
    assert torch.equal(y.detach(), w.detach()[ids])
    gy = torch.randn(4, K, generator=g, device="cuda").bfloat16()
    d, = torch.autograd.grad(y, w, gy)
    assert torch.equal(d[V - 1], (gy[0].float() + gy[3].float()).bfloat16()) and torch.equal(d[V - 3], gy[2])
    assert not d[1:V - 3].any() and not d[V - 2].any()


def test_outputs_past_32_bits():
    N, V, K = 70000, 3, 32768
    g = torch.Generator(device="cuda").manual_seed(8)
    w = torch.randn(V, K, generator=g, device="cuda").bfloat16().requires_grad_(True)
    ids = torch.randint(0, 2, (N,), generator=g, device="cuda")
    ids[-2:] = 2
    y = embed(ids, w)
    for i in (0, 65535, 65536, N - 1):
        assert torch.equal(y[i], w[ids[i]])
    gy = torch.zeros(N, K, dtype=torch.bfloat16, device="cuda")
    gy[-3:] = torch.randn(3, K, generator=g, device="cuda").bfloat16()
    d, = torch.autograd.grad(y, w, gy)
    assert torch.equal(d[2], (gy[-2].float() + gy[-1].float()).bfloat16())
    assert torch.equal(d[ids[-3]], gy[-3]) and not d[1 - ids[-3]].any()


def test_second_derivatives_and_tangents_are_refused():
    ids, w, gy = make(5, 9, 8, torch.float32, seed=9)
    w.requires_grad_(True)
    gy.requires_grad_(True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(embed(ids, w), w, gy, create_graph=True)
    import torch.autograd.forward_ad as fwad
    with fwad.dual_level():
        dual = fwad.make_dual(w.detach(), torch.ones_like(w))
        with pytest.raises(RuntimeError, match="forward-mode"):
            embed(ids, dual)
