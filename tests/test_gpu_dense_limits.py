"""``fused_linear`` where a sum leaves the 16-bit type's range or lies near zero.

The inputs are powers of two and their small multiples, so that the exact sums, derivatives and gradients are
known; where a tolerance is needed it is the accumulation's and the output's rounding, as in the general tests.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import ravel_lm_b200._lib as L
    L.load()
    yield
    torch.cuda.synchronize()
    assert L.device_error(torch.cuda.current_stream().cuda_stream) == 0


# one row (plain loads), few rows (single CTAs), a long sum (divided over a cluster), many rows (pairs)
@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("M,K,N", [(1, 64, 72), (5, 64, 72), (24, 8192, 512), (2100, 256, 2056)])
def test_sums_beyond_float16(M, K, N, act):
    """Sums of +-96000 are infinite in float16, where they are kept for the backward; the derivative is 1 or 0.

    d x[m, k] = sum_n gy[m, n] act' w[n, k]: products of at most (N + 8) float32 roundings and the output's.
    """
    from ravel_lm_b200.dense import fused_linear
    g = torch.Generator(device="cuda").manual_seed(M)
    sign = torch.where(torch.rand(N, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    x = torch.full((M, K), 64.0, device="cuda").half().requires_grad_(True)
    w = (sign[:, None] * (1500.0 / K)).expand(N, K).contiguous().half().requires_grad_(True)
    b = torch.zeros(N, device="cuda").half().requires_grad_(True)
    gy = torch.randn(M, N, generator=g, device="cuda").half()
    y = fused_linear(x, w, b, activation=act)
    assert bool((y[:, sign < 0] == 0).all()) and bool((y[:, sign > 0] == math.inf).all())
    dx, dw, db = torch.autograd.grad(y, [x, w, b], gy)
    dz = torch.where(sign > 0, gy.double(), torch.zeros_like(gy).double())
    for name, got, want, size, n in (
            ("dx", dx, dz @ w.detach().double(), dz.abs() @ w.detach().double().abs(), N),
            ("dw", dw, dz.t() @ x.detach().double(), dz.abs().t() @ x.detach().double().abs(), M),
            ("db", db, dz.sum(0), dz.abs().sum(0), M)):
        tol = (n + 8) * 2.0 ** -23 * size + U[torch.float16] * want.abs() + TINY[torch.float16]
        over = want.abs() > 65000  # d w may leave float16 itself
        ok = ((got.double() - want).abs() <= tol) | over
        assert bool(ok.all()), f"{name}: {int((~ok).sum())} of {ok.numel()} wrong"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
def test_derivative_at_infinity(act, dtype):
    """dz of a kept sum of +inf is dy, of -inf zero; NaN stays NaN."""
    import ravel_lm_b200._lib as L
    M, N = 20, 264
    z = torch.zeros(M, N, dtype=dtype, device="cuda")
    z[:, 0::3], z[:, 1::3] = math.inf, -math.inf
    z[3, 2], z[7, 5] = math.nan, math.nan
    gy = torch.randn(M, N, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    dz = torch.empty_like(gy)
    code = L.RAVEL_BF16 if dtype == torch.bfloat16 else L.RAVEL_F16
    codes = {"relu": L.RAVEL_ACT_RELU, "gelu": L.RAVEL_ACT_GELU, "silu": L.RAVEL_ACT_SILU}
    L.call("ravel_linear_dz", gy.data_ptr(), N, z.data_ptr(), N, codes[act], dz.data_ptr(), N, None, M, N, None, 0, None,
           0, None, 0, code, None, 0, torch.cuda.current_stream().cuda_stream)
    assert torch.equal(dz[:, 0::3], gy[:, 0::3])
    assert not dz[:, 1::3].any() and not torch.isnan(dz[:, 1::3]).any()
    assert torch.isnan(dz[3, 2]) and torch.isnan(dz[7, 5]) and int(torch.isnan(dz).sum()) == 2


# one row (plain loads), few rows (single CTAs), a long sum (divided over a cluster), many rows (pairs)
@pytest.mark.parametrize("M,K,N", [(1, 64, 72), (5, 64, 72), (24, 8192, 512), (2100, 256, 2056)])
def test_relu_of_sums_that_underflow(M, K, N):
    """z = +-2^-27 is 0 in float16, where it is kept for the backward; its derivative is 1 or 0, that of an exact
    zero 0.  The bias gradient of a gradient of ones counts them (in float16: exactly to 2048, else to its rounding)."""
    from ravel_lm_b200.dense import fused_linear
    x = torch.zeros(M, K, device="cuda").half()
    x[:, 3] = 2.0 ** -13
    w = torch.zeros(N, K, device="cuda").half()
    w[0::3, 3], w[1::3, 3] = 2.0 ** -14, -2.0 ** -14
    b = torch.zeros(N, device="cuda").half()
    for t in (x, w, b):
        t.requires_grad_(True)
    dx, dw, db = torch.autograd.grad(fused_linear(x, w, b, activation="relu"), [x, w, b],
                                     torch.ones(M, N, device="cuda").half())
    on = (torch.arange(N, device="cuda") % 3 == 0).double()
    assert bool(((db.double() - M * on).abs() <= U[torch.float16] * M * on).all())
    # d w[n, 3] = M 2^-13, d x[m, 3] = 2^-14 for each of the positive columns: exact sums, one rounding
    assert bool(((dw[:, 3].double() - M * 2.0 ** -13 * on).abs() <= U[torch.float16] * M * 2.0 ** -13 * on).all())
    want = float(on.sum()) * 2.0 ** -14
    assert bool(((dx[:, 3].double() - want).abs() <= U[torch.float16] * want).all())


def near_zero(M, K, N, col, dtype, scale=1.0, sign=1.0, dead=()):
    """Column `col` sums to sign scale (255 2^-26 - 2^-20) > 0 (sign 1), in an order in which a product of 1 hides
    the 255 small ones from an accumulator of some 25 bits until a product of -1 takes it away.  The other columns
    sum to scale, those in `dead` to 0."""
    x = torch.zeros(M, K, device="cuda")
    x[:, 0], x[:, 1:256], x[:, 256], x[:, 300] = 1.0, 2.0 ** -13, 1.0, 2.0 ** -10
    w = torch.zeros(N, K, device="cuda")
    w[:, 0] = scale
    for n in dead:
        w[n] = 0.0
    w[col] = 0.0
    w[col, 0], w[col, 1:256], w[col, 256], w[col, 300] = (sign * scale * v for v in (1.0, 2.0 ** -13, -1.0, -2.0 ** -10))
    x, w = x.to(dtype), w.to(dtype)
    exact = float(x[0].double() @ w[col].double())
    assert exact == sign * scale * (255 * 2.0 ** -26 - 2.0 ** -20)
    return x, w


# the only column; the only one of its group of 8 (and of its strip of 256); a group whose other columns are dead
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,col,dead", [(1, 0, ()), (3, 1, (0, 2)), (129, 128, ()), (257, 256, ()), (258, 257, (256,)),
                                        (513, 512, ()), (64, 20, (16, 17, 18, 19, 21, 22, 23))])
def test_relu_sign_without_neighbours(N, col, dead, dtype):
    """Whatever stands beside a sum near zero, its derivative is that of the float32 sum: lanes of 8 elements a chunk
    of 256 keep the 248 small products of lanes 1 to 31 (3.7e-6) beside the 2^-20 taken away."""
    from ravel_lm_b200.dense import fused_linear
    for M in (2, 40, 300):
        for sign in (1.0, -1.0):
            x, w = near_zero(M, 512, N, col, dtype, sign=sign, dead=dead)
            b = torch.zeros(N, device="cuda", dtype=dtype).requires_grad_(True)
            db, = torch.autograd.grad(fused_linear(x, w, b, activation="relu"), b, torch.ones(M, N, device="cuda", dtype=dtype))
            want = torch.ones(N, device="cuda", dtype=torch.float64) * M
            want[list(dead)] = 0
            want[col] = M if sign > 0 else 0
            assert bool(((db.double() - want).abs() <= U[dtype] * want).all()), (M, sign, db[col])


def test_relu_sign_of_a_sum_that_underflows():
    """The same with a sum of 1e-8, which float16 does not hold: its kept sign is only the tensor cores'."""
    from ravel_lm_b200.dense import fused_linear
    for M in (2, 40, 300):
        for sign in (1.0, -1.0):
            x, w = near_zero(M, 512, 72, 30, torch.float16, scale=2.0 ** -8, sign=sign)
            b = torch.zeros(72, device="cuda").half().requires_grad_(True)
            db, = torch.autograd.grad(fused_linear(x, w, b, activation="relu"), b, torch.ones(M, 72, device="cuda").half())
            want = torch.full((72,), float(M), device="cuda")
            want[30] = M if sign > 0 else 0
            assert torch.equal(db.float(), want), (M, sign, db[30])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,col", [(72, 30), (257, 256), (1, 0)])
def test_relu_sign_of_a_sum_swallowed_whole(N, col, dtype):
    """The same without the 2^-20: what an accumulator of some 25 bits leaves of 1 + 255 2^-26 - 1 may be 0."""
    from ravel_lm_b200.dense import fused_linear
    for M in (2, 40, 300):
        for sign in (1.0, -1.0):
            x, w = near_zero(M, 512, N, col, dtype, sign=sign)
            w[col, 300] = 0.0
            assert float(x[0].double() @ w[col].double()) == sign * 255 * 2.0 ** -26
            b = torch.zeros(N, device="cuda", dtype=dtype).requires_grad_(True)
            db, = torch.autograd.grad(fused_linear(x, w, b, activation="relu"), b, torch.ones(M, N, device="cuda", dtype=dtype))
            want = torch.full((N,), float(M), device="cuda", dtype=torch.float64)
            want[col] = M if sign > 0 else 0
            assert bool(((db.double() - want).abs() <= U[dtype] * want).all()), (M, sign, db[col])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_relu_of_rows_and_columns_of_zeros(dtype):
    """Rows of x and columns of weights that are zero throughout (-0 among them) leave the bias; where that is 0 too the
    derivative is 0.  Beside them the other sums, and in a zero column of weights the sums that a zero bias leaves."""
    from ravel_lm_b200.dense import fused_linear
    M, K, N = 700, 1000, 520
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(M, K, generator=g, device="cuda").to(dtype)
    w = (torch.randn(N, K, generator=g, device="cuda") * K ** -0.5).to(dtype)
    b = torch.randn(N, generator=g, device="cuda").to(dtype)
    x[::5] = 0.0
    x[::10] = -0.0
    w[::7] = -0.0
    b[::3] = 0.0
    z = x.double() @ w.double().t() + b.double()
    gy = torch.randn(M, N, generator=g, device="cuda").to(dtype)
    b.requires_grad_(True)
    db, = torch.autograd.grad(fused_linear(x, w, b, activation="relu"), b, gy)
    sure = (z == 0) | (z.abs() > (K / 32 + 16) * 2.0 ** -24 * 4)  # as in the general test of signs
    dz = gy.double() * (z > 0)
    tol = (M + 8) * 2.0 ** -23 * dz.abs().sum(0) + U[dtype] * dz.sum(0).abs() + (gy.double().abs() * ~sure).sum(0)
    assert bool(((db.double() - dz.sum(0)).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("density", [0.02, 0.3])
def test_relu_of_sparse_inputs(density, dtype):
    """Ones, minus ones and zeros: sums are small whole numbers, many of them 0, and every derivative is known."""
    from ravel_lm_b200.dense import fused_linear
    M, K, N = 900, 512, 600
    g = torch.Generator(device="cuda").manual_seed(2)

    def sparse(*shape):
        keep = torch.rand(*shape, generator=g, device="cuda") < density
        sign = torch.where(torch.rand(*shape, generator=g, device="cuda") < 0.5, -1.0, 1.0)
        return (keep * sign).to(dtype)
    x, w, b = sparse(M, K), sparse(N, K), sparse(N)
    z = x.double() @ w.double().t() + b.double()
    assert float((z == 0).double().mean()) > 0.02
    for t in (x, w, b):
        t.requires_grad_(True)
    gy = torch.ones(M, N, device="cuda", dtype=dtype)
    dx, dw, db = torch.autograd.grad(fused_linear(x, w, b, activation="relu"), [x, w, b], gy)
    dz = (z > 0).double()
    for got, want in ((dx, dz @ w.detach().double()), (dw, dz.t() @ x.detach().double()), (db, dz.sum(0))):
        assert bool(((got.double() - want).abs() <= U[dtype] * want.abs()).all())  # whole numbers, rounded once
