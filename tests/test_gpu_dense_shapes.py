"""Every launch shape of the matrix product, in every direction and with every epilogue, against the formula in 64
bits under the general tests' tolerances; each test first checks that its sizes reach the shape they stand for."""
from __future__ import annotations

import pytest
import torch

from dense_shapes import CASES, ROWS, plan, plans
from test_gpu_dense import ACTS, check, make, step

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import ravel_lm_b200._lib as L
    yield L.load()
    torch.cuda.synchronize()
    assert L.device_error(torch.cuda.current_stream().cuda_stream) == 0


def check_step(M, K, N, act, dtype, bias=True, residual=True):
    x, w, b, r = make(M, K, N, dtype, seed=M + K, bias=bias, residual=residual, grad=True)
    gy = torch.randn(M, N, generator=torch.Generator(device="cuda").manual_seed(N), device="cuda").to(dtype)
    y, g = step(x, w, b, r, act, gy)
    check(x, w, b, r, act, y, g, gy)
    y2, g2 = step(x, w, b, r, act, gy)
    assert torch.equal(y, y2) and all(torch.equal(g[n], g2[n]) for n in g), "the same inputs give the same bits"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("sizes,y,dx,dw", CASES)
def test_step(lib, sizes, y, dx, dw, act, dtype):
    assert plans(lib, *sizes) == (y, dx, dw)
    check_step(*sizes, act, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bias,residual", [(False, True), (True, False), (False, False)])
@pytest.mark.parametrize("sizes", [(40, 4864, 5024), (24, 4509, 5023), (24, 8192, 512), (24, 3888, 41)])
def test_divided_sums_with_parts_of_the_epilogue(lib, sizes, bias, residual, dtype):
    assert plans(lib, *sizes)[0][2] > 1
    check_step(*sizes, "silu", dtype, bias, residual)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("K,N,warps", ROWS)
def test_one_row(lib, K, N, warps, act, dtype):
    assert plan(lib, 1, N, K, 0) == (0, warps, 1)
    check_step(1, K, N, act, dtype)
