"""CPU-only checks of the dense operators' boundary: C-ABI refusals before any launch, workspace sizes, and the
Python functions' refusals (no CPU path)."""
from __future__ import annotations

import ctypes

import pytest
import torch

INVALID, WORKSPACE, UNSUPPORTED = 1, 2, 4
P = 4096  # a pointer that is never followed (16-byte aligned)


@pytest.fixture(scope="module")
def lib():
    import ravel_lm_b200._lib as L
    return L.load()


def matmul(lib, A=P, lda=64, a_mn=0, B=P, ldb=64, b_mn=0, M=8, N=8, K=64, bias=None, res=None, ldr=8, act=0, y=P, ldy=8,
           z=None, ldz=8, dtype=1):
    return lib.ravel_matmul(A, lda, a_mn, B, ldb, b_mn, M, N, K, bias, res, ldr, act, y, ldy, z, ldz, dtype, None)


def test_matmul_refuses_on_the_host(lib):
    assert matmul(lib, M=-1) == INVALID
    assert matmul(lib, act=7) == INVALID
    assert matmul(lib, dtype=0) == UNSUPPORTED
    assert matmul(lib, M=(1 << 30) + 1) == UNSUPPORTED
    assert matmul(lib, a_mn=1) == UNSUPPORTED                       # MN-major A with K-major B
    assert matmul(lib, b_mn=1, bias=P) == UNSUPPORTED               # an epilogue on a gradient product
    assert matmul(lib, A=None) == INVALID
    assert matmul(lib, y=None) == INVALID
    assert matmul(lib, lda=56) == INVALID                           # rows shorter than K
    assert matmul(lib, ldy=7) == INVALID
    assert matmul(lib, A=P + 2) == INVALID                          # TMA: 16-byte addresses
    assert matmul(lib, ldb=68) == INVALID                           # ... and pitches
    assert matmul(lib, M=0, A=None, y=None) == 0                    # nothing to do


def test_dz_pad_and_norm_refuse_on_the_host(lib):
    def dz(g, ldg, z, ldz, act, out, ldd, gb, M, N, dtype, scratch, sb, stream, x=None, w=None):
        return lib.ravel_linear_dz(g, ldg, z, ldz, act, out, ldd, gb, M, N, x, 8, w, 8, None, 8, dtype, scratch, sb, stream)
    assert dz(P, 8, None, 8, 2, P, 8, None, 4, 8, 1, None, 0, None) == INVALID      # gelu needs z
    assert dz(P, 8, None, 8, 0, None, 8, P, 4, 8, 1, None, 0, None) == WORKSPACE
    assert dz(P, 8, None, 8, 0, P, 8, None, 4, 8, 3, None, 0, None) == UNSUPPORTED
    assert dz(P, 8, P, 8, 1, P, 8, None, 4, 8, 1, None, 0, None, x=P) == INVALID       # x without a weight
    assert dz(P, 8, P, 8, 1, P, 8, None, 4, 8, 1, None, 0, None, x=P + 2, w=P) == INVALID
    assert lib.ravel_linear_dz_scratch_bytes(100, 256) >= 256 * 4
    assert lib.ravel_linear_dz_scratch_bytes(-1, 256) == 0
    assert lib.ravel_pad_rows(P, 4, 3, 8, P, 8, 1, None) == INVALID                 # rows overlap
    assert lib.ravel_pad_rows(None, 8, 0, 8, None, 8, 1, None) == 0
    f = ctypes.c_float(1e-5)
    fwd = lib.ravel_layer_norm_fwd
    assert fwd(P, 8, None, None, f, P, None, None, 4, 0, 0, None) == INVALID
    assert fwd(P, 8, None, None, f, P, P, None, 4, 8, 0, None) == INVALID           # mean without rstd
    assert fwd(P, 8, None, None, f, P, None, None, 4, 8, 3, None) == UNSUPPORTED
    bwd = lib.ravel_layer_norm_bwd
    assert bwd(P, 8, None, P, 8, P, P, P, P, None, 4, 8, 0, None, 0, None) == INVALID  # one weight gradient
    assert bwd(P, 8, None, P, 8, P, P, P, P, P, 4, 8, 0, None, 0, None) == WORKSPACE
    assert lib.ravel_layer_norm_scratch_bytes(1, 100) == 2 * 100 * 4


def test_distill_refuses_on_the_host(lib):
    def fwd(R=2, V=8, k=2, T=1.0, red=2, dtype=0, tdtype=0, idt=1, losses=P, out=P, scratch=P, sb=1 << 20, grad=None,
            stat=None):
        return lib.ravel_distill_topk_fwd(P, V, P, idt, P, tdtype, R, V, k, T, 1.0, red, losses, stat, out, grad, dtype,
                                          scratch, sb, None)
    assert fwd(V=0) == INVALID
    assert fwd(T=0.0) == INVALID
    assert fwd(T=float("nan")) == INVALID
    assert fwd(idt=2) == INVALID
    assert fwd(dtype=3) == UNSUPPORTED
    assert fwd(tdtype=3) == UNSUPPORTED
    assert fwd(k=5000) == UNSUPPORTED


def test_python_refusals_without_a_gpu():
    from ravel_lm_b200.dense import fused_linear
    from ravel_lm_b200.distill import distill_topk_loss
    from ravel_lm_b200.glue import layer_norm
    x, w = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        fused_linear(x, w)
    with pytest.raises(ValueError, match="activation"):
        fused_linear(x, w, activation="swish")
    with pytest.raises(ValueError, match="weight"):
        fused_linear(x, w[:, :7])
    with pytest.raises(TypeError):
        fused_linear(x.float(), w.float())
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        layer_norm(x, eps=1e-5)
    with pytest.raises(ValueError):
        layer_norm(x, torch.zeros(7, dtype=torch.bfloat16))
    ids = torch.zeros(2, 3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        distill_topk_loss(x, ids, torch.zeros(2, 3))
    with pytest.raises(ValueError, match="reduction"):
        distill_topk_loss(x, ids, torch.zeros(2, 3), reduction="max")
    with pytest.raises(ValueError, match="temperature"):
        distill_topk_loss(x, ids, torch.zeros(2, 3), temperature=0.0)


def test_distill_refuses_a_gradient_without_the_statistics(lib):
    """grad needs stat, with which the count that the mean's gradient divides by is made."""
    for reduction in (1, 2):
        for args in ((2, 8, 2), (0, 8, 2)):
            R, V, k = args
            rc = lib.ravel_distill_topk_fwd(P, V, P, 1, P, 0, R, V, k, 1.0, 1.0, reduction, P, None, P, P, 0, P, 1 << 20, None)
            assert rc == INVALID


def test_forward_mode_tangents_are_refused():
    """There is no forward-mode derivative; a tangent on any tensor raises instead of being lost."""
    import torch.autograd.forward_ad as fw
    from ravel_lm_b200.dense import fused_linear
    from ravel_lm_b200.distill import distill_topk_loss
    from ravel_lm_b200.glue import layer_norm
    x, w, b = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.bfloat16)
    r, g, ids, t = torch.zeros(2, 4, dtype=torch.bfloat16), torch.ones(8, dtype=torch.bfloat16), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    with fw.dual_level():
        def dual(v):
            return fw.make_dual(v, torch.ones_like(v))
        calls = [lambda: fused_linear(dual(x), w), lambda: fused_linear(x, dual(w)), lambda: fused_linear(x, w, dual(b)),
                 lambda: fused_linear(x, w, b, activation="silu", residual=dual(r)), lambda: layer_norm(dual(x)),
                 lambda: layer_norm(x, dual(g)), lambda: layer_norm(x, g, dual(g)), lambda: distill_topk_loss(dual(x), ids, t),
                 lambda: distill_topk_loss(x, ids, dual(t))]
        for call in calls:
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call()
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        fused_linear(x, w)


def test_the_launch_shapes_are_all_tested(lib):
    """The sizes of the GPU tests reach every launch shape in every direction (on 148 SMs, which a machine without a
    GPU is taken to have), and every number of warps per row."""
    from dense_shapes import CASES, ONE32, ONE64, ONE128, PAIR128, PAIR256, ROWS, SPLIT2, SPLIT4, plan, plans
    every = {PAIR256, PAIR128, ONE128, ONE64, SPLIT2, SPLIT4}
    got = [plans(lib, *sizes) for sizes, *_ in CASES]
    assert got == [tuple(case[1:]) for case in CASES]
    assert {p[0] for p in got} == every | {ONE32}
    assert {p[1] for p in got} == {p[2] for p in got} == every
    assert [plan(lib, 1, N, K, 0) for K, N, _ in ROWS] == [(0, warps, 1) for *_, warps in ROWS]
    assert {warps for *_, warps in ROWS} == {1, 2, 4, 8}
    out = (ctypes.c_int * 3)()
    assert lib.ravel_matmul_plan(0, 8, 8, 0, out) == INVALID
    assert lib.ravel_matmul_plan(8, 8, 8, 0, None) == INVALID
