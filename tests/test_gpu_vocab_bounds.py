"""The vocabulary operators and the optimizer step write nothing outside the buffers they are given: each output and
workspace lies at its exact size between guard bytes, which have to be as they were."""
from __future__ import annotations

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

GUARD = 8192
MARK = 0xA5


@pytest.fixture(scope="module")
def lib():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import ravel_lm_b200._lib as L
    yield L.load()
    torch.cuda.synchronize()
    assert L.device_error(torch.cuda.current_stream().cuda_stream) == 0


class Guarded:
    def __init__(self):
        self.all = []

    def __call__(self, nbytes, fill=MARK):
        t = torch.full((nbytes + 2 * GUARD,), MARK, dtype=torch.uint8, device="cuda")
        if fill != MARK:
            t[GUARD:GUARD + nbytes] = fill
        self.all.append((t, nbytes))
        return t.data_ptr() + GUARD

    def tensor(self, src):
        """A copy of ``src`` between guards: its pointer, and the tensor."""
        n = src.numel() * src.element_size()
        p = self(n)
        v = self.all[-1][0][GUARD:GUARD + n].view(src.dtype).view(src.shape)
        v.copy_(src)
        return p, v

    def check(self, what):
        torch.cuda.synchronize()
        for i, (t, n) in enumerate(self.all):
            assert bool((t[:GUARD] == MARK).all()) and bool((t[GUARD + n:] == MARK).all()), (what, i)


@pytest.mark.parametrize("dt,code", [(torch.float32, 0), (torch.bfloat16, 1), (torch.float16, 2)])
def test_embedding(lib, dt, code):
    gen = torch.Generator(device="cuda").manual_seed(0)
    es = torch.tensor([], dtype=dt).element_size()
    for N, V, K in ((1, 1, 1), (7, 3, 5), (100, 17, 8), (129, 1025, 33), (1025, 40, 24), (3000, 70000, 12), (5000, 9, 260)):
        for bad in (False, True):
            g = Guarded()
            ids = torch.randint(0, V, (N,), generator=gen, device="cuda")
            pi, _ = g.tensor(ids)
            pw, _ = g.tensor(torch.randn(V, K, generator=gen, device="cuda").to(dt))
            pg, _ = g.tensor(torch.randn(N, K, generator=gen, device="cuda").to(dt))
            y, dw = g(N * K * es), g(V * K * es)
            sb = lib.ravel_embedding_scratch_bytes(N, V, K)
            scratch = g(sb, 0xFF if bad else 0)  # whatever a workspace held before
            assert lib.ravel_embedding_fwd(pi, 1, pw, K, N, V, K, 1.0, y, code, None) == 0
            assert lib.ravel_embedding_bwd(pi, 1, pg, K, N, V, K, 1.0, -1, dw, code, scratch, sb, None) == 0
            g.check((N, V, K))


CE_SIZES = [(1, 8, 1), (3, 16, 6), (100, 24, 96), (128, 40, 300), (129, 8, 129), (257, 33, 97), (1000, 72, 224), (40, 264, 1000),
            (300, 8, 20000), (2000, 16, 33)]


@pytest.mark.parametrize("code", [1, 2])
@pytest.mark.parametrize("M,K,V", CE_SIZES + [(1500, 1000, 24003)])
def test_cross_entropy(lib, code, M, K, V):
    dt = torch.bfloat16 if code == 1 else torch.float16
    gen = torch.Generator(device="cuda").manual_seed(M + V)
    ld = (K + 7) // 8 * 8
    for reduction, grads in ((2, True), (2, False), (0, True)):
        g = Guarded()
        px, _ = g.tensor(torch.randn(M, K, generator=gen, device="cuda").to(dt))
        pw, _ = g.tensor((torch.randn(V, ld, generator=gen, device="cuda") * K ** -0.5).to(dt))
        t = torch.randint(0, V, (M,), generator=gen, device="cuda")
        t[::5] = -100
        pt, _ = g.tensor(t)
        sizes = (ctypes.c_int64 * 3)()
        assert lib.ravel_linear_ce_slabs(M, K, V, sizes) == 0
        losses, out, factor = g(4 * M), g(4), g(4)
        sx = g(sizes[0] * M * sizes[2] * 4) if grads else None
        sw = g(sizes[1] * V * sizes[2] * 4) if grads else None
        sb = lib.ravel_linear_ce_scratch_bytes(M, K, V)
        wb = lib.ravel_linear_ce_work_bytes(M, K, V, int(grads and reduction == 2), code)
        scratch, work = g(sb, 0xFF), g(wb, 0xFF)
        first = (sx, sw) if reduction == 2 else (None, None)
        assert lib.ravel_linear_ce_fwd(px, K, pw, ld, pt, 1, M, K, V, -100, reduction, int(reduction == 0), losses,
                                       out if reduction else None, factor if grads else None, *first, code, scratch, sb,
                                       work, wb, None) == 0
        g.check(("fwd", reduction, grads))
        if not grads:
            continue
        up = None
        if reduction == 0:
            pu, _ = g.tensor(torch.randn(M, generator=gen, device="cuda"))
            wb2 = lib.ravel_linear_ce_work_bytes(M, K, V, 1, code)
            work2 = g(wb2, 0xFF)
            assert lib.ravel_linear_ce_grad(pw, ld, pu, M, K, V, factor, sx, sw, code, scratch, sb, work2, wb2, None) == 0
            g.check("grad")
        else:
            up, _ = g.tensor(torch.ones(1, device="cuda"))
        dx, dw = g(M * K * 2), g(V * K * 2)
        assert lib.ravel_linear_ce_bwd(sx, sw, up, factor, M, K, V, dx, dw, code, None) == 0
        g.check("bwd")
        n = M * K * 2
        got = next(b[GUARD:GUARD + n] for b, m in g.all if b.data_ptr() + GUARD == dx).view(dt)
        assert bool(torch.isfinite(got).all())  # no leftovers of a workspace


@pytest.mark.parametrize("code,dt", [(0, torch.float32), (1, torch.bfloat16)])
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw(lib, code, dt, bits):
    import ravel_lm_b200._lib as L
    for sizes in ([1], [255, 257], [2048, 7, 4097], [33] * 60):
        for off in (0, 1):
            g = Guarded()
            arr = (L.AdamTensor * len(sizes))()
            for a, n in zip(arr, sizes):
                def buf(kind, count=n, fill=0):
                    es = torch.tensor([], dtype=kind).element_size()
                    return g(count * es, fill) if not off else g.tensor(torch.zeros(count + 1, dtype=kind))[0] + es
                a.param, a.grad = buf(dt), buf(dt)
                a.master = buf(torch.float32) if code else None
                state = torch.float32 if bits == 32 else torch.uint8
                a.exp_avg, a.exp_avg_sq = buf(state), buf(state)
                if bits == 8:
                    a.exp_avg_exponents, a.exp_avg_sq_exponents = g((n + 255) // 256, 0), g((n + 255) // 256, 0)
                a.n = n
            step, norm = g(8, 0), g(4, 0)
            sb = lib.ravel_adamw_scratch_bytes(arr, len(sizes), 1.0)
            scratch = g(sb, 0xFF)
            for _ in range(2):
                assert lib.ravel_adamw(arr, len(sizes), code, bits, step, 1e-3, None, 0.9, 0.99, 1e-8, 0.0, 1.0, None, norm,
                                       scratch, sb, None) == 0
            g.check((sizes, off))


def ce_slabs(lib, g, M, K, V, dt, code, seed):
    """A mean loss's gradient sums by ``ravel_linear_ce_fwd``: slabs of d x and of d W, an upstream gradient of 1, the factor."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    px, _ = g.tensor(torch.randn(M, K, generator=gen, device="cuda").to(dt))
    ld = (K + 7) // 8 * 8
    pw, _ = g.tensor((torch.randn(V, ld, generator=gen, device="cuda") * K ** -0.5).to(dt))
    pt, _ = g.tensor(torch.randint(0, V, (M,), generator=gen, device="cuda"))
    up, _ = g.tensor(torch.ones(1, device="cuda"))
    sizes = (ctypes.c_int64 * 3)()
    assert lib.ravel_linear_ce_slabs(M, K, V, sizes) == 0
    sx, sw = g(sizes[0] * M * sizes[2] * 4), g(sizes[1] * V * sizes[2] * 4)
    losses, out, factor = g(4 * M), g(4), g(4)
    sb, wb = lib.ravel_linear_ce_scratch_bytes(M, K, V), lib.ravel_linear_ce_work_bytes(M, K, V, 1, code)
    assert lib.ravel_linear_ce_fwd(px, K, pw, ld, pt, 1, M, K, V, -100, 2, 0, losses, out, factor, sx, sw, code, g(sb), sb,
                                   g(wb), wb, None) == 0
    return sx, sw, up, factor


@pytest.mark.parametrize("code", [1, 2])
@pytest.mark.parametrize("M,K,V", [(8, 64, 40), (3, 4, 2), (300, 72, 500), (7, 65, 30), (5, 66, 9)])
def test_cross_entropy_gradients_at_any_address(lib, code, M, K, V):
    """Gradients inside a flat buffer: off 16 and off 8 bytes, either or both, they are the aligned ones."""
    dt = torch.bfloat16 if code == 1 else torch.float16
    g = Guarded()
    sx, sw, up, factor = ce_slabs(lib, g, M, K, V, dt, code, seed=M)

    def run(off_x, off_w):
        got = []
        ptrs = []
        for n, off in ((M * K, off_x), (V * K, off_w)):
            ptrs.append(g(2 * (n + off)) + 2 * off)
            got.append(g.all[-1][0])
        assert lib.ravel_linear_ce_bwd(sx, sw, up, factor, M, K, V, *ptrs, code, None) == 0
        g.check((off_x, off_w))
        for t, off in zip(got, (off_x, off_w)):
            assert bool((t[:GUARD + 2 * off] == MARK).all())  # nothing before it either
        return [t[GUARD + 2 * off:-GUARD].view(torch.int16).clone() for t, off in zip(got, (off_x, off_w))]
    want = run(0, 0)
    for off_x, off_w in ((1, 0), (0, 1), (1, 1), (2, 3), (4, 8)):
        got = run(off_x, off_w)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), (off_x, off_w)


@pytest.mark.parametrize("code", [1, 2])
def test_single_losses_of_no_rows_have_a_gradient_of_zero(lib, code):
    """Whatever stood in the workspaces: there is no row, and no upstream gradient."""
    K, V = 16, 50
    g = Guarded()
    gen = torch.Generator(device="cuda").manual_seed(0)
    pw, _ = g.tensor(torch.randn(V, K, generator=gen, device="cuda").to(torch.bfloat16 if code == 1 else torch.float16))
    sizes = (ctypes.c_int64 * 3)()
    assert lib.ravel_linear_ce_slabs(0, K, V, sizes) == 0
    sw = g(sizes[1] * V * sizes[2] * 4, 0xFF)
    sb, wb = lib.ravel_linear_ce_scratch_bytes(0, K, V), lib.ravel_linear_ce_work_bytes(0, K, V, 1, code)
    scratch, work, factor, dw = g(sb, 0xFF), g(wb, 0xFF), g(4, 0xFF), g(V * K * 2, 0xFF)
    assert lib.ravel_linear_ce_fwd(None, K, pw, K, None, 1, 0, K, V, -100, 0, 1, None, None, None, None, None, code, scratch,
                                   sb, work, wb, None) == 0
    assert lib.ravel_linear_ce_grad(pw, K, None, 0, K, V, factor, None, sw, code, scratch, sb, work, wb, None) == 0
    assert lib.ravel_linear_ce_bwd(None, sw, None, factor, 0, K, V, None, dw, code, None) == 0
    g.check("no rows")
    got = next(b[GUARD:GUARD + V * K * 2] for b, _ in g.all if b.data_ptr() + GUARD == dw)
    assert not got.any()
