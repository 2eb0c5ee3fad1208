"""CPU-only checks of the vocabulary operators' and the optimizer step's boundary: C-ABI refusals before any launch,
workspace sizes, and the Python functions' refusals (no CPU path)."""
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


def test_embedding_refuses_on_the_host(lib):
    def fwd(ids=P, it=1, w=P, ldw=8, N=4, V=9, K=8, y=P, dt=0):
        return lib.ravel_embedding_fwd(ids, it, w, ldw, N, V, K, 1.0, y, dt, None)
    assert fwd(N=-1) == INVALID and fwd(V=0) == INVALID and fwd(it=7) == INVALID
    assert fwd(dt=3) == UNSUPPORTED and fwd(N=(1 << 30) + 1) == UNSUPPORTED
    assert fwd(ids=None) == INVALID and fwd(w=None) == INVALID and fwd(y=None) == INVALID and fwd(ldw=7) == INVALID
    assert fwd(N=0, ids=None, y=None) == 0 and fwd(K=0) == 0

    def bwd(g=P, ldg=8, N=10000, V=9, K=8, dw=P, dt=0, scratch=P, sb=None):
        sb = lib.ravel_embedding_scratch_bytes(N, V, K) if sb is None else sb
        return lib.ravel_embedding_bwd(P, 1, g, ldg, N, V, K, 1.0, -1, dw, dt, scratch, sb, None)
    assert bwd(dw=None) == INVALID and bwd(g=None) == INVALID and bwd(ldg=7) == INVALID
    assert bwd(scratch=None) == WORKSPACE and bwd(sb=100) == WORKSPACE and bwd(scratch=P + 8) == WORKSPACE
    assert lib.ravel_embedding_scratch_bytes(-1, 9, 8) == 0
    # a few ids take one launch without scratch, unless the vocabulary has too many rows for its blocks
    assert lib.ravel_embedding_scratch_bytes(512, 65536, 8) == 0 and lib.ravel_embedding_scratch_bytes(513, 65536, 8) > 0
    assert lib.ravel_embedding_scratch_bytes(512, 1 << 24, 8) > 0
    assert lib.ravel_embedding_scratch_bytes(1 << 20, 1 << 17, 1024) > (1 << 17) + 16 * (1 << 20)
    # the pieces of sums are a part of the gradients read, not more
    assert lib.ravel_embedding_scratch_bytes(1 << 20, 1 << 17, 1024) < (1 << 20) * 1024 * 2 // 8


def test_cross_entropy_refuses_on_the_host(lib):
    def fwd(x=P, ldx=64, w=P, ldw=64, t=P, tt=1, M=8, K=64, V=100, red=2, losses=P, out=P, factor=P, sx=P, sw=P, dt=1,
            scratch=P, sb=1 << 40, work=P, wb=1 << 40):
        return lib.ravel_linear_ce_fwd(x, ldx, w, ldw, t, tt, M, K, V, -100, red, 0, losses, out, factor, sx, sw, dt,
                                       scratch, sb, work, wb, None)
    assert fwd(M=-1) == INVALID and fwd(K=0) == INVALID and fwd(V=0) == INVALID and fwd(tt=5) == INVALID
    assert fwd(dt=0) == UNSUPPORTED and fwd(V=1 << 30) == UNSUPPORTED
    assert fwd(x=None) == INVALID and fwd(w=None) == INVALID and fwd(t=None) == INVALID and fwd(losses=None) == INVALID
    assert fwd(ldx=63) == INVALID and fwd(ldw=63) == INVALID and fwd(ldw=68) == INVALID and fwd(w=P + 2) == INVALID
    assert fwd(red=3) == INVALID and fwd(out=None) == INVALID and fwd(factor=None) == INVALID
    assert fwd(red=0) == INVALID                     # single losses have no gradient for an upstream gradient of 1
    assert fwd(sw=P + 4) == INVALID
    assert fwd(scratch=None) == WORKSPACE and fwd(sb=64) == WORKSPACE and fwd(wb=64) == WORKSPACE
    sizes = (ctypes.c_int64 * 3)()
    assert lib.ravel_linear_ce_slabs(8, 64, 100, sizes) == 0 and sizes[0] >= 1 and sizes[1] >= 1 and sizes[2] == 64
    assert lib.ravel_linear_ce_slabs(8, 65, 100, sizes) == 0 and sizes[2] == 68
    assert lib.ravel_linear_ce_slabs(8, 0, 100, sizes) == INVALID
    # never the logits of every row: at most 512 MB of them, or of 1024 rows
    for M, V in ((1 << 20, 50000), (1 << 17, 1 << 18)):
        per_row = 2 * V + 4 * (V // 32 + 1) * 2
        assert lib.ravel_linear_ce_work_bytes(M, 64, V, 1, 2) <= max((512 << 20), 1024 * per_row) * 1.2
    assert lib.ravel_linear_ce_scratch_bytes(8, 0, 100) == 0
    # a tile of 128 or 256 columns writes four parts (a maximum and a sum) a row, whatever the vocabulary leaves of it
    for M in (1, 100, 128, 129, 5000):
        for V in (1, 6, 96, 97, 128, 129, 224, 256, 257, 300, 32003):
            parts = 4 * -(-V // 128) if M <= 128 else 4 * -(-V // 256)
            for dt in (1, 2):
                assert lib.ravel_linear_ce_work_bytes(M, 64, V, 0, dt) >= parts * M * 8, (M, V)
                assert lib.ravel_linear_ce_work_bytes(M, 64, V, 1, dt) >= max(parts * M * 8, M * V * 2), (M, V)

    def grad(w=P, ldw=64, up=P, M=8, K=64, V=100, factor=P, sx=P, sw=P, dt=1, scratch=P, sb=1 << 40, work=P, wb=1 << 40):
        return lib.ravel_linear_ce_grad(w, ldw, up, M, K, V, factor, sx, sw, dt, scratch, sb, work, wb, None)
    assert grad(up=None) == INVALID and grad(factor=None) == INVALID and grad(w=None) == INVALID
    assert grad(wb=10) == WORKSPACE and grad(dt=3) == UNSUPPORTED

    def bwd(sx=P, sw=P, up=P, factor=P, gx=P, gw=P, dt=1):
        return lib.ravel_linear_ce_bwd(sx, sw, up, factor, 8, 64, 100, gx, gw, dt, None)
    assert bwd(sx=None) == INVALID and bwd(sw=None) == INVALID and bwd(factor=None) == INVALID
    assert bwd(sx=None, sw=None, gx=None, gw=None) == 0


def test_adamw_refuses_on_the_host(lib):
    import ravel_lm_b200._lib as L

    def tensors(**k):
        t = dict(param=P, grad=P, master=None, exp_avg=P, exp_avg_sq=P, exp_avg_exponents=None, exp_avg_sq_exponents=None,
                 n=5)
        t.update(k)
        return (L.AdamTensor * 1)(L.AdamTensor(**t))

    def go(t=None, count=1, dt=0, bits=32, st=P, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, mx=0.0, norm=None, scratch=P, sb=1 << 30):
        return lib.ravel_adamw(t or tensors(), count, dt, bits, st, lr, None, b1, b2, eps, 0.0, mx, norm, None, scratch, sb,
                               None)
    assert go(count=-1) == INVALID and go(dt=3) == UNSUPPORTED and go(bits=16) == UNSUPPORTED
    assert go(st=None) == INVALID and go(b1=1.0) == INVALID and go(b2=-0.1) == INVALID and go(eps=-1.0) == INVALID
    assert go(mx=-1.0) == INVALID and go(norm=P) == INVALID
    assert go(tensors(n=-1)) == INVALID and go(tensors(grad=None)) == INVALID and go(tensors(param=None)) == INVALID
    assert go(tensors(exp_avg=None)) == INVALID
    assert go(dt=1) == INVALID                                     # a 16-bit parameter without a master
    assert go(bits=8) == INVALID                                   # 8-bit states without exponents
    assert go(scratch=None) == WORKSPACE and go(sb=8) == WORKSPACE and go(mx=1.0, sb=64) == WORKSPACE
    assert go(scratch=P + 4) == WORKSPACE
    t = tensors()
    assert lib.ravel_grad_norm(t, 1, 0, None, P, 1 << 30, None) == INVALID
    assert lib.ravel_grad_norm(t, 1, 0, P, P, 8, None) == WORKSPACE
    assert lib.ravel_adamw_scratch_bytes(t, 1, 1.0) >= 64 + lib.ravel_grad_norm_scratch_bytes(t, 1)
    assert lib.ravel_state_values(P, P, -1, 1, P, 0, None) == INVALID
    assert lib.ravel_state_values(P, P, 4, 1, P, 2, None) == UNSUPPORTED
    assert lib.ravel_state_values(None, None, 0, 1, None, 0, None) == 0


def test_vocab_functions_refuse():
    from ravel_lm_b200.vocab import linear_cross_entropy, token_embedding
    ids, w = torch.zeros(3, dtype=torch.long), torch.zeros(5, 8)
    with pytest.raises(ValueError, match=r"weight \[V, K\]"):
        token_embedding(ids, w[0])
    with pytest.raises(ValueError, match=r"weight \[V, K\]"):
        token_embedding(ids, w[:0])
    with pytest.raises(TypeError, match="int32 or int64"):
        token_embedding(ids.float(), w)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        token_embedding(ids, w.double())
    with pytest.raises(ValueError, match="padding_idx"):
        token_embedding(ids, w, padding_idx=5)
    with pytest.raises(ValueError, match="finite"):
        token_embedding(ids, w, scale=float("inf"))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        token_embedding(ids, w)
    x, h = torch.zeros(3, 8).bfloat16(), w.bfloat16()
    with pytest.raises(ValueError, match="reduction must be"):
        linear_cross_entropy(x, h, ids, reduction="max")
    with pytest.raises(ValueError, match=r"x \[..., K\]"):
        linear_cross_entropy(x, h[:, :4], ids)
    with pytest.raises(ValueError, match="leading dimensions"):
        linear_cross_entropy(x, h, ids[:2])
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        linear_cross_entropy(x.float(), w, ids)
    with pytest.raises(TypeError, match="one dtype"):
        linear_cross_entropy(x, h.half(), ids)
    with pytest.raises(TypeError, match="int32 or int64"):
        linear_cross_entropy(x, h, ids.bool())
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        linear_cross_entropy(x, h, ids)


def test_optimizer_functions_refuse():
    from ravel_lm_b200.optim import AdamW, adamw_step, global_norm, state_values
    p, g, m, v = ([torch.zeros(300)] for _ in range(4))
    step = torch.zeros(1, dtype=torch.long)

    def go(p=p, g=g, m=m, v=v, step=step, **k):
        return adamw_step(p, g, m, v, step, **{"lr": 1e-3, **k})
    with pytest.raises(ValueError, match="at least one"):
        go([], [], [], [])
    with pytest.raises(ValueError, match="one length"):
        go(g=g * 2)
    with pytest.raises(ValueError, match="masters"):
        go(masters=p)
    with pytest.raises(ValueError, match="masters"):
        go([p[0].half()], [g[0].half()])
    with pytest.raises(ValueError, match="come together"):
        go(exp_avg_exponents=m)
    with pytest.raises(ValueError, match="wrong number"):
        go(m=[torch.zeros(299)])
    with pytest.raises(TypeError, match=r"exp_avgs\[0\] must be Byte"):
        e = [torch.zeros(2, dtype=torch.int8)]
        go(exp_avg_exponents=e, exp_avg_sq_exponents=e)
    with pytest.raises(ValueError, match="contiguous"):
        go([torch.zeros(20, 15).t()], [torch.zeros(15, 20)], [torch.zeros(15, 20)], [torch.zeros(15, 20)])
    with pytest.raises(ValueError, match="parameter's shape"):
        go(g=[torch.zeros(3, 100)])
    with pytest.raises(TypeError, match="parameter's dtype"):
        go(g=[g[0].half()])
    with pytest.raises(TypeError, match="one int64"):
        go(step=step.int())
    with pytest.raises(TypeError, match="float32"):
        go(lr=torch.zeros(1, dtype=torch.float64))
    with pytest.raises(ValueError, match="betas"):
        go(betas=(1.0, 0.9))
    with pytest.raises(ValueError, match="negative"):
        go(lr=-1.0)
    with pytest.raises(ValueError, match="max_norm"):
        go(max_norm=0.0)
    with pytest.raises(ValueError, match="with max_norm only"):
        go(norm=torch.zeros((), dtype=torch.float64))
    with pytest.raises(ValueError, match="twice"):
        go(p * 2, g * 2, m * 2, v * 2)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        go()
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        global_norm(g)
    with pytest.raises(ValueError, match="at least one"):
        global_norm([])
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        state_values(torch.zeros(4, dtype=torch.uint8), torch.zeros(1, dtype=torch.int8), signed=True, dtype=torch.float16)
    with pytest.raises(ValueError, match="one exponent per block"):
        state_values(torch.zeros(4, dtype=torch.uint8), torch.zeros(2, dtype=torch.int8), signed=True)
    for k in (dict(lr=-1.0), dict(eps=-1.0), dict(weight_decay=-1.0), dict(betas=(0.9, 1.0)), dict(state_bits=16),
              dict(max_norm=-1.0)):
        with pytest.raises(ValueError):
            AdamW([torch.nn.Parameter(torch.zeros(3))], **k)


def test_the_option_for_positive_second_moments(lib):
    import ravel_lm_b200._lib as L
    t = (L.AdamTensor * 1)(L.AdamTensor(param=P, grad=P, exp_avg=P, exp_avg_sq=P, n=5))

    def go(bits):
        return lib.ravel_adamw(t, 1, 0, bits, P, 1e-3, None, 0.9, 0.99, 1e-8, 0.0, 0.0, None, None, P, 1 << 30, None)
    assert go(8 | L.RAVEL_STATE_POSITIVE) == INVALID == go(8)  # 8-bit states: exponents are missing
    assert go(32 | L.RAVEL_STATE_POSITIVE) == UNSUPPORTED and go(16 | L.RAVEL_STATE_POSITIVE) == UNSUPPORTED
    from ravel_lm_b200.optim import adamw_step
    z = [torch.zeros(3)]
    with pytest.raises(ValueError, match="8-bit states only"):
        adamw_step(z, z, z, z, torch.zeros(1, dtype=torch.long), lr=1e-3, positive_exp_avg_sq=True)


def _stepped(bits):
    """An optimizer of two CPU parameters with states as after a step (no kernel runs here)."""
    from ravel_lm_b200.optim import AdamW
    ps = [torch.nn.Parameter(torch.full((300,), float(i))) for i in range(2)]
    o = AdamW(ps, lr=1e-2, state_bits=bits)
    step = torch.ones(1, dtype=torch.int64)
    for p in ps:
        p.grad = torch.ones_like(p)
        o.state[p] = o._new_state(p, step)
    return ps, o


def test_a_capture_makes_no_states_and_copies_no_count(monkeypatch):
    ps, o = _stepped(32)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    group = o.param_groups[0]
    assert o._buckets(group) == [ps]  # every state is there
    step = o.state[ps[1]]["step"]
    ps[0].grad = None
    with pytest.raises(RuntimeError, match="before a capture"):
        o._buckets(group)
    assert o.state[ps[1]]["step"] is step
    ps[0].grad = torch.ones(300)
    del o.state[ps[0]]
    with pytest.raises(RuntimeError, match="before a capture"):
        o._buckets(group)
    assert ps[0] not in o.state
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    assert o._buckets(group) == [[ps[0]], [ps[1]]]


@pytest.mark.parametrize("bits", [32, 8])
def test_a_refused_state_dict_changes_nothing(bits):
    _, src = _stepped(40 - bits)
    src.param_groups[0]["lr"] = 0.5
    ps, o = _stepped(bits)
    kept = {p: dict(o.state[p]) for p in ps}
    with pytest.raises(ValueError, match="state_bits"):
        o.load_state_dict(src.state_dict())
    assert o.param_groups[0]["lr"] == 1e-2 and all(a is b for a, b in zip(o.param_groups[0]["params"], ps))
    assert set(o.state) == set(ps)
    for p in ps:
        assert o.state[p].keys() == kept[p].keys() and all(o.state[p][k] is v for k, v in kept[p].items())


def test_states_of_another_optimizer_or_dtype_are_refused():
    ps, o = _stepped(32)
    for p in ps:
        assert set(o.state[p]) == o._state_names(p)
    other = torch.optim.AdamW([torch.nn.Parameter(torch.zeros(300)) for _ in range(2)], lr=0.5)
    for p in other.param_groups[0]["params"]:
        p.grad = torch.ones_like(p)
    other.step()
    with pytest.raises(ValueError, match="not this optimizer's"):
        o.load_state_dict(other.state_dict())
    from ravel_lm_b200.optim import AdamW
    half = AdamW([torch.nn.Parameter(torch.zeros(300).bfloat16()) for _ in range(2)], lr=1e-2)
    p = half.param_groups[0]["params"][0]
    assert set(half._new_state(p, torch.ones(1, dtype=torch.int64))) == half._state_names(p)
    with pytest.raises(ValueError, match="parameter of torch.bfloat16"):  # there is no master
        half.load_state_dict(o.state_dict())
    assert o.param_groups[0]["lr"] == 1e-2 and not half.state
    fresh = AdamW([torch.nn.Parameter(torch.zeros(300)) for _ in range(2)], lr=0.1)
    fresh.load_state_dict(o.state_dict())
    a, b = (fresh.state[q] for q in fresh.param_groups[0]["params"])
    assert a["step"] is b["step"] and int(a["step"]) == 1 and fresh.param_groups[0]["lr"] == 1e-2


def test_a_users_own_entries_in_the_states_are_loaded():
    ps, o = _stepped(32)
    o.state[ps[0]]["mine"] = torch.ones(2)
    d = o.state_dict()
    o.load_state_dict(d)
    assert torch.equal(o.state[ps[0]]["mine"], torch.ones(2)) and "mine" not in o.state[ps[1]]


def test_a_short_last_piece_does_not_choose_the_launch_shape(lib):
    """Rows go in pieces; d weight's shape is the full pieces', and only its parts have to fit the last one's rows."""
    def plan(M, K, V):
        p = (ctypes.c_int * 6)()
        assert lib.ravel_linear_ce_plan(M, K, V, p) == 0
        sizes = (ctypes.c_int64 * 3)()
        assert lib.ravel_linear_ce_slabs(M, K, V, sizes) == 0 and [p[2], p[5]] == list(sizes[:2])
        return list(p)
    for M, K, V in ((16384, 512, 131072), (16384, 1024, 131072), (4096, 64, 262144), (4096, 2048, 262144)):
        even = plan(M, K, V)
        for rest in (1, 100, 193):
            assert plan(M + rest, K, V)[:5] == even[:5], (M, K, V, rest)
        assert plan(M + 1, K, V)[5] == 1  # one row: a single part
    for M in (1, 24, 128, 192):  # few rows: tiles by the estimate, in one part (a part has 4 chunks of 64 at least)
        for K, V in ((2048, 32000), (64, 300)):
            assert plan(M, K, V)[5] == 1
    p = (ctypes.c_int * 6)()
    assert lib.ravel_linear_ce_plan(0, 8, 8, p) == INVALID and lib.ravel_linear_ce_plan(8, 8, 8, None) == INVALID
    assert lib.ravel_linear_ce_plan(8, 0, 8, p) == INVALID


def test_unaligned_gradient_sums_are_refused(lib):
    """The outputs' kernel reads slabs 16 bytes at a time."""
    def bwd(sx=P, sw=P):
        return lib.ravel_linear_ce_bwd(sx, sw, P, P, 8, 64, 100, P, P, 1, None)
    assert bwd(sx=P + 4) == INVALID and bwd(sw=P + 8) == INVALID


def test_a_scale_past_float32_is_refused():
    from ravel_lm_b200.vocab import token_embedding
    ids, w = torch.zeros(3, dtype=torch.long), torch.zeros(5, 8)
    for scale in (1e39, -1e300):
        with pytest.raises(ValueError, match="finite"):  # it would be an infinity to the kernel
            token_embedding(ids, w, scale=scale)


@pytest.mark.parametrize("bits", [32, 8])
def test_the_optimizer_refuses_cpu_parameters_without_a_gpu_too(bits):
    from ravel_lm_b200.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        AdamW([p], state_bits=bits).step()
