"""``distill_topk_loss`` on logits at the ends of their type.

The softmax depends on differences only, so the formula is taken in 64 bits of the values less their row's
maximum.  A difference is rounded once and multiplied by the rounded log2(e) / T: an exponent (in base 2) is off by at
most 3 e D, D its own size, and only those above -150 matter; the general tests' bounds then hold with D in
place of the logits' magnitude.
"""
from __future__ import annotations

import pytest
import torch

from test_gpu_distill import DTYPES, E, check, make, reference, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import ravel_lm_b200._lib as L
    L.load()
    yield
    torch.cuda.synchronize()
    assert L.device_error(torch.cuda.current_stream().cuda_stream) == 0


class Shifted:
    """Logits less their row's maximum, as the 64-bit formula takes them."""

    def __init__(self, s):
        x = s.detach().double()
        self.x, self.dtype = x - x.amax(1, keepdim=True), s.dtype

    def detach(self):
        return self.x


def shifted_teacher(ids, t):
    t64 = t.double()
    live = (ids >= 0) & (t64 != -torch.inf)
    top = torch.where(live, t64, torch.full_like(t64, -torch.inf)).amax(1, keepdim=True)
    # 400 below the largest is nothing, in float32 and in the formula
    return torch.where(live, (t64 - top).clamp_min(-400.0), torch.full_like(t64, -torch.inf))


def check_ends(s, ids, t, T):
    """Losses and gradient of every row by reduction="none", then loss and gradient of the mean."""
    from ravel_lm_b200.distill import distill_topk_loss
    want, grad, rows, tl, tg, tiny = reference(Shifted(s), ids, shifted_teacher(ids, t), T)
    losses = distill_topk_loss(s, ids, t, temperature=T, reduction="none")
    got, = torch.autograd.grad(losses, s, torch.ones_like(losses))
    within(losses, want, tl + 1e-30, "losses")
    within(got, grad, tg + tiny, "d logits")
    loss = distill_topk_loss(s, ids, t, temperature=T)
    got, = torch.autograd.grad(loss, s)
    n = max(1, int(rows.sum()))
    within(loss, want.sum() / n, (tl.sum() + (len(want) / 1024 + 64) * E * want.abs().sum()) / n + 1e-30, "loss")
    within(got, grad / n, tg / n + 8 * E * (grad / n).abs() + tiny, "d logits of the mean")


# rows held in registers, read twice, and starting off 16 bytes
@pytest.mark.parametrize("V", [100, 1025, 20001, 65536])
@pytest.mark.parametrize("T", [0.5, 1.0, 2.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_at_the_ends_of_the_type(dtype, T, V):
    """Rows whose logits, or whose live teacher logits, are all the type's lowest value (a padding value) or all its
    highest are uniform; values that differ by the whole range leave the largest alone."""
    lo, hi = torch.finfo(dtype).min, torch.finfo(dtype).max
    s, ids, t = make(12, V, 6, dtype, seed=V, ragged=False)
    with torch.no_grad():
        s[0] = lo
        s[1] = hi
        t[2] = lo
        t[3] = hi
        s[4], t[4] = lo, lo
        ids[4, 3:] = -1
        t[5, 1:] = lo            # one entry has all of the teacher's weight
        s[6, : V // 2] = lo      # a masked half that the teacher does not name
        ids[6] = ids[6] % (V - V // 2) + V // 2
        s[7], t[7, ::2] = lo, float("-inf")
        t[8, 2:], ids[8, 2:] = lo, -1
    check_ends(s, ids, t, T)


@pytest.mark.parametrize("dtype", DTYPES)
def test_an_entry_at_the_lowest_value(dtype):
    """A student's logit of the lowest value that the teacher names makes a large loss, and an infinite one only
    where float32 cannot hold it."""
    s, ids, t = make(6, 500, 4, dtype, seed=3, ragged=False)
    with torch.no_grad():
        ids[2] = torch.arange(4, device="cuda") * 7
        s[2, 7] = torch.finfo(dtype).min
    check_ends(s, ids, t, 1.0)


def test_a_common_offset_does_not_matter():
    """Logits and teacher logits far from zero, float32: 2^20 + multiples of 1/8 are exact."""
    s, ids, t = make(9, 3001, 12, torch.float32, seed=4)
    with torch.no_grad():
        s.copy_((s * 8).round() / 8 + 2.0 ** 20)
        t = (t * 8).round() / 8 - 2.0 ** 20
    check_ends(s, ids, t, 1.0)


# the forward keeps 12 bytes an entry in shared memory, beside what the kernel has of its own: around and at the
# largest k, for blocks of 128, 256 and 512 threads
@pytest.mark.parametrize("R,V,dtype", [(160, 1000, torch.bfloat16), (160, 9001, torch.float16), (3, 20000, torch.float32)])
@pytest.mark.parametrize("k", [4084, 4085, 4090, 4093, 4096])
def test_the_largest_k(R, V, dtype, k):
    s, ids, t = make(R, V, k, dtype, seed=k)
    for reduction in ("mean", "none"):
        check(s, ids, t, 2.0, reduction)
