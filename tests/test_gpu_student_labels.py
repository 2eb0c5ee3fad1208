"""The example trained on next tokens: token_embedding, the event memory and the dense operators, linear_cross_entropy on
the tied head, AdamW.  One step's loss and gradients against the same model in float64 torch operations, and
the step itself against the formula; it runs with 32-bit and 8-bit states."""
from __future__ import annotations

import importlib.util
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def example():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    spec = importlib.util.spec_from_file_location("distill_student", ROOT / "examples" / "distill_student.py")
    mod = importlib.util.module_from_spec(spec)
    sys.modules["distill_student"] = mod
    spec.loader.exec_module(mod)
    import ravel_lm_b200._lib as L
    yield mod
    torch.cuda.synchronize()
    assert L.device_error(torch.cuda.current_stream().cuda_stream) == 0


def _reference(student, tokens, targets):
    """The mean cross entropy in float64 with elementary operations on the same weights."""
    from ravel_lm_b200 import memory_lookups
    P = {n: p.detach().double().requires_grad_(True) for n, p in student.named_parameters()}

    def norm(x, w, b):
        xc = x - x.mean(-1, keepdim=True)
        return xc / torch.sqrt((xc * xc).mean(-1, keepdim=True) + 1e-5) * w + b
    x = P["embed"][tokens]
    B, L, _ = x.shape
    for i, blk in enumerate(student.blocks):
        q = {k: P[f"blocks.{i}.{k}"] for k in ("n1w", "n1b", "n2w", "n2b", "inw", "inb", "outw", "upw", "upb", "downw")}
        pay = norm(x, q["n1w"], q["n1b"]) @ q["inw"].t() + q["inb"]
        vals, _, _, _ = memory_lookups(tokens, pay.view(B, L, blk.heads, blk.payload), address_space=blk.space,
                                       n_literal_heads=blk.heads, bos_token_id=0)
        x = x + vals.reshape(B, L, -1) @ q["outw"].t()
        h = norm(x, q["n2w"], q["n2b"]) @ q["upw"].t() + q["upb"]
        x = x + (h * torch.sigmoid(h)) @ q["downw"].t()
    s = norm(x, P["nw"], P["nb"]) @ P["embed"].t()
    lp = torch.log_softmax(s, -1)
    live = targets >= 0
    loss = -(lp.gather(-1, targets.clamp_min(0)[..., None])[..., 0] * live).sum() / live.sum()
    return loss, dict(zip(P, torch.autograd.grad(loss, list(P.values()))))


def test_one_step_against_float64(example):
    from ravel_lm_b200.optim import AdamW
    torch.manual_seed(3)
    student = example.Student(vocab=515, d=128, layers=2, heads=4, payload=32, space=256).cuda()
    tokens = torch.randint(1, 515, (4, 101), device="cuda")
    targets = tokens[:, 1:].clone()
    targets[1, 60:] = -100  # a padded sequence
    loss = student.loss(tokens[:, :-1], targets)
    loss.backward()
    l64, g64 = _reference(student, tokens[:, :-1], targets)
    # about 20 roundings to bfloat16 (2^-9 rms each, random signs) lie between the embedding and a gradient:
    # 2^-9 sqrt(20) = 0.9%, and three times that
    for name, a, b in [("loss", loss, l64), *((n, p.grad, g64[n]) for n, p in student.named_parameters())]:
        rel = float((a.detach().double() - b.detach()).norm() / b.detach().norm())
        assert rel < 0.027, f"{name}: {rel}"
    # the step: the first moves every parameter by lr sign(g) (1 - eps / |g|), from masters equal to the parameters
    before = {n: p.detach().double() for n, p in student.named_parameters()}
    AdamW(student.parameters(), lr=1e-3, weight_decay=0.1).step()
    for n, p in student.named_parameters():
        g = p.grad.double()
        want = before[n] * (1 - 1e-4) - 1e-3 * g / (g.abs() + 1e-8)
        # a float32 step and one rounding
        assert bool(((p.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-8).all()), n


@pytest.mark.parametrize("state_bits", [32, 8])
@pytest.mark.parametrize("labels", [True, False])
def test_it_trains_and_decodes(example, labels, state_bits):
    student, losses = example.train(steps=5, batch=3, length=40, labels=labels, state_bits=state_bits)
    assert len(losses) == 5 and all(map(torch.isfinite, map(torch.tensor, losses)))
    assert all(torch.isfinite(p).all() for p in student.parameters())
    tokens = torch.randint(1, student.embed.shape[0], (2, 5), device="cuda")
    caches = student.caches(2)
    for t in range(5):
        logits = student.decode(tokens[:, max(0, t - 2):t + 1], caches)
    assert logits.shape == (2, student.embed.shape[0]) and torch.isfinite(logits).all()
