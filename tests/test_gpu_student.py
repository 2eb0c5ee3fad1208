"""The example that runs the dense operators together around the event memory: a student
distilled from a teacher's top logits learns, one step's gradients agree with the same model
in float64 torch operations, and decoding token by token gives the full forward's logits."""
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


def test_the_student_learns(example):
    student, losses = example.train(steps=60, batch=8, length=128)
    assert all(torch.isfinite(p).all() for p in student.parameters())
    assert sum(losses[-5:]) < 0.7 * sum(losses[:5]), (losses[:5], losses[-5:])


def _reference(student, tokens, ids, logits, T):
    """The student's loss in float64 with elementary operations on the same weights."""
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
    logq = torch.log_softmax(s / T, -1)
    logp = torch.log_softmax(logits.double() / T, -1)
    loss = T * T * (logp.exp() * (logp - logq.gather(-1, ids))).sum(-1).mean()
    return s, loss, dict(zip(P, torch.autograd.grad(loss, list(P.values()))))


def test_one_step_against_float64(example):
    torch.manual_seed(3)
    student = example.Student(vocab=515, d=128, layers=2, heads=4, payload=32, space=256).cuda()
    ids, logits = example.teacher(515, 12)
    tokens = torch.randint(1, 515, (4, 100), device="cuda")
    out = student(tokens)
    loss = example.distill_topk_loss(out, ids[tokens], logits[tokens], temperature=2.0)
    grads = dict(zip([n for n, _ in student.named_parameters()],
                     torch.autograd.grad(loss, list(student.parameters()))))
    s64, loss64, g64 = _reference(student, tokens, ids[tokens], logits[tokens], 2.0)
    # about 20 roundings to bfloat16 (2^-9 rms each, random signs) lie between the embedding and a gradient:
    # 2^-9 sqrt(20) = 0.9%, and three times that
    for name, a, b in [("logits", out, s64), ("loss", loss, loss64), *((n, grads[n], g64[n]) for n in g64)]:
        rel = float((a.detach().double() - b.detach()).norm() / b.detach().norm())
        assert rel < 0.027, f"{name}: {rel}"


def test_decoding_gives_the_forward_pass(example):
    torch.manual_seed(4)
    student = example.Student(vocab=300, d=64, layers=2, heads=3, payload=16, space=128).cuda()
    tokens = torch.randint(1, 300, (3, 24), device="cuda")
    with torch.no_grad():
        full = student(tokens)
    caches = student.caches(3)
    steps = torch.stack([student.decode(tokens[:, max(0, t - 2):t + 1], caches) for t in range(24)], 1)
    # the same products in another order: a last bit of a bfloat16 intermediate may differ here and there
    rel = float((steps.double() - full.double()).norm() / full.double().norm())
    assert rel < 0.01, rel
