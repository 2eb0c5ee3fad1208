"""A RAVEL language model trained on a teacher's top logits, and decoded token by token.

Every dense piece around the event memory runs on this package's kernels:

    layer_norm -> fused_linear (packed input projection, bias)
               -> memory_lookups (literal addresses of the token ids, latest value)
               -> fused_linear (read-out, residual)
    layer_norm -> fused_linear (feed-forward, SiLU) -> fused_linear (residual)
    layer_norm -> fused_linear (the tied head) -> distill_topk_loss

in bfloat16.  The teacher is a fixed random bigram table whose k largest logits per
position are known, as they would be from a stored corpus.  Decoding runs the same
weights one token at a time: ``RavelLayerCache.step`` in place of the lookups, and the
projections' form for few rows.

    python examples/distill_student.py [--steps 200]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

from ravel_lm_b200 import RavelLayerCache, literal_addresses_from_tokens, memory_lookups  # noqa: E402
from ravel_lm_b200.dense import fused_linear  # noqa: E402
from ravel_lm_b200.distill import distill_topk_loss  # noqa: E402
from ravel_lm_b200.glue import layer_norm  # noqa: E402

Tensor = torch.Tensor


class Block(torch.nn.Module):
    """Memory read-out and feed-forward, each behind a LayerNorm."""

    def __init__(self, d: int, heads: int, payload: int, space: int, dtype=torch.bfloat16):
        super().__init__()
        self.heads, self.payload, self.space = heads, payload, space

        def p(*shape, scale=1.0, shift=0.0):
            return torch.nn.Parameter((torch.randn(*shape) * scale + shift).to(dtype))
        self.n1w, self.n1b = p(d, scale=0.0, shift=1.0), p(d, scale=0.0)
        self.n2w, self.n2b = p(d, scale=0.0, shift=1.0), p(d, scale=0.0)
        self.inw, self.inb = p(heads * payload, d, scale=d ** -0.5), p(heads * payload, scale=0.0)
        self.outw = p(d, heads * payload, scale=(heads * payload) ** -0.5)
        self.upw, self.upb = p(4 * d, d, scale=d ** -0.5), p(4 * d, scale=0.0)
        self.downw = p(d, 4 * d, scale=(4 * d) ** -0.5)

    def feed_forward(self, x: Tensor) -> Tensor:
        h = fused_linear(layer_norm(x, self.n2w, self.n2b), self.upw, self.upb, activation="silu")
        return fused_linear(h, self.downw, residual=x)

    def forward(self, x: Tensor, tokens: Tensor) -> Tensor:
        B, T, _ = x.shape
        pay = fused_linear(layer_norm(x, self.n1w, self.n1b), self.inw, self.inb)
        values, _, _, _ = memory_lookups(tokens, pay.view(B, T, self.heads, self.payload), address_space=self.space,
                                         n_literal_heads=self.heads, bos_token_id=0)
        return self.feed_forward(fused_linear(values.reshape(B, T, -1), self.outw, residual=x))

    def step(self, x: Tensor, addresses: Tensor, cache: RavelLayerCache) -> Tensor:
        """One token per stream: x [B, d], the token's literal addresses [B, heads]."""
        pay = fused_linear(layer_norm(x, self.n1w, self.n1b), self.inw, self.inb)
        values, _ = cache.step(addresses, addresses, pay.view(-1, self.heads, self.payload))
        return self.feed_forward(fused_linear(values.reshape(x.shape[0], -1), self.outw, residual=x))


class Student(torch.nn.Module):
    """Up to three literal heads: the first three address families hash a token and the two before it, whatever
    the position, so that a decoded token needs only those."""

    def __init__(self, vocab: int = 1024, d: int = 256, layers: int = 2, heads: int = 3, payload: int = 32,
                 space: int = 1024):
        super().__init__()
        self.heads, self.space = heads, space
        self.embed = torch.nn.Parameter((torch.randn(vocab, d) * d ** -0.5).bfloat16())
        self.blocks = torch.nn.ModuleList(Block(d, heads, payload, space) for _ in range(layers))
        self.nw = torch.nn.Parameter(torch.ones(d).bfloat16())
        self.nb = torch.nn.Parameter(torch.zeros(d).bfloat16())

    def head(self, x: Tensor) -> Tensor:
        return fused_linear(layer_norm(x, self.nw, self.nb), self.embed)

    def forward(self, tokens: Tensor) -> Tensor:
        x = torch.nn.functional.embedding(tokens, self.embed)
        for block in self.blocks:
            x = block(x, tokens)
        return self.head(x)

    def caches(self, streams: int) -> list[RavelLayerCache]:
        return [RavelLayerCache.empty(streams, self.heads, self.space, b.payload, device=self.embed.device,
                                      dtype=self.embed.dtype) for b in self.blocks]

    @torch.no_grad()
    def decode(self, history: Tensor, caches: list[RavelLayerCache]) -> Tensor:
        """Logits [B, vocab] after the last token of ``history`` [B, up to 3] (the literal addresses of a token
        hash it and the two before it); the caches hold the tokens before it."""
        addresses = literal_addresses_from_tokens(history, address_space=self.space, n_heads=self.heads,
                                                  bos_token_id=0)[:, -1]
        x = torch.nn.functional.embedding(history[:, -1], self.embed)
        for block, cache in zip(self.blocks, caches):
            x = block.step(x, addresses, cache)
        return self.head(x)


def teacher(vocab: int, k: int, seed: int = 0, device: str = "cuda") -> tuple[Tensor, Tensor]:
    """ids [vocab, k] and logits [vocab, k]: what the teacher expects after each token."""
    g = torch.Generator(device=device).manual_seed(seed)
    table = torch.randn(vocab, vocab, generator=g, device=device) * 3.0
    logits, ids = table.topk(k, dim=1)
    return ids, logits.bfloat16()


def train(steps: int = 200, batch: int = 16, length: int = 256, k: int = 16, lr: float = 2e-3, seed: int = 0,
          report: bool = False) -> tuple[Student, list[float]]:
    torch.manual_seed(seed)
    student = Student().cuda()
    vocab = student.embed.shape[0]
    ids, logits = teacher(vocab, k, seed)
    opt = torch.optim.AdamW(student.parameters(), lr=lr, weight_decay=0.0)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    losses = []
    for i in range(steps):
        tokens = torch.randint(1, vocab, (batch, length), generator=g, device="cuda")
        loss = distill_topk_loss(student(tokens), ids[tokens], logits[tokens], temperature=2.0)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        losses.append(loss.detach())
        if report and (i + 1) % 50 == 0:
            print(f"step {i + 1}: loss {float(losses[-1]):.4f}", flush=True)
    return student, [float(v) for v in losses]


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--steps", type=int, default=200)
    a = ap.parse_args()
    student, losses = train(a.steps, report=True)
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f}")
    tokens = torch.randint(1, student.embed.shape[0], (4, 16), device="cuda")
    caches = student.caches(4)
    for t in range(tokens.shape[1]):
        logits = student.decode(tokens[:, max(0, t - 2):t + 1], caches)
    print("next tokens:", logits.argmax(-1).tolist())


if __name__ == "__main__":
    main()
