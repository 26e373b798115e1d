"""A trained prompt adapter on the text operators: token ids -> the context a FLUX DiT (``txt``) or an
SDXL UNet (``context``) reads. It is the token-wise kind that concept learning trains (a learned token
table, normed gated feed-forward blocks, a projection to the context width); every matrix product,
norm and lookup, forward and backward, runs on this package's kernels
(:mod:`diffucore_b200.text`).

``python -m diffucore_b200.prompt`` fits one to given context vectors (here: those of a frozen, randomly
initialised teacher) and runs a small FLUX DiT on the learned context.
"""

from __future__ import annotations

import argparse
import math
import time

import torch
import torch.nn as nn

from .text import GatedFeedForward, LayerNorm, Linear, TokenEmbedding


class PromptBlock(nn.Module):
    """``x + down(act(gate(norm x)) * up(norm x))``."""

    def __init__(self, dim: int, hidden: int, activation: str, device, dtype):
        super().__init__()
        self.norm = LayerNorm(dim, device=device, dtype=dtype)
        self.ff = GatedFeedForward(dim, hidden, activation, device=device, dtype=dtype)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.ff(self.norm(x), residual=x)


class PromptAdapter(nn.Module):
    """Token ids [..., L] -> context [..., L, context_dim] in ``dtype``. ``padding_idx`` tokens keep
    their initial embedding (no gradient)."""

    def __init__(self, vocab: int, dim: int, hidden: int, context_dim: int, depth: int = 2, activation: str = "silu",
                 padding_idx: int | None = None, device=None, dtype=torch.bfloat16):
        super().__init__()
        self.embed = TokenEmbedding(vocab, dim, scale=math.sqrt(dim), padding_idx=padding_idx, device=device,
                                    dtype=dtype)
        self.blocks = nn.ModuleList(PromptBlock(dim, hidden, activation, device, dtype) for _ in range(depth))
        self.norm = LayerNorm(dim, device=device, dtype=dtype)
        self.proj = Linear(dim, context_dim, device=device, dtype=dtype)

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        x = self.embed(ids)
        for block in self.blocks:
            x = block(x)
        return self.proj(self.norm(x))


def fit_context(adapter: PromptAdapter, ids: torch.Tensor, context: torch.Tensor, steps: int, lr: float = 1e-3):
    """Train ``adapter`` to give ``context`` [B, L, context_dim] for ``ids`` [B, L] (mean squared error,
    Adam). Returns the loss of each step. The optimizer keeps fp32 copies of the 16-bit parameters:
    steps of a thousandth of a weight are below their rounding."""
    params = [p for p in adapter.parameters() if p.requires_grad]
    master = [p.detach().float().requires_grad_() for p in params]
    opt = torch.optim.Adam(master, lr=lr)
    losses = []
    for _ in range(steps):
        out = adapter(ids)
        loss = (out.float() - context.float()).square().mean()
        grads = torch.autograd.grad(loss, params)
        for m, g in zip(master, grads):
            m.grad = g.float()
        opt.step()
        with torch.no_grad():
            for p, m in zip(params, master):
                p.copy_(m)
        losses.append(loss.detach())
    return [float(v) for v in losses]


def main(argv: list[str] | None = None) -> None:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--prompts", type=int, default=16)
    ap.add_argument("--tokens", type=int, default=77)
    ap.add_argument("--vocab", type=int, default=49408)
    ap.add_argument("--dim", type=int, default=1024)
    ap.add_argument("--hidden", type=int, default=2816)
    ap.add_argument("--context", type=int, default=2048)
    ap.add_argument("--depth", type=int, default=2)
    ap.add_argument("--seed", type=int, default=0)
    args = ap.parse_args(argv)

    from . import flux
    torch.manual_seed(args.seed)
    dev = torch.device("cuda", torch.cuda.current_device())

    def make() -> PromptAdapter:
        return PromptAdapter(args.vocab, args.dim, args.hidden, args.context, args.depth, padding_idx=0, device=dev)

    ids = torch.randint(1, args.vocab, (args.prompts, args.tokens), device=dev)
    ids[:, args.tokens // 2:] = 0                            # padded prompts
    with torch.no_grad():
        target = make()(ids)
    adapter = make()
    fit_context(adapter, ids, target, 3)                     # warm-up
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    losses = fit_context(adapter, ids, target, args.steps)
    ms = (time.perf_counter() - t0) * 1e3 / args.steps
    print(f"fit {args.prompts} x {args.tokens} tokens: loss {losses[0]:.4f} -> {losses[-1]:.4f}, {ms:.2f} ms per step")

    cfg = flux.FluxConfig(context_in_dim=args.context, hidden_size=256, num_heads=2, depth=1, depth_single_blocks=1)
    model = flux.build_flux(cfg, args.seed, dev, group=256)
    with torch.no_grad():
        context = adapter(ids[:1])
        img = torch.randn(1, 64, cfg.in_channels, device=dev, dtype=torch.bfloat16)
        out = model(img, flux.img_ids(8, 8, patch=1, device=dev), context,
                    flux.txt_ids(args.tokens, device=dev), torch.tensor([1.0], device=dev),
                    torch.zeros(1, cfg.vec_in_dim, device=dev, dtype=torch.bfloat16))
    print(f"DiT on the learned context: output {tuple(out.shape)}, finite {bool(torch.isfinite(out.float()).all())}")


if __name__ == "__main__":
    main()
