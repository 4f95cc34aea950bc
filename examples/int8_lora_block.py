"""Train adapters on a block whose weights and activation checkpoints are in 8 bits, then serve it.

The block is an MLP between two norms (the norm after it, its gate and residual
scale, the norm before the next block), at this framework's model widths:

    y = MLP(h) with adapters         int8_lora_mlp
    h', z' = sandwich_norm(y, z)     and its codes when serving: sandwich_norm_int8

The adapters learn a teacher's change of the block from synthetic tokens, and
serving multiplies by them as trained: weights and activations between layers are
codes, the adapters' small factors and products 16 bits wide.

    python examples/int8_lora_block.py [--tokens 4096] [--steps 30] [--rank 16]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import anima_flat_b200 as afb  # noqa: E402


def make_block(dim: int, hidden: int, rank: int, device, gen) -> dict:
    """Frozen weights in 8 bits, norm weights, modulation, and fresh adapters."""
    randn = lambda *s: torch.randn(*s, generator=gen, device=device)  # noqa: E731
    bf = torch.bfloat16
    return dict(
        up=afb.quantize_weight_int8((randn(hidden, dim) / dim**0.5).to(bf), backward=True),
        down=afb.quantize_weight_int8((randn(dim, hidden) / hidden**0.5).to(bf), backward=True),
        lora_up=afb.LoRA((randn(rank, dim) / dim**0.5).to(bf), torch.zeros(hidden, rank, dtype=bf, device=device)),
        lora_down=afb.LoRA((randn(rank, hidden) / hidden**0.5).to(bf), torch.zeros(dim, rank, dtype=bf, device=device)),
        gate=(0.5 + 0.1 * randn(1, dim)).to(bf), shift=(0.1 * randn(1, dim)).to(bf),
        scale=(1 + 0.1 * randn(1, dim)).to(bf), post=1 + 0.1 * randn(dim), pre=1 + 0.1 * randn(dim),
    )


def run_block(p: dict, h: torch.Tensor, z: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    y = afb.int8_lora_mlp(h, p["up"], p["down"], p["lora_up"], p["lora_down"])
    return afb.sandwich_norm(y, z, p["gate"], p["post"], p["pre"], p["shift"], p["scale"])


def serve_block(p: dict, q: torch.Tensor, s: torch.Tensor, z: torch.Tensor):
    """The block with its adapters on codes: codes in, codes out."""

    def layer(q, s, weight, lora):
        x = afb.int8_restore(q, s).flatten(0, 1)  # the adapter's first factor is 16 bits wide
        y = afb.int8_linear((q.flatten(0, 1), s), weight).addmm_(x @ lora.a.t(), lora.b.t())
        return y.view(*q.shape[:-1], -1)

    gq, gs, _, _ = afb.gelu_int8(layer(q, s, p["up"], p["lora_up"]))
    y = layer(gq, gs, p["down"], p["lora_down"])
    return afb.sandwich_norm_int8(y, z, p["gate"], p["post"], p["pre"], p["shift"], p["scale"])


def train(tokens: int = 4096, steps: int = 30, rank: int = 16, dim: int = 2048, hidden: int = 8192,
          device: str = "cuda", seed: int = 0, verbose: bool = True) -> list[float]:
    gen = torch.Generator(device=device).manual_seed(seed)
    p = make_block(dim, hidden, rank, device, gen)
    randn = lambda *s: torch.randn(*s, generator=gen, device=device)  # noqa: E731
    teacher = dict(p, lora_down=afb.LoRA(p["lora_down"].a, (0.5 * randn(dim, rank)).to(torch.bfloat16)))
    params = [t.requires_grad_(True) for t in (*p["lora_up"], *p["lora_down"])]
    opt = torch.optim.Adam(params, lr=2e-2)
    losses = []
    for step in range(steps):
        h, z = (randn(1, tokens, dim).to(torch.bfloat16) for _ in range(2))
        with torch.no_grad():
            target, _ = run_block(teacher, h, z)
        out, _ = run_block(p, h, z)
        loss = (out.float() - target.float()).square().mean()
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        losses.append(loss.item())
        if verbose and (step % 5 == 0 or step == steps - 1):
            print(f"step {step:3d}  loss {losses[-1]:.5f}")
    if verbose:
        with torch.no_grad():
            h, z = (randn(1, tokens, dim).to(torch.bfloat16) for _ in range(2))
            q, s, z = serve_block(p, *afb.rowquant_int8(h), z)
        print(f"served {tokens} tokens: codes {list(q.shape)} {q.dtype}, residual {list(z.shape)} {z.dtype}")
        kept = tokens * (dim + 2 * hidden)
        print(f"activations kept for the backward pass of the MLP: {kept / 2**20:.0f} MiB "
              f"(bf16: {2 * kept / 2**20:.0f} MiB)")
    return losses


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=4096)
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--rank", type=int, default=16)
    a = ap.parse_args()
    train(a.tokens, a.steps, a.rank)


if __name__ == "__main__":
    main()
