"""Fits a scene in codes: every splat's colour is a row of a learned codebook.

Each splat keeps a colour of its own only while the scene is fitted.  In a step

  logits    how near that colour is to every row of the codebook
  codes     the likeliest row of each splat                       (code_log_probs, top=1)
  colours   those rows, scaled by a gain per splat                (lookup_codes)
  image     the rasterizer's; the loss is its mean squared error
            + rate * the codes' mean cost in bits                 (code_log_probs)
            + even * (balance loss - 1), so that rows stay in use (code_balance)

The colour's gradient goes to the codebook's rows (sums over the splats that name them) and, straight
through, to the splats' own colours; rate and balance reach both through the logits.  What is stored in the
end is the codebook, one code and one gain per splat.

  python examples/train_coded_scene.py [--steps 300] [--splats 4096] [--codes 64] [--size 256]
"""
from __future__ import annotations

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fast-mac-gsplat_amd"))

import torch_gsplat_bridge_fast as gs  # noqa: E402


def target_scene(splats: int, size: int, seed: int, device):
    """Splats whose colours come from twelve hues, and the image they make."""
    g = torch.Generator().manual_seed(seed)
    means = torch.rand(splats, 2, generator=g) * size
    inv = 1.0 / (1.0 + 5.0 * torch.rand(splats, generator=g)).square()
    conics = torch.stack([inv, torch.zeros(splats), inv], -1)
    opacities = 0.2 + 0.7 * torch.rand(splats, generator=g)
    depths = torch.rand(splats, generator=g)
    hues = torch.rand(12, 3, generator=g)
    colors = hues[torch.randint(0, 12, (splats,), generator=g)] * (0.6 + 0.4 * torch.rand(splats, 1, generator=g))
    return [t.to(device) for t in (means, conics, colors, opacities, depths)]


def train(steps=300, splats=4096, codes=64, size=256, rate=1e-4, even=1e-4, temperature=0.05, seed=0, device="cuda:0",
          report=None):
    """Returns {"loss", "mse", "bits", "used"}: of every step, and what is stored: {"codebook", "codes", "gains"}."""
    means, conics, colors, opacities, depths = target_scene(splats, size, seed, device)
    config = gs.RasterConfig(height=size, width=size)
    with torch.no_grad():
        target = gs.rasterize_projected_gaussians(means, conics, colors, opacities, depths, config)
    g = torch.Generator().manual_seed(seed + 1)
    own = torch.rand(splats, 3, generator=g).to(device).requires_grad_(True)
    book = torch.rand(codes, 3, generator=g).to(device).requires_grad_(True)
    gains = torch.ones(splats, device=device, requires_grad=True)
    opt = torch.optim.Adam([own, book, gains], lr=0.02)
    history = {"loss": [], "mse": [], "bits": [], "used": []}
    for step in range(steps):
        logits = 2.0 * own @ book.t() - book.square().sum(-1)   # nearness, up to a constant per splat
        with torch.no_grad():
            chosen = gs.code_log_probs(logits, top=1, temperature=temperature).top_codes[:, 0]
        cost = gs.code_log_probs(logits, chosen, temperature=temperature).log_probs.mean() / -math.log(2.0)
        balance = gs.code_balance(logits / temperature, chosen)
        through = own - own.detach()
        image = gs.rasterize_projected_gaussians(means, conics, gs.lookup_codes(chosen, book, gains) + through, opacities,
                                                 depths, config)
        mse = (image - target).square().mean()
        loss = mse + rate * cost + even * (balance.loss - 1.0)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        for k, v in (("loss", loss), ("mse", mse), ("bits", cost), ("used", (balance.counts > 0).sum())):
            history[k].append(v.detach())
        if report and (step % report == 0 or step == steps - 1):
            print(f"step {step:4d}  mse {float(mse.detach()):.5f}  bits per splat {float(cost.detach()):.2f}  "
                  f"codes in use {int(history['used'][-1])} of {codes}", flush=True)
    history = {k: torch.stack(v).float().cpu() for k, v in history.items()}
    small = torch.int16 if codes <= 1 << 15 else torch.int32  # (lookup_codes takes int32 and int64)
    return history, {"codebook": book.detach(), "codes": chosen.to(small), "gains": gains.detach()}


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=300)
    ap.add_argument("--splats", type=int, default=4096)
    ap.add_argument("--codes", type=int, default=64)
    ap.add_argument("--size", type=int, default=256)
    a = ap.parse_args()
    train(a.steps, a.splats, a.codes, a.size, report=20)
