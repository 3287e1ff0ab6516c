"""Fits a scene whose codes are decoders: every splat has a few features, and its codes name the maps that turn them
into a colour and an opacity.

Codes are anchors on the image; a splat has the nearest two, with weights by distance.  In a step

  groups    the splats' codes by code                              (group_codes, once: they stay)
  rows      features, a copy for each code                         (rows_by_code)
  decoded   a map that all share + a map of low rank by code       (code_adapters, beside rows @ shared)
  values    weighted sums over a splat's codes                     (rows_from_codes)
  image     the rasterizer's; the loss is its mean squared error
  clipping  the gradients of features and maps, together           (clip_gradients)

  python examples/train_code_decoders.py [--steps 300] [--splats 4096] [--codes 64] [--size 256]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fast-mac-gsplat_amd"))

import torch_gsplat_bridge_fast as gs  # noqa: E402

VALUES = 4  # a colour and an opacity


def decode(features, groups, weights, shared, down, up):
    """[N, VALUES] of features [N, F]: by each of a splat's codes, weighted."""
    rows = gs.rows_by_code(features, groups)
    decoded = gs.code_adapters(rows, groups, down, up, base=rows @ shared.t(), by_code=True)
    return gs.rows_from_codes(decoded, groups, weights)


def anchors(means, codes, size):
    """The two nearest of `codes` anchors on a grid, and their weights."""
    side = max(1, int(round(codes ** 0.5)))
    at = (torch.arange(codes, device=means.device) + 0.5)
    grid = torch.stack([at % side, at.div(side, rounding_mode="floor") + 0.5], -1) * (size / side)
    near = torch.cdist(means, grid).topk(2, largest=False)
    return near.indices.to(torch.int32), torch.softmax(-near.values / (size / side), -1)


def train(steps=300, splats=4096, codes=64, size=256, features=16, rank=4, limit=0.05, seed=0, device="cuda:0", report=None):
    """Returns {"loss", "norm"} of every step, and the parameters."""
    g = torch.Generator().manual_seed(seed)
    means = (torch.rand(splats, 2, generator=g) * size).to(device)
    inv = 1.0 / (1.0 + 5.0 * torch.rand(splats, generator=g)).square()
    conics, depths = torch.stack([inv, torch.zeros(splats), inv], -1).to(device), torch.rand(splats, generator=g).to(device)
    config = gs.RasterConfig(height=size, width=size)
    chosen, weights = anchors(means, codes, size)
    groups = gs.group_codes(chosen, codes, several=True)

    def image_of(values):
        shaped = torch.sigmoid(values)
        return gs.rasterize_projected_gaussians(means, conics, shaped[:, :3].contiguous(), shaped[:, 3].contiguous(), depths, config)

    def normal(*shape, scale=1.0):
        return (scale * torch.randn(*shape, generator=g)).to(device)

    with torch.no_grad():
        target = image_of(normal(codes, VALUES)[chosen[:, 0].long()])
    params = {"features": normal(splats, features, scale=0.5), "shared": normal(VALUES, features, scale=features ** -0.5),
              "down": normal(codes, rank, features, scale=features ** -0.5), "up": normal(codes, VALUES, rank, scale=0.01)}
    for t in params.values():
        t.requires_grad_(True)
    opt = torch.optim.Adam(params.values(), lr=0.02)
    history = {"loss": [], "norm": []}
    for step in range(steps):
        values = decode(params["features"], groups, weights, params["shared"], params["down"], params["up"])
        loss = (image_of(values) - target).square().mean()
        opt.zero_grad(set_to_none=True)
        loss.backward()
        norm = gs.clip_gradients([t.grad for t in params.values()], limit)
        opt.step()
        history["loss"].append(loss.detach())
        history["norm"].append(norm)
        if report and (step % report == 0 or step == steps - 1):
            print(f"step {step:4d}  loss {float(loss.detach()):.5f}  gradients' norm {float(norm):.4f}", flush=True)
    return {k: torch.stack(v).cpu() for k, v in history.items()}, params


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=300)
    ap.add_argument("--splats", type=int, default=4096)
    ap.add_argument("--codes", type=int, default=64)
    ap.add_argument("--size", type=int, default=256)
    a = ap.parse_args()
    train(a.steps, a.splats, a.codes, a.size, report=20)
