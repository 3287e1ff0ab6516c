"""examples/train_code_decoders.py: it runs, its gradients are clipped, and those of its decoder are the formula's."""
import importlib.util
import os

import pytest
import torch

import torch_gsplat_bridge_fast as gs
from oracle.codes_reference import E

pytestmark = pytest.mark.gpu


def _example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_code_decoders.py")
    spec = importlib.util.spec_from_file_location("train_code_decoders", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    return example


@pytest.mark.parametrize("splats,codes", [(1500, 16), (9000, 81)])
def test_runs(gpu, splats, codes, monkeypatch):
    norms = []

    def clip(grads, limit, out=None):
        norm = gs_clip(grads, limit, out)
        norms.append((float(norm), torch.stack([g.double().square().sum() for g in grads]).sum().sqrt().item(), limit))
        return norm
    gs_clip = gs.clip_gradients
    monkeypatch.setattr(gs, "clip_gradients", clip)
    history, params = _example().train(steps=4, splats=splats, codes=codes, size=64)
    assert len(norms) == 4 and bool(torch.isfinite(history["loss"]).all())
    for before, after, limit in norms:
        assert 0 < before < float("inf")
        assert abs(after - min(before, limit)) <= 8 * E * limit  # (norm, factor and products rounded once each)
    assert all(bool(t.grad.any()) and bool(t.grad.isfinite().all()) for t in params.values())


def test_decoder(gpu):
    """Values and gradients beside the formula in 64 bits: the map is linear in each input, so that the same formula of
    all inputs' sizes bounds the sums of the terms' sizes, and no value is a sum of more than `terms` roundings."""
    example = _example()
    N, K, F, r = 700, 9, 16, 4
    g = torch.Generator().manual_seed(1)
    codes = torch.randint(-1, K, (N, 2), generator=g)
    ts = [torch.randn(*s, generator=g) for s in ((N, F), (N, 2), (example.VALUES, F), (K, r, F), (K, example.VALUES, r))]
    grad = torch.randn(N, example.VALUES, generator=g)

    def formula(x, w, shared, down, up):
        c, has = codes.clamp(min=0), (codes >= 0).double()
        h = torch.matmul(down[c], x[:, None, :, None])
        y = (x @ shared.t())[:, None] + torch.matmul(up[c], h)[..., 0]
        return (y * (w * has)[..., None]).sum(1)

    def both(ts, grad):
        ts = [t.double().requires_grad_(True) for t in ts]
        out = formula(*ts)
        return [out.detach(), *torch.autograd.grad(out, ts, grad.double())]

    want, size = both(ts, grad), both([t.abs() for t in ts], grad.abs())
    leaves = [t.to(gpu).requires_grad_(True) for t in ts]
    groups = gs.group_codes(codes.to(gpu), K, several=True)
    out = example.decode(leaves[0], groups, leaves[1], *leaves[2:])
    got = [out, *torch.autograd.grad(out, leaves, grad.to(gpu))]
    terms = 2 * (2 * N + F + r + example.VALUES + 16)
    for k, (a, b, s) in enumerate(zip(got, want, size)):
        assert bool(((a.detach().cpu().double() - b).abs() <= terms * E * s + 1e-30).all()), k
