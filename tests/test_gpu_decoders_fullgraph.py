"""torch.compile(fullgraph=True) of the operators of decoders by code and of clipping: torch.ops.gsplat_hip.*, without a graph
break, the same bits as the Python calls."""
import pytest
import torch

import torch_gsplat_bridge_fast as gs

pytestmark = pytest.mark.gpu

ops = torch.ops.gsplat_hip


def _ops(codes, x, dn, up, w):
    both = ops.group_codes(codes, 12, True)
    rows = ops.rows_by_code(x, *both)
    mapped = ops.code_adapters(rows, *both, dn, up, None, 1.0, True)[0]
    return ops.rows_from_codes(mapped, *both, w)


def _calls(codes, x, dn, up, w):
    both = gs.group_codes(codes, 12, several=True)
    return gs.rows_from_codes(gs.code_adapters(gs.rows_by_code(x, both), both, dn, up, by_code=True), both, w)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_fullgraph(gpu, dtype):
    g = torch.Generator().manual_seed(0)
    codes = torch.randint(-1, 12, (300, 2), generator=g).to(gpu)
    leaves = [torch.randn(*s, generator=g).to(t).to(gpu).requires_grad_(True)
              for s, t in (((300, 40), dtype), ((12, 6, 40), dtype), ((12, 24, 6), dtype), ((300, 2), torch.float32))]
    got, want = torch.compile(_ops, backend="aot_eager", fullgraph=True)(codes, *leaves), _calls(codes, *leaves)
    assert torch.equal(got, want)
    grad = torch.randn(300, 24, generator=g).to(dtype).to(gpu)
    for a, b in zip(torch.autograd.grad(got, leaves, grad), torch.autograd.grad(want, leaves, grad)):
        assert torch.equal(a, b)


def test_fullgraph_clip(gpu):
    a, b = torch.full((9,), 2.0, device=gpu), torch.full((16,), 2.0, device=gpu, dtype=torch.bfloat16)
    out = [torch.zeros_like(a), torch.zeros_like(b)]
    norm = torch.compile(lambda g, o: ops.clip_gradients_into(g, o, 5.0), backend="aot_eager", fullgraph=True)([a, b], out)
    assert float(norm) == 10.0 and all(bool((t == 1.0).all()) for t in out) and bool((a == 2.0).all())
    norm = torch.compile(lambda g: ops.clip_gradients_(g, 2.5), backend="aot_eager", fullgraph=True)([a, b])
    assert float(norm) == 10.0 and bool((a == 0.5).all()) and bool((b == 0.5).all())
