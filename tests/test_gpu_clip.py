"""Clipped gradients of many tensors on the GPU against the 64-bit formulas (oracle/decoders_reference.py)."""
import math

import pytest
import torch

import torch_gsplat_bridge_fast as gs
from oracle import decoders_reference as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _check(gpu, grads, max_norm, what=""):
    (norm, bound), want = R.clip(grads, max_norm)
    # into tensors of their own
    on = [g.to(gpu) for g in grads]
    out = [torch.full_like(g, 7.0) for g in on]
    got = gs.clip_gradients(on, max_norm, out=out)
    assert got.dtype == F32 and got.shape == ()
    R.check(got, (norm, bound), what + " norm")
    for k, (o, w) in enumerate(zip(out, want)):
        R.check(o, w, f"{what} out[{k}]")
    for g, o in zip(grads, on):
        assert torch.equal(g.nan_to_num(7.0), o.cpu().nan_to_num(7.0))
    # in place: the same bits
    got2 = gs.clip_gradients(on, max_norm)
    assert torch.equal(got.nan_to_num(7.0), got2.nan_to_num(7.0))
    for o, g in zip(out, on):
        assert torch.equal(o.nan_to_num(7.0), g.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n", [1, 2, 3, 7, 8, 9, 255, 256, 257, 4095, 4096, 4097, 9001, 100003])
def test_sizes(gpu, dtype, n):
    g = torch.randn(n, generator=_gen(n)).to(dtype)
    norm = float(g.double().norm())
    for share in (0.1, 0.999, 1.001, 10.0):
        _check(gpu, [g], norm * share, f"n={n} {dtype} share={share}")


@pytest.mark.parametrize("count", [1, 2, 5, 100, 127, 128, 129, 300, 1000])
def test_many_tensors(gpu, count):
    """Of all types and shapes, empty ones among them."""
    g = _gen(count)
    grads = []
    for k in range(count):
        shape = ((k * 37) % 91, 1 + k % 5) if k % 7 else ()
        grads.append((torch.randn(shape, generator=g) * 10.0 ** (k % 3 - 1)).to((F32, BF16, F16)[k % 3]))
    norm = math.sqrt(sum(float(t.double().square().sum()) for t in grads))
    _check(gpu, grads, 0.3 * norm)
    _check(gpu, grads, 2.0 * norm)


def test_large(gpu):
    grads = [torch.randn(3000017, generator=_gen(1)), torch.randn(5, generator=_gen(2)).to(BF16),
             torch.randn(1 << 21, generator=_gen(3)).to(F16)]
    _check(gpu, grads, 100.0)


def test_more_tensors_than_sums_a_workgroup_adds_up(gpu):
    flat = torch.randn(5000 * 3, generator=_gen(1))
    _check(gpu, list(flat.split(3)), 1.0)


def test_range(gpu):
    """Squares past float32's range, and below it; norms past it."""
    _check(gpu, [torch.randn(1000, generator=_gen(1)) * 1e30], 1.0)
    _check(gpu, [torch.randn(1000, generator=_gen(1)) * 1e-30], 1e-29)
    _check(gpu, [torch.randn(1000, generator=_gen(1)) * 1e-42], 1e-42)
    _check(gpu, [torch.full((100,), 3e38)], 1.0)
    _check(gpu, [torch.full((100,), 65504.0).to(F16)], 1.0)
    _check(gpu, [torch.zeros(100), torch.zeros(3).to(BF16)], 1.0)
    _check(gpu, [torch.zeros(100)], 0.0)
    _check(gpu, [torch.ones(100)], 0.0)
    _check(gpu, [torch.randn(100, generator=_gen(2))], math.inf)
    _check(gpu, [torch.zeros(0), torch.zeros(0, 3).to(BF16)], 1.0)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_not_finite(gpu, bad, dtype):
    """The gradients stay as they are, and the norm says so."""
    g = torch.randn(5000, generator=_gen(1)).to(dtype)
    g[4321] = bad
    _check(gpu, [torch.randn(100, generator=_gen(2)), g], 0.5)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layouts(gpu, dtype):
    """Transposed tensors, parts of one buffer at every alignment, columns, tensors of one value repeated."""
    a = torch.randn(37, 20, generator=_gen(1)).to(dtype).to(gpu)
    flat = torch.randn(200, generator=_gen(2)).to(dtype).to(gpu)
    wide = torch.randn(50, 9, generator=_gen(3)).to(dtype).to(gpu)
    first, left = flat.clone(), wide.clone()
    grads = [a.t(), flat[1:4], flat[4:51], flat[60:197], wide[:, 2:7]]
    (norm, bound), want = R.clip([g.cpu() for g in grads], 3.0)
    R.check(gs.clip_gradients(grads, 3.0), (norm, bound), "norm")
    for k, (g, w) in enumerate(zip(grads, want)):
        R.check(g, w, f"in place [{k}]")
    inside = torch.zeros(200, dtype=torch.bool, device=gpu)
    for lo, hi in ((1, 4), (4, 51), (60, 197)):
        inside[lo:hi] = True
    assert torch.equal(flat[~inside], first[~inside])
    assert torch.equal(wide[:, :2], left[:, :2]) and torch.equal(wide[:, 7:], left[:, 7:])
    # out in another layout than the gradient
    g = torch.randn(31, 17, generator=_gen(4)).to(dtype)
    out = torch.zeros(17, 31, dtype=dtype, device=gpu).t()
    (norm, bound), want = R.clip([g], 2.0)
    R.check(gs.clip_gradients([g.to(gpu)], 2.0, out=[out]), (norm, bound), "norm")
    R.check(out, want[0], "out of another layout")
    # a broadcast gradient, into a tensor of its own
    one = torch.ones(1, dtype=dtype, device=gpu).expand(100)
    out = torch.zeros(100, dtype=dtype, device=gpu)
    assert float(gs.clip_gradients([one], 5.0, out=[out])) == 10.0 and bool((out == 0.5).all())


def test_none_and_sequences(gpu):
    a, b = torch.full((9,), 2.0, device=gpu), torch.full((16,), 2.0, device=gpu)
    assert float(gs.clip_gradients((a, None, b), 5.0)) == 10.0
    assert bool((a == 1.0).all()) and bool((b == 1.0).all())
    out = [torch.zeros_like(a), None, torch.zeros_like(b)]
    gs.clip_gradients([a, None, b], 2.5, out=out)
    assert bool((out[0] == 0.5).all()) and bool((out[2] == 0.5).all())
    gs.clip_gradients((t for t in (a, b)), math.inf)


def test_out_may_be_the_gradient(gpu):
    a, b = torch.full((9,), 2.0, device=gpu), torch.full((16,), 2.0, device=gpu)
    c = torch.zeros_like(b)
    assert float(gs.clip_gradients([a, b], 5.0, out=[a, c])) == 10.0
    assert bool((a == 1.0).all()) and bool((b == 2.0).all()) and bool((c == 1.0).all())


def test_shared_memory_is_refused(gpu):
    t = torch.ones(32, device=gpu)
    for g, out in (([t, t], None), ([t[:6], t[5:]], None), ([t[:6], t[6:12]], [t[6:12], t[:6]]), ([t[:6]], [t[1:7]])):
        with pytest.raises(ValueError, match="must not share memory"):
            gs.clip_gradients(g, 1.0, out=out)
    assert bool((t == 1.0).all())


def test_versions(gpu):
    """Autograd sees that the tensors were written."""
    x = torch.ones(4, device=gpu, requires_grad=True)
    y = x.detach() * 2
    z = (x * y).sum()
    gs.clip_gradients([y], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def test_of_parameters(gpu):
    p = [torch.randn(5, 3, device=gpu, requires_grad=True), torch.randn(7, device=gpu, requires_grad=True),
         torch.randn(2, device=gpu, requires_grad=True)]
    (p[0].square().sum() * 3 + p[1].square().sum()).backward()
    want = [t.grad.clone() for t in p[:2]]
    norm = gs.clip_gradients([t.grad for t in p], 0.5)
    (n, bound), out = R.clip([w.cpu() for w in want], 0.5)
    R.check(norm, (n, bound), "norm")
    for t, w in zip(p, out):
        R.check(t.grad, w, "grad")


def test_graph_capture_of_many_tensors(gpu):
    """Several tables of tensors in a captured graph: nothing of the host's is needed when it is replayed."""
    sizes = [1 + (k * 37) % 300 for k in range(400)]
    flat = torch.zeros(sum(sizes), device=gpu)
    out = torch.zeros_like(flat)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gs.clip_gradients(list(flat.split(sizes)), 2.0, out=list(out.split(sizes)))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = gs.clip_gradients(list(flat.split(sizes)), 2.0, out=list(out.split(sizes)))
    for k in range(3):
        new = torch.randn(flat.numel(), generator=_gen(k))
        flat.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        (want, bound), outs = R.clip([new], 2.0)
        R.check(norm, (want, bound), "norm")
        R.check(out, outs[0], "out")
        eager = flat.clone()
        assert torch.equal(gs.clip_gradients(list(eager.split(sizes)), 2.0), norm) and torch.equal(eager, out)
