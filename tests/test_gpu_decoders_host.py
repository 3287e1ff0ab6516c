"""Decoders by code and clipped gradients where something intercepts operations or saved tensors, on several threads and
streams and in captured graphs: the same values, gradients and refusals as in the plain case."""
import threading

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import torch_gsplat_bridge_fast as gs

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _inputs(gpu, seed=0, n=300, k=12, d=40, e=24, r=6, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-1, k, (n, 2), generator=g).to(gpu)
    x, dn, up, w = (torch.randn(*s, generator=g).to(dtype).to(gpu) for s in ((n, d), (k, r, d), (k, e, r), (n, 2)))
    return codes, x, dn, up, w.float()


def _all(codes, x, dn, up, w):
    """A number of every differentiable output, and the outputs: two codes per splat there and back, and one beside a
    map that all share."""
    K = dn.shape[0]
    both = gs.group_codes(codes, K, several=True)
    rows = gs.rows_by_code(x, both)
    mapped = gs.code_adapters(rows, both, dn, up, by_code=True)
    out = gs.rows_from_codes(mapped, both, w)
    one = gs.group_codes(codes[:, 0].contiguous(), K)
    beside = gs.code_adapters(x, one, dn, up, base=out, scale=0.5)
    value = out.float().square().sum() + beside.float().sum() + rows.float().square().sum()
    return value, [*both, *one, rows, mapped, out, beside]


def _grads(gpu, seed=0, run=_all, **k):
    codes, x, dn, up, w = _inputs(gpu, seed, **k)
    leaves = [t.requires_grad_(True) for t in (x, dn, up, w)]
    value, outs = run(codes, x, dn, up, w)
    grads = list(torch.autograd.grad(value, leaves))
    copies = [g.clone() for g in grads]
    norm = gs.clip_gradients(copies, 1.0)
    return [t.detach() for t in outs] + [norm, *copies, *grads]


def _same(a, b):
    assert len(a) == len(b)
    for u, v in zip(a, b):
        assert u.dtype == v.dtype and torch.equal(u, v)


def test_saved_tensors_on_the_host(gpu):
    def run(*a):
        with torch.autograd.graph.save_on_cpu():
            return _all(*a)
    _same(_grads(gpu, run=run), _grads(gpu))


def test_saved_tensors_in_another_layout(gpu):
    """Hooks that give back strided copies."""
    def run(*a):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(),
                                                      lambda t: torch.stack([t, t], -1)[..., 0]):
            return _all(*a)
    _same(_grads(gpu, run=run), _grads(gpu))


@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpoint(gpu, reentrant):
    codes, *ts = _inputs(gpu)
    leaves = [t.requires_grad_(True) for t in ts]
    checkpoint(lambda *a: _all(codes, *a)[0], *leaves, use_reentrant=reentrant).backward()
    _same([t.grad for t in leaves], _grads(gpu)[-4:])


def test_inference_and_no_grad(gpu):
    want = _grads(gpu)[:10]
    for mode in (torch.inference_mode, torch.no_grad):
        with mode():
            _same(_all(*_inputs(gpu))[1], want)


def test_clip_of_inference_tensors(gpu):
    with torch.inference_mode():
        t = torch.full((4,), 2.0, device=gpu)
        assert float(gs.clip_gradients([t], 1.0)) == 4.0 and bool((t == 0.5).all())


@pytest.mark.parametrize("size", [300, 6000])
def test_threads(gpu, size):
    """Four threads, each with a stream and inputs of its own."""
    wants = [_grads(gpu, s, n=size) for s in range(4)]
    torch.cuda.synchronize()
    errors = []

    def work(s):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got = _grads(gpu, s, n=size)
                    torch.cuda.current_stream().synchronize()
                    _same(got, wants[s])
        except BaseException as e:  # (an assertion of a thread is the test's)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if errors:
        raise errors[0]


def test_another_stream(gpu):
    """Work follows the current stream, forward and backward, without a synchronisation between."""
    want = _grads(gpu, 3, n=20000)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _grads(gpu, 3, n=20000)
    side.synchronize()
    _same(got, want)


def test_forward_mode_is_refused(gpu):
    """There is no forward derivative: a dual input raises, and no tangent gets lost."""
    codes, x, dn, up, w = _inputs(gpu)
    two, one = gs.group_codes(codes, 12, several=True), gs.group_codes(codes[:, 0], 12)
    rows = gs.rows_by_code(x, two)
    calls = ((lambda t: gs.rows_by_code(t, two), x), (lambda t: gs.rows_from_codes(t, two), rows),
             (lambda t: gs.rows_from_codes(rows, two, t), w), (lambda t: gs.code_adapters(t, one, dn, up), x),
             (lambda t: gs.code_adapters(x, one, t, up), dn), (lambda t: gs.code_adapters(x, one, dn, t), up))
    for f, t in calls:
        for train in (False, True):
            with pytest.raises((RuntimeError, NotImplementedError)):
                with torch.autograd.forward_ad.dual_level():
                    f(torch.autograd.forward_ad.make_dual(t.detach().clone().requires_grad_(train), torch.ones_like(t)))
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(f, (t,), (torch.ones_like(t),))
    with torch.autograd.forward_ad.dual_level():
        _same(_all(codes, x, dn, up, w)[1], _grads(gpu)[:10])


def test_functional_gradients_are_refused(gpu):
    codes, x, dn, up, w = _inputs(gpu)
    one = gs.group_codes(codes[:, 0], 12)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: gs.code_adapters(t, one, dn, up).sum())(x)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: gs.rows_by_code(t, one).sum())(x)


def test_vmap(gpu):
    parts = [_inputs(gpu, s) for s in range(3)]
    got = torch.vmap(lambda *a: tuple(_all(*a)[1]))(*(torch.stack(t) for t in zip(*parts)))
    for k, part in enumerate(parts):
        _same([t[k] for t in got], _all(*part)[1])


def test_compile(gpu):
    run = torch.compile(_all, backend="aot_eager")
    _same(_grads(gpu, run=run), _grads(gpu))


def test_differentiated_once(gpu):
    """A gradient taken under create_graph says so when it is to be differentiated again."""
    codes, x, dn, up, w = _inputs(gpu)
    leaves = [t.requires_grad_(True) for t in (x, dn, up, w)]
    one, two = gs.group_codes(codes[:, 0], 12), gs.group_codes(codes, 12, several=True)
    for y, leaf in ((gs.code_adapters(x, one, dn, up).square().sum(), dn), (gs.rows_by_code(x, one).square().sum(), x),
                    (gs.rows_from_codes(gs.rows_by_code(x, two).detach().requires_grad_(True), two, w).square().sum(), w)):
        g, = torch.autograd.grad(y, leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="cannot be differentiated again"):
            torch.autograd.grad(g.sum(), leaf)


def test_operators(gpu):
    """torch.ops.gsplat_hip.*: the same values as the Python calls, and their autograd formulas."""
    ops = torch.ops.gsplat_hip
    codes, *ts = _inputs(gpu)

    def run(codes, x, dn, up, w):
        both = ops.group_codes(codes, 12, True)
        rows = ops.rows_by_code(x, *both)
        mapped = ops.code_adapters(rows, *both, dn, up, None, 1.0, True)[0]
        out = ops.rows_from_codes(mapped, *both, w)
        one = ops.group_codes(codes[:, 0].contiguous(), 12, False)
        beside = ops.code_adapters(x, *one, dn, up, out, 0.5, False)[0]
        return out.square().sum() + beside.sum() + rows.square().sum(), [*both, *one, rows, mapped, out, beside]

    _same(_grads(gpu, run=run), _grads(gpu))
    g = [torch.full((4,), 2.0, device=gpu), torch.full((9,), 2.0, device=gpu, dtype=BF16)]
    out = [torch.zeros_like(t) for t in g]
    n = ops.clip_gradients_into(g, out, 1.0)
    v = [t._version for t in g]
    assert torch.equal(n, ops.clip_gradients_(g, 1.0))
    assert all(torch.equal(a, b) for a, b in zip(g, out)) and all(t._version > k for t, k in zip(g, v))


def test_inputs_that_are_not_plain(gpu):
    """Tensor subclasses take the operators and get the same values."""
    class Sub(torch.Tensor):
        pass

    codes, x, dn, up, w = _inputs(gpu)
    one = gs.group_codes(codes[:, 0], 12)
    _same([t.as_subclass(torch.Tensor) for t in gs.group_codes(codes[:, 0].as_subclass(Sub), 12)], one)
    assert torch.equal(gs.rows_by_code(x.as_subclass(Sub), one).as_subclass(torch.Tensor), gs.rows_by_code(x, one))
    assert torch.equal(gs.code_adapters(x.as_subclass(Sub), one, dn, up).as_subclass(torch.Tensor),
                       gs.code_adapters(x, one, dn, up))
    t = x.clone()
    assert torch.equal(gs.clip_gradients([t.as_subclass(Sub)], 1.0).as_subclass(torch.Tensor),
                       gs.clip_gradients([x.clone()], 1.0))


@pytest.mark.parametrize("n,dtype", [(200, torch.float32), (7000, BF16)])
def test_graph_capture(gpu, n, dtype):
    """A step of all of them in a captured graph, replayed with new values between eager work; two graphs."""
    codes, x, dn, up, w = _inputs(gpu, n=n, dtype=dtype)
    leaves = [t.requires_grad_(True) for t in (x, dn, up, w)]

    def step():
        value, outs = _all(codes, x, dn, up, w)
        grads = torch.autograd.grad(value, leaves)
        clipped = [torch.empty_like(g) for g in grads]
        norm = gs.clip_gradients(grads, 3.0, out=clipped)
        again = gs.clip_gradients(clipped, 1.0)
        return [*outs, *grads, *clipped, norm, again]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        graphs.append((graph, held))
    for k in range(4):
        with torch.no_grad():
            new = _inputs(gpu, seed=k + 1, n=n, dtype=dtype)
            for t, v in zip((codes, x, dn, up, w), new):
                t.copy_(v)
        for graph, held in graphs:
            graph.replay()
            torch.cuda.synchronize()
            got = [t.detach().clone() for t in held]
            for a, b in zip(got, step()):
                assert torch.equal(a, b.detach())
