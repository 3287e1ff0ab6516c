"""lookup_codes, code_log_probs and code_balance where something intercepts operations or saved tensors, and on several
threads: the same values, gradients and refusals as in the plain case."""
import threading

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import torch_gsplat_bridge_fast as gs

pytestmark = pytest.mark.gpu


def _inputs(gpu, seed=0, n=300, k=45, d=6):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, k, generator=g).to(gpu)
    codes = torch.randint(-1, k, (n,), generator=g).to(gpu)
    book = torch.randn(k, d, generator=g).to(gpu)
    scales = torch.rand(n, generator=g).to(gpu)
    return x, codes, book, scales


def _all(x, codes, book, scales):
    """A number of every differentiable output, and the outputs."""
    p, b = gs.code_log_probs(x, codes, top=3, temperature=0.8), gs.code_balance(x, codes)
    out = gs.lookup_codes(codes, book, scales, 0.5)
    value = p.log_probs.sum() + 2 * p.entropy.sum() + p.top_log_probs.square().sum() + b.loss + b.mean_probs.square().sum() \
        + out.square().sum()
    return value, [p.log_probs, p.entropy, p.top_log_probs, p.top_codes, b.loss, b.counts, b.mean_probs, out]


def _grads(gpu, seed=0, run=_all):
    x, codes, book, scales = _inputs(gpu, seed)
    leaves = [t.requires_grad_(True) for t in (x, book, scales)]
    value, outs = run(x, codes, book, scales)
    return [t.detach() for t in outs] + list(torch.autograd.grad(value, leaves))


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
    x, codes, book, scales = _inputs(gpu)
    leaves = [t.requires_grad_(True) for t in (x, book, scales)]
    checkpoint(lambda *a: _all(*a)[0], x, codes, book, scales, use_reentrant=reentrant).backward()
    _same([t.grad for t in leaves], _grads(gpu)[-3:])


def test_inference_and_no_grad(gpu):
    want = _grads(gpu)[:-3]
    for mode in (torch.inference_mode, torch.no_grad):
        with mode():
            _same(_all(*_inputs(gpu))[1], want)


def test_threads(gpu):
    """Four threads, each with a stream and inputs of its own."""
    wants = [_grads(gpu, s) for s in range(4)]
    torch.cuda.synchronize()
    errors = []

    def work(s):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = _grads(gpu, s)
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


def test_forward_mode_is_refused(gpu):
    """There is no forward derivative: a dual input raises, and no tangent gets lost."""
    x, codes, book, scales = _inputs(gpu)
    calls = (lambda x, b, s: gs.code_log_probs(x, codes).entropy, lambda x, b, s: gs.code_balance(x, codes).loss,
             lambda x, b, s: gs.lookup_codes(codes, b), lambda x, b, s: gs.lookup_codes(codes, book, s))
    for train in (False, True):
        ts = [t.detach().clone().requires_grad_(train) for t in (x, book, scales)]
        for f in calls:
            with pytest.raises((RuntimeError, NotImplementedError)):
                with torch.autograd.forward_ad.dual_level():
                    f(*(torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)) for t in ts))
    for f in calls:
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(f, (x, book, scales), tuple(torch.ones_like(t) for t in (x, book, scales)))
    # a level alone is nothing to refuse
    with torch.autograd.forward_ad.dual_level():
        _same(_all(x, codes, book, scales)[1], _grads(gpu)[:-3])


def test_functional_gradients_are_refused(gpu):
    """As the rasterizer's: torch.func's transforms of autograd need what an autograd node in C++ does not have."""
    x, codes, book, scales = _inputs(gpu)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: gs.code_log_probs(t, codes).entropy.sum())(x)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: gs.lookup_codes(codes, t).sum())(book)


def test_vmap(gpu):
    parts = [_inputs(gpu, s) for s in range(3)]
    x, codes, book, scales = (torch.stack(t) for t in zip(*parts))
    got = torch.vmap(lambda *a: tuple(_all(*a)[1]))(x, codes, book, scales)
    for k, part in enumerate(parts):
        _same([t[k] for t in got], _all(*part)[1])


def test_compile(gpu):
    run = torch.compile(_all, backend="aot_eager")
    _same(_grads(gpu, run=run), _grads(gpu))
