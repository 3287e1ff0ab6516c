"""torch.ops.gsplat_hip.*_backward called directly: tensors that do not go together are refused (a kernel would read
past them), and strided ones give what contiguous ones give."""
import pytest
import torch

import torch_gsplat_bridge_fast as gs  # noqa: F401  (registers the operators)

pytestmark = pytest.mark.gpu

ops = torch.ops.gsplat_hip


def _refuses(op, given, name, bad):
    with pytest.raises(ValueError, match=name):
        op(**{**given, name: bad})


def _strided(t):
    """The same values, not contiguous."""
    return torch.stack([t, t], -1)[..., 0]


def _check(op, given, sized, plain):
    """sized: tensors whose every axis is checked; plain: those that may be strided."""
    want = op(**given)
    want = want if isinstance(want, tuple) else (want,)
    got = op(**{k: _strided(v) if k in plain else v for k, v in given.items()})
    for a, b in zip(want, got if isinstance(got, tuple) else (got,)):
        assert torch.equal(a, b)
    for name in sized:
        t = given[name]
        for axis in range(t.ndim):
            if t.shape[axis] > 1:
                _refuses(op, given, name, t.narrow(axis, 0, t.shape[axis] - 1))
        _refuses(op, given, name, t.flatten() if t.ndim > 1 else t[None])
        _refuses(op, given, name, t.double())
        with pytest.raises((ValueError, RuntimeError)):
            op(**{**given, name: t.cpu()})


def test_lookup(gpu):
    codes = torch.randint(-1, 40, (3, 50), device=gpu)
    given = dict(grad=torch.randn(3, 50, 7, device=gpu), codes=codes, codebook=torch.randn(40, 7, device=gpu),
                 scales=torch.rand(3, 50, device=gpu), factor=1.5, need_codebook=True, need_scales=True)
    _check(ops.lookup_codes_backward, given, ["grad", "scales"], ["grad", "codes", "codebook", "scales"])
    with pytest.raises(ValueError, match="codes must be int32 or int64"):
        ops.lookup_codes_backward(**{**given, "codes": codes.to(torch.int16)})
    with pytest.raises(ValueError, match="scales must match codes"):
        ops.lookup_codes_backward(**{**given, "codes": codes[:2]})


@pytest.mark.parametrize("top", [0, 4])
def test_log_probs(gpu, top):
    logits, codes = torch.randn(3, 50, 33, device=gpu), torch.randint(-1, 33, (3, 50), device=gpu)
    _, entropy, _, top_codes, stats = ops.code_log_probs(logits, codes, top, 1.0)
    given = dict(g_log_probs=torch.randn(3, 50, device=gpu), g_entropy=torch.randn(3, 50, device=gpu),
                 g_top=torch.randn(3, 50, top, device=gpu), logits=logits, codes=codes, top_codes=top_codes, stats=stats,
                 entropy=entropy, temperature=1.0)
    sized = ["g_log_probs", "g_entropy", "stats", "entropy"] + (["g_top"] if top else [])
    _check(ops.code_log_probs_backward, given, sized, ["g_log_probs", "g_entropy", "g_top", "codes", "stats", "entropy", "top_codes"])
    with pytest.raises(ValueError, match="codes must match logits"):
        ops.code_log_probs_backward(**{**given, "codes": codes[:2]})
    with pytest.raises(ValueError, match="temperature"):
        ops.code_log_probs_backward(**{**given, "temperature": 0.0})
    for bad in (top_codes.long(), top_codes[:2], top_codes.new_zeros(3, 50, 34)):
        with pytest.raises(ValueError, match="top"):
            ops.code_log_probs_backward(**{**given, "top_codes": bad})


@pytest.mark.parametrize("batch", [(), (3,)])
def test_balance(gpu, batch):
    logits, codes = torch.randn(*batch, 50, 33, device=gpu), torch.randint(-1, 33, (*batch, 50), device=gpu)
    _, counts, mean, stats, totals = ops.code_balance(logits, codes)
    given = dict(g_loss=torch.randn(batch, device=gpu), g_mean=torch.randn_like(mean), logits=logits, counts=counts,
                 stats=stats, totals=totals)
    _check(ops.code_balance_backward, given, ["g_loss", "g_mean", "counts", "stats", "totals"],
           ["g_loss", "g_mean", "counts", "stats", "totals"])
    with pytest.raises(ValueError, match=r"\[G,K\] or \[B,G,K\]"):
        ops.code_balance_backward(**{**given, "logits": logits[None, None]})
