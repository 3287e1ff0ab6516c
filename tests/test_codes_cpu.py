"""Scenes in codes without a GPU: refusals, fake implementations, the C ABI's checks, and the 64-bit
formulas the GPU tests compare with."""
import ctypes
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import torch_gsplat_bridge_fast as gs
from oracle import codes_reference as R
from torch_gsplat_bridge_fast import _lib


def _raises(match, f, *a, **k):
    with pytest.raises(ValueError, match=match):
        f(*a, **k)


def test_lookup_refusals():
    c, b = torch.zeros(5, dtype=torch.int32), torch.zeros(7, 3)
    _raises("codes must be int32 or int64", gs.lookup_codes, c.float(), b)
    _raises("codes must be int32 or int64", gs.lookup_codes, c.to(torch.int16), b)
    _raises("codebook must be float32, bfloat16 or float16", gs.lookup_codes, c, b.double())
    _raises(r"codebook must have shape \[K,D\]", gs.lookup_codes, c, b[0])
    _raises(r"codebook must have shape \[K,D\]", gs.lookup_codes, c, b[:0])
    _raises(r"codebook must have shape \[K,D\]", gs.lookup_codes, c, b[:, :0])
    _raises("scales must be float32", gs.lookup_codes, c, b, torch.ones(5, dtype=torch.bfloat16))
    _raises("scales must match codes shape", gs.lookup_codes, c, b, torch.ones(4))
    _raises("must be ROCm device tensors", gs.lookup_codes, c, b)
    _raises("must be on the same device", gs.lookup_codes, c, b.to("meta"))


def test_log_probs_refusals():
    c, x = torch.zeros(5, dtype=torch.int64), torch.zeros(5, 9)
    _raises("logits must be float32, bfloat16 or float16", gs.code_log_probs, x.double(), c)
    _raises("logits must have a last axis", gs.code_log_probs, x[:, :0], c)
    _raises("logits must have a last axis", gs.code_log_probs, x[0, 0])
    _raises("codes must match logits shape", gs.code_log_probs, x, c[:4])
    _raises("codes must be int32 or int64", gs.code_log_probs, x, c.float())
    _raises(r"top must lie in \[0, 9\]", gs.code_log_probs, x, c, top=10)
    _raises(r"top must lie in \[0, 64\]", gs.code_log_probs, torch.zeros(5, 100), c, top=65)
    _raises("top must lie in", gs.code_log_probs, x, c, top=-1)
    for T in (0.0, -1.0, math.inf, math.nan, 1e-40):
        _raises("temperature must lie in", gs.code_log_probs, x, c, temperature=T)
    _raises("must be ROCm device tensors", gs.code_log_probs, x, c)


def test_balance_refusals():
    c, x = torch.zeros(2, 5, dtype=torch.int64), torch.zeros(2, 5, 9)
    _raises("logits must be float32, bfloat16 or float16", gs.code_balance, x.double(), c)
    _raises(r"logits must have shape \[G,K\] or \[B,G,K\]", gs.code_balance, x[0, 0], c[0, 0])
    _raises(r"logits must have shape \[G,K\] or \[B,G,K\]", gs.code_balance, x[None], c[None])
    _raises("codes must have the shape of logits", gs.code_balance, x, c[:, :4])
    _raises("codes must have the shape of logits", gs.code_balance, x, c[..., None][..., :0])
    _raises("codes must be int32 or int64", gs.code_balance, x, c.float())
    _raises("at least one image", gs.code_balance, x[:0], c[:0])
    _raises("must be ROCm device tensors", gs.code_balance, x, c)


def test_fake_implementations():
    ops = torch.ops.gsplat_hip
    with FakeTensorMode():
        c = torch.zeros(2, 5, dtype=torch.int32)
        out = ops.lookup_codes(c, torch.zeros(7, 3, dtype=torch.bfloat16), None, 1.0)
        assert out.shape == (2, 5, 3) and out.dtype == torch.bfloat16
        x = torch.zeros(2, 5, 9, dtype=torch.float16)
        lp, H, tl, tc, st = ops.code_log_probs(x, c, 3, 1.0)
        assert lp.shape == H.shape == (2, 5) and tl.shape == tc.shape == (2, 5, 3)
        assert lp.dtype == torch.float32 and tc.dtype == torch.int32
        assert ops.code_log_probs(x, None, 0, 1.0)[0].shape == (0,)
        loss, counts, mean, _, _ = ops.code_balance(x, c)
        assert loss.shape == (2,) and counts.shape == mean.shape == (2, 9) and counts.dtype == torch.int32
        assert ops.code_balance(x[0], c[0])[0].shape == ()


def _refused(rc, text):
    assert rc == 1 and text in _lib.lib().gsplat_hip_last_error().decode()


def test_c_abi_checks():
    L, d = _lib.lib(), ctypes.c_void_p(256)

    def lookup(**kw):
        m = _lib.LookupMeta(10, 5, 3, 3, 0, 4, 1.0)
        for k, v in kw.items():
            setattr(m, k, v)
        return m
    _refused(L.gsplat_hip_lookup_forward(None, d, d, None, d, None), "meta is NULL")
    for kw, text in ((dict(rows=-1), "rows"), (dict(rows=(1 << 29) + 1), "rows"), (dict(num_codes=0), "num_codes"),
                     (dict(width=0), "width"), (dict(stride=2), "stride"), (dict(dtype=3), "dtype"), (dict(code_bytes=2), "code_bytes")):
        _refused(L.gsplat_hip_lookup_forward(lookup(**kw), d, d, None, d, None), text)
        _refused(L.gsplat_hip_lookup_backward(lookup(**kw), d, d, d, None, d, None, d, 1 << 30, None), text)
        assert L.gsplat_hip_lookup_backward_workspace_bytes(lookup(**kw)) == 0
    _refused(L.gsplat_hip_lookup_forward(lookup(), None, d, None, d, None), "NULL pointer")
    many = lookup(rows=100_000)  # (few splats need no workspace)
    need = L.gsplat_hip_lookup_backward_workspace_bytes(many)
    assert need > 0
    assert L.gsplat_hip_lookup_backward(many, d, d, d, None, d, None, d, need - 1, None) == 3

    def probs(**kw):
        m = _lib.ProbsMeta(10, 5, 2, 5, 0, 4, 1.0)
        for k, v in kw.items():
            setattr(m, k, v)
        return m
    for kw, text in ((dict(rows=1 << 31), "rows"), (dict(num_codes=0), "num_codes"), (dict(top=6), "top"), (dict(top=-1), "top"),
                     (dict(num_codes=100, stride=100, top=65), "top"), (dict(stride=4), "stride"), (dict(dtype=-1), "dtype"),
                     (dict(code_bytes=1), "code_bytes"), (dict(temperature=0.0), "temperature"),
                     (dict(temperature=float("nan")), "temperature"), (dict(temperature=float("inf")), "temperature")):
        _refused(L.gsplat_hip_code_probs_forward(probs(**kw), d, d, d, d, d, d, None, d, 1 << 30, None), text)
        _refused(L.gsplat_hip_code_probs_backward(probs(**kw), d, d, d, d, d, d, d, d, d, None), text)
    _refused(L.gsplat_hip_code_probs_forward(probs(), d, None, d, d, d, d, None, d, 1 << 30, None), "log_probs goes with codes")
    _refused(L.gsplat_hip_code_probs_forward(probs(), d, d, d, d, None, None, None, d, 1 << 30, None), "NULL pointer")
    _refused(L.gsplat_hip_code_probs_backward(probs(), d, None, d, d, d, d, d, d, d, None), "NULL pointer")

    def balance(**kw):
        m = _lib.BalanceMeta(10, 2, 5, 1, 0, 5, 4)
        for k, v in kw.items():
            setattr(m, k, v)
        return m
    for kw, text in ((dict(batch=0), "batch"), (dict(batch=65536), "batch"), (dict(choices=0), "choices"), (dict(rows=-1), "rows"),
                     (dict(rows=1 << 30), "rows"), (dict(num_codes=0), "num_codes"), (dict(stride=4), "stride"), (dict(dtype=9), "dtype")):
        _refused(L.gsplat_hip_code_balance_forward(balance(**kw), d, d, d, d, d, d, d, d, 1 << 40, None), text)
        _refused(L.gsplat_hip_code_balance_backward(balance(**kw), d, d, d, d, d, d, d, None), text)
    _refused(L.gsplat_hip_code_balance_forward(balance(), d, None, d, d, d, d, d, d, 1 << 40, None), "NULL pointer")


def test_reference_against_autograd():
    """The 64-bit formulas' gradients against torch's own derivatives of their values."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 6, 17, generator=g, dtype=torch.float64)
    codes = torch.randint(-1, 17, (2, 6), generator=g)
    gl, ge, gt = torch.randn(2, 6, generator=g), torch.randn(2, 6, generator=g), torch.randn(2, 6, 2, generator=g)
    xg = x.clone().requires_grad_(True)
    lp = torch.log_softmax(xg / 0.7, -1)
    loss = ((lp.gather(-1, codes.clamp(min=0)[..., None])[..., 0] * gl * (codes >= 0)).sum()
            - ((lp.exp() * lp).sum(-1) * ge).sum() + (lp.topk(2, -1).values * gt).sum())
    want, = torch.autograd.grad(loss, xg)
    R.U[torch.float64], R.TINY[torch.float64] = 0.0, 1e-300
    try:
        got = R.probs(x, codes, 2, 0.7, gl, ge, gt)
        torch.testing.assert_close(got["g_logits"][0], want, rtol=1e-10, atol=1e-12)
        p = torch.softmax(xg, -1) * (codes >= 0)[..., None]
        rows = (codes >= 0).sum(-1, keepdim=True)
        counts = torch.stack([torch.bincount(c[c >= 0], minlength=17) for c in codes]).double()
        mean = p.sum(1) / rows
        gm = torch.randn(2, 17, generator=g, dtype=torch.float64)
        loss = 17 * (counts / rows * mean).sum(-1)
        want, = torch.autograd.grad((loss * torch.tensor([0.5, 2.0])).sum() + (mean * gm).sum(), xg)
        got = R.balance(x, codes, torch.tensor([0.5, 2.0]), gm)
        torch.testing.assert_close(got["g_logits"][0], want, rtol=1e-10, atol=1e-12)
        torch.testing.assert_close(got["loss"][0], loss.detach(), rtol=1e-12, atol=0)
    finally:
        del R.U[torch.float64], R.TINY[torch.float64]


def test_bounds_notice_mistakes():
    """A wrong value in the oracle's place is outside its bound."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 40, generator=g)
    codes = torch.randint(0, 40, (5,), generator=g)
    want = R.probs(x, codes, 2, 1.0, torch.ones(5), torch.ones(5), torch.ones(5, 2))
    for k, (v, b) in want.items():
        R.check(v.to(torch.int32 if b is None else torch.float32), (v, b), k)
        with pytest.raises(AssertionError):
            R.check(v.to(torch.int32) + 1 if b is None else v.float() * 1.001, (v, b), k)
    with pytest.raises(AssertionError):
        R.check(want["entropy"][0].float().clone().fill_(math.nan), want["entropy"], "NaN")
