"""Decoders by code and clipped gradients without a GPU: refusals, fake implementations, the C ABI's checks, and
the 64-bit formulas the GPU tests compare with."""
import ctypes
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import torch_gsplat_bridge_fast as gs
from oracle import decoders_reference as R
from torch_gsplat_bridge_fast import _lib

BF16 = torch.bfloat16


def _raises(match, f, *a, **k):
    with pytest.raises(ValueError, match=match):
        f(*a, **k)


def _groups(n=5, S=1, K=3):
    i32 = dict(dtype=torch.int32)
    return gs.CodeGroups(torch.zeros(n * S, **i32), torch.zeros(n, S, **i32), torch.zeros(K + 1, **i32))


def test_group_refusals():
    c = torch.zeros(5, dtype=torch.int32)
    _raises("codes must be int32 or int64", gs.group_codes, c.float(), 3)
    _raises("at least one code", gs.group_codes, c, 0)
    _raises("codes are supported, not 4294967303", gs.group_codes, c, (1 << 32) + 7)
    _raises("last axis of at least one choice", gs.group_codes, c[0], 3, several=True)
    _raises("last axis of at least one choice", gs.group_codes, c[:, None][:, :0], 3, several=True)
    _raises("must be ROCm device tensors", gs.group_codes, c, 3)
    for n in ((1 << 29) + 1, (1 << 32) + 7):
        _raises(f"choices are supported, not {n}", gs.group_codes, torch.empty(n, dtype=torch.int32, device="meta"), 3)
    _raises("choices per splat are supported", gs.group_codes,
            torch.empty(1, (1 << 20) + 1, dtype=torch.int32, device="meta"), 3, several=True)


def test_rows_refusals():
    x, g = torch.zeros(5, 4), _groups()
    _raises("rows must be float32, bfloat16 or float16", gs.rows_by_code, x.double(), g)
    _raises("rows must have a last axis", gs.rows_by_code, x[:, :0], g)
    _raises("rows must have a last axis", gs.rows_by_code, x[0, 0], g)
    _raises("a row per splat", gs.rows_by_code, x[:4], g)
    _raises("a row per splat", gs.rows_by_code, x[None], g)
    _raises("must be int32", gs.rows_by_code, x, g._replace(order=g.order.long()))
    _raises("what group_codes returns", gs.rows_by_code, x, g._replace(order=g.order[:4]))
    _raises("must be ROCm device tensors", gs.rows_by_code, x, g)
    two = _groups(S=2)
    y = torch.zeros(10, 4)
    _raises("a row per choice", gs.rows_from_codes, x, two)
    _raises("a row per choice", gs.rows_from_codes, y[None], two)
    _raises("weights must be float32", gs.rows_from_codes, y, two, torch.zeros(5, 2, dtype=BF16))
    _raises("weights must match codes shape", gs.rows_from_codes, y, two, torch.zeros(5))
    _raises("must be ROCm device tensors", gs.rows_from_codes, y, two, torch.zeros(5, 2))
    _raises("values per row are supported", gs.rows_by_code, torch.empty(5, (1 << 32) + 7, device="meta"), g)


def test_adapters_refusals():
    x, g, dn, up = torch.zeros(5, 4), _groups(), torch.zeros(3, 2, 4), torch.zeros(3, 6, 2)
    f = gs.code_adapters
    _raises("rows must be float32", f, x.double(), g, dn, up)
    _raises("down must have the rows' type", f, x, g, dn.to(BF16), up)
    _raises("up must have the rows' type", f, x, g, dn, up.half())
    _raises("base must have the rows' type", f, x, g, dn, up, torch.zeros(5, 6, dtype=BF16))
    _raises("down and up must have shapes", f, x, g, dn[0], up)
    _raises("down and up must have shapes", f, x, g, dn[:, :0], up[..., :0])
    _raises("must fit each other", f, x, g, dn, up[:2])
    _raises("must fit each other", f, x, g, dn[:, :1], up)
    _raises("must fit each other", f, x[:, :3], g, dn, up)
    _raises("must fit each other", f, x, _groups(K=4), dn, up)
    _raises("a row per splat", f, x[:4], g, dn, up)
    _raises("base must have the shape", f, x, g, dn, up, torch.zeros(6))
    _raises("several codes per splat", f, x, _groups(S=2), dn, up)
    _raises("a row per choice", f, x, _groups(S=2), dn, up, by_code=True)
    _raises("ranks are supported, not 129", f, x, g, torch.zeros(3, 129, 4), torch.zeros(3, 6, 129))
    _raises("must be ROCm device tensors", f, x, g, dn, up, torch.zeros(5, 6))


def test_clip_refusals():
    a, b = torch.zeros(5, 4), torch.zeros(3, dtype=BF16)
    f = gs.clip_gradients
    _raises("at least one gradient", f, [], 1.0)
    _raises("at least one gradient", f, [None], 1.0)
    _raises("gradients must be float32", f, [a.double()], 1.0)
    for m in (-1.0, math.nan):
        _raises("max_norm must be at least 0", f, [a], m)
    _raises("out must have a tensor for each", f, [a, b], 1.0, out=[a])
    _raises("must not require gradients", f, [a.requires_grad_(True)], 1.0)
    a = a.detach()
    _raises("types, shapes and devices", f, [a], 1.0, out=[b])
    _raises("types, shapes and devices", f, [a], 1.0, out=[a[:4]])
    _raises("must be on the same device", f, [a, a.to("meta")], 1.0)
    _raises("must be ROCm device tensors", f, [a, b], 1.0)


@pytest.mark.parametrize("make", [
    lambda t: ([t, t], None), lambda t: ([t[:6], t[5:]], None), lambda t: ([t[:5], t[5:], t], None),
    lambda t: ([t[:6], t[6:12]], [t[5:11], t[12:18]]), lambda t: ([t[:6], t[6:12]], [t[6:12], t[:6]]),
    lambda t: ([t[:6], t[6:12]], [t[12:18], t[12:18]]), lambda t: ([t[:6], t[6:12]], [t[:6], t[:6]])])
def test_clip_shared_memory_is_refused(make, monkeypatch):
    """Whatever is written may be nobody else's, read or written."""
    from torch_gsplat_bridge_fast import gradients
    monkeypatch.setattr(gradients, "_check_device", lambda **k: None)
    g, out = make(torch.zeros(18))
    _raises("must not share memory", gradients._check_clip, g, g if out is None else out, 1.0)


def test_clip_neighbours_are_not_refused(monkeypatch):
    from torch_gsplat_bridge_fast import gradients
    monkeypatch.setattr(gradients, "_check_device", lambda **k: None)
    t = torch.zeros(18)
    gradients._check_clip([t[6:12], t[:6], t[12:12]], [t[6:12], t[:6], t[12:12]], 1.0)
    gradients._check_clip([t[:6], t[6:9]], [t[:6], t[9:12]], 1.0)
    gradients._check_clip([t[:6], t[:6]], [t[6:12], t[12:]], 1.0)


def test_fake_implementations():
    ops = torch.ops.gsplat_hip
    with FakeTensorMode():
        c = torch.zeros(2, 5, dtype=torch.int64)
        order, places, starts = ops.group_codes(c, 7, False)
        assert order.shape == (10,) and places.shape == (2, 5, 1) and starts.shape == (8,)
        assert order.dtype == places.dtype == starts.dtype == torch.int32
        order, places, starts = ops.group_codes(c, 7, True)
        assert places.shape == (2, 5)
        x = torch.zeros(2, 4, dtype=BF16)
        y = ops.rows_by_code(x, order, places, starts)
        assert y.shape == (10, 4) and y.dtype == BF16
        assert ops.rows_from_codes(y, order, places, starts, None).shape == (2, 4)
        out, hidden = ops.code_adapters(y, order, places, starts, torch.zeros(7, 3, 4, dtype=BF16),
                                        torch.zeros(7, 6, 3, dtype=BF16), None, 1.0, True)
        assert out.shape == (10, 6) and out.dtype == BF16 and hidden.shape == (10, 3) and hidden.dtype == torch.float32
        assert ops.clip_gradients_([y, x], 1.0).shape == ()


def _refused(rc, text):
    assert rc == 1 and text in _lib.lib().gsplat_hip_last_error().decode()


def test_c_abi_refusals():
    L, d = _lib.lib(), ctypes.c_void_p(256)
    for m, text in ((_lib.GroupMeta((1 << 29) + 1, 3, 4), "choices must lie"), (_lib.GroupMeta(5, 0, 4), "num_codes must lie"),
                    (_lib.GroupMeta(5, 3, 2), "code_bytes"), (_lib.GroupMeta(-1, 3, 4), "choices must lie")):
        _refused(L.gsplat_hip_group_codes(m, d, d, d, d, None, 0, None), text)
        assert L.gsplat_hip_group_codes_workspace_bytes(m) == 0
    m = _lib.GroupMeta(100000, 300, 4)
    _refused(L.gsplat_hip_group_codes(m, None, d, d, d, d, 1 << 30, None), "NULL")
    assert L.gsplat_hip_group_codes(m, d, d, d, d, d, 16, None) == 3
    assert "workspace too small" in L.gsplat_hip_last_error().decode()
    for m, text in ((_lib.RowsMeta(5, 0, 3, 3, 0), "choices must lie"), (_lib.RowsMeta(1 << 28, 4, 3, 3, 0), "splats * choices"),
                    (_lib.RowsMeta(5, 1, 0, 3, 0), "width must lie"), (_lib.RowsMeta(5, 1, 3, 2, 0), "stride"),
                    (_lib.RowsMeta(5, 1, 3, 3, 3), "dtype")):
        _refused(L.gsplat_hip_rows_by_code(m, d, d, d, d, None, d, None), text)
        _refused(L.gsplat_hip_rows_from_codes(m, d, d, None, d, None), text)
        _refused(L.gsplat_hip_rows_from_codes_backward(m, d, d, d, d, d, None, d, None, None), text)
    _refused(L.gsplat_hip_rows_by_code(_lib.RowsMeta(5, 1, 3, 3, 0), d, None, d, d, None, d, None), "NULL")
    _refused(L.gsplat_hip_rows_from_codes_backward(_lib.RowsMeta(5, 1, 3, 3, 0), d, None, d, d, d, d, d, d, None), "NULL")
    ok = (5, 3, 2, 4, 6, 4, 0, 0, 1.0)
    for at, v, text in ((0, -1, "rows must lie"), (1, 0, "num_codes"), (2, 129, "rank must lie"), (2, 0, "rank must lie"),
                        (3, 0, "width_in"), (4, (1 << 20) + 1, "width_out"), (5, 3, "stride"), (6, 7, "dtype")):
        m = _lib.AdaptersMeta(*(v if k == at else x for k, x in enumerate(ok)))
        _refused(L.gsplat_hip_code_adapters_forward(m, *[d] * 10, 0, None), text)
        _refused(L.gsplat_hip_code_adapters_backward(m, *[d] * 12, 0, None), text)
    _refused(L.gsplat_hip_code_adapters_forward(_lib.AdaptersMeta(5, 1 << 28, 128, 1 << 10, 6, 1 << 10, 0, 0, 1.0),
                                                *[d] * 10, 0, None), "at most 2^40")
    one = (_lib.ClipTensor * 1)()
    one[0].source, one[0].to, one[0].size, one[0].dtype = 256, 256, 5, 0
    _refused(L.gsplat_hip_clip_gradients(one, 1, -1.0, d, d, 1 << 20, None), "max_norm")
    _refused(L.gsplat_hip_clip_gradients(one, 1, math.nan, d, d, 1 << 20, None), "max_norm")
    _refused(L.gsplat_hip_clip_gradients(one, -1, 1.0, d, d, 1 << 20, None), "count")
    _refused(L.gsplat_hip_clip_gradients(one, 1, 1.0, None, d, 1 << 20, None), "NULL")
    one[0].dtype = 3
    _refused(L.gsplat_hip_clip_gradients(one, 1, 1.0, d, d, 1 << 20, None), "dtype")
    one[0].dtype, one[0].size = 0, -1
    _refused(L.gsplat_hip_clip_gradients(one, 1, 1.0, d, d, 1 << 20, None), "sizes must lie")
    one[0].size = 5
    assert L.gsplat_hip_clip_gradients(one, 1, 1.0, d, None, 0, None) == 3


# ---- the formulas themselves, against autograd and against loops


def test_group_formula():
    codes = torch.tensor([[2, -1], [0, 2], [5, 2], [0, -7]])
    order, places, starts = R.group(codes, 4, several=True)
    assert order.tolist() == [2, 6, 0, 3, 5, 1, 4, 7]
    assert places.tolist() == [[2, -1], [0, 3], [-2, 4], [1, -2]]
    assert starts.tolist() == [0, 2, 2, 5, 5]


@pytest.mark.parametrize("S", [1, 3])
def test_rows_formulas(S):
    gen = torch.Generator().manual_seed(S)
    codes = torch.randint(-1, 4, (9, S), generator=gen)
    groups = R.group(codes, 4, several=True)
    x = torch.randn(9, 5, generator=gen, dtype=torch.float64, requires_grad=True)
    w = torch.rand(9, S, generator=gen, dtype=torch.float64, requires_grad=True)
    g = torch.randn(9, 5, generator=gen, dtype=torch.float64)
    place, keep = groups[1].long(), (groups[1] >= 0).double()
    splat = groups[0].long() // S
    y = x[splat] * (torch.arange(9 * S) < int(groups[2][-1])).double()[:, None]
    out = (y[place.clamp(min=0)] * (w * keep)[..., None]).sum(1)
    gx, gw = torch.autograd.grad(out, [x, w], g)
    y32 = R.by_code(x.detach().float(), groups)["out"][0].float()
    back = R.from_codes(y32, groups, w.detach().float(), g.float())
    assert torch.allclose(back["out"][0], out.detach(), atol=1e-5)
    assert torch.allclose(back["g_weights"][0], gw, atol=1e-5)
    there = R.by_code(x.detach().float(), groups, back["g_rows"][0].float())
    assert torch.allclose(there["g_rows"][0], gx, atol=1e-5)


@pytest.mark.parametrize("by_code", [False, True])
def test_adapters_formulas(by_code):
    gen = torch.Generator().manual_seed(3)
    f64 = dict(dtype=torch.float64, generator=gen)
    codes = torch.randint(-1, 4, (11,), generator=gen)
    groups = R.group(codes, 4)
    c = codes[groups[0].long()] if by_code else codes
    x, dn, up = (torch.randn(*s, **f64).float().double().requires_grad_(True) for s in ((11, 6), (4, 3, 6), (4, 5, 3)))
    base, g = torch.randn(11, 5, **f64).float().double(), torch.randn(11, 5, **f64).float().double()
    h = (dn[c.clamp(min=0)] @ x[..., None]) * (c >= 0).double()[:, None, None]
    out = base + 0.7 * (up[c.clamp(min=0)] @ h)[..., 0]
    want = torch.autograd.grad(out, [x, dn, up], g)
    r = R.adapters(x.detach().float(), groups, dn.detach().float(), up.detach().float(), base.float(), 0.7, by_code, g.float())
    assert torch.allclose(r["out"][0], out.detach())
    for k, t in zip(("g_rows", "g_down", "g_up"), want):
        assert torch.allclose(r[k][0], t)


def test_clip_formula():
    g = [torch.tensor([3.0, 0.0]), torch.tensor([4.0], dtype=BF16)]
    (norm, _), out = R.clip(g, 2.5)
    assert float(norm) == 5.0 and out[0][0].tolist() == [1.5, 0.0] and out[1][0].tolist() == [2.0]
    (norm, _), out = R.clip(g, 7.0)
    assert out[0][0].tolist() == [3.0, 0.0]
    (norm, _), out = R.clip([torch.tensor([math.inf, 1.0])], 1.0)
    assert math.isinf(float(norm)) and out[0][0].tolist() == [math.inf, 1.0]
