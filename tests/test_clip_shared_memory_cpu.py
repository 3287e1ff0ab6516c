"""What clip_gradients writes may be nobody else's: strided tensors that share memory, and such that only lie between one
another's values.  The host's check, without a GPU."""
import math
import random

import pytest
import torch

from torch_gsplat_bridge_fast import gradients


@pytest.fixture(autouse=True)
def _any_device(monkeypatch):
    monkeypatch.setattr(gradients, "_check_device", lambda **k: None)


def _refused(g, out=None):
    with pytest.raises(ValueError, match="must not share memory"):
        gradients._check_clip(g, g if out is None else out, 1.0)


def _taken(g, out=None):
    gradients._check_clip(g, g if out is None else out, 1.0)


def _wide(rows=6, columns=10, dtype=torch.float32):
    return torch.zeros(rows, columns, dtype=dtype)


def test_columns_that_share_values_are_refused():
    b, one, two = _wide(), torch.ones(6, 3), torch.ones(6, 3)
    _refused([one, two], [b[:, :3], b[:, 2:5]])
    _refused([b[:, :3], b[:, 2:5]])
    _refused([b[:, :3], b[:, 3:6], b[:, 5:]])
    _refused([b[:, :3], b])
    _refused([b[:, :3], b[1]])
    _refused([b[:, :3], b[1, 2:3]])
    _refused([b[:3, :3], b[2:, 2:4]])
    _refused([b[::2, :3], b[1::2, :3], b[4:, 1:2]])
    _refused([b[:, 0], b[0]])
    _refused([b[:, ::2], b[:, ::3]])
    _refused([b.t()[:3], b[:, 1:2]])


def test_columns_beside_one_another_are_taken():
    b = _wide()
    _taken([b[:, :2], b[:, 2:7], b[:, 7:]])
    _taken([b[:, 7:], b[:, :2], b[:, 2:7]])
    _taken([b[:3, :3], b[3:, 2:4], b[:2, 5:]])
    _taken([b[::2], b[1::2]])
    _taken([b[::2, :4], b[1::2, :4], b[:, 4:]])
    _taken([b[:, ::2], b[:, 1::2]])
    _taken([b[:, :3], b[1, 3:]])
    _taken([b[:, 0], b[0, 1:]])
    _taken([torch.ones(6, 2), torch.ones(6, 5)], [b[:, :2], b[:, 2:7]])


def test_what_is_read_beside_what_is_written():
    b, out = _wide(), torch.zeros(6, 3)
    _taken([b[:, :3], b[:, 1:4]], [out, torch.zeros(6, 3)])  # (read twice)
    _refused([b[:, :3], torch.ones(6, 4)], [out, b[:, 2:6]])
    _refused([b[:, :3]], [b[:, 1:4]])
    _taken([b[:, :3], torch.ones(6, 4)], [out, b[:, 3:7]])
    _taken([b[:, :3]], [b[:, :3]])
    square = torch.zeros(4, 4)
    _taken([square.t()], [square])  # (a tensor's own values, in another layout)
    _refused([square.t(), torch.ones(2)], [square, square[1, :2]])


def test_tensors_that_repeat_their_own_values():
    one = torch.ones(3)
    _refused([one, torch.ones(1).expand(5)])
    _refused([torch.ones(1, 4).expand(3, 4)])
    _refused([torch.zeros(10).as_strided((4, 3), (2, 1))])
    _refused([torch.ones(4, 3)], [torch.zeros(10).as_strided((4, 3), (2, 1))])
    _taken([torch.ones(1).expand(5)], [torch.zeros(5)])
    _taken([torch.zeros(10).as_strided((4, 3), (2, 1))], [torch.ones(4, 3)])
    _taken([torch.zeros(20).as_strided((2, 3), (3, 2))])  # (offsets 0 2 4 3 5 7)
    _refused([torch.zeros(20).as_strided((3, 3), (4, 2))])  # (4 twice)


def test_types_of_one_buffer():
    b = torch.zeros(24)
    _refused([b[:8], b.view(torch.bfloat16)[15:20]])
    _taken([b[:8], b.view(torch.bfloat16)[16:20]])
    wide = b.view(6, 4)
    halves = b.view(torch.bfloat16).view(6, 8)
    _taken([wide[:, :2], halves[:, 4:]])
    _refused([wide[:, :2], halves[:, 3:]])


def _addresses(t):
    at = torch.arange(t.numel()) * 0
    for k, (n, s) in enumerate(zip(t.shape, t.stride())):
        below = math.prod(t.shape[k + 1:])
        at = at + (torch.arange(t.numel()) // below % n) * s
    return [int(a) + t.storage_offset() for a in at]


def test_against_the_values_places():
    """Random views of one buffer: exactly those that share a value are refused."""
    rng, buffer, seen = random.Random(1), torch.zeros(1000), [0, 0]
    for _ in range(4000):
        views = []
        for _ in range(rng.choice((1, 2, 2, 3))):
            nd = rng.randint(1, 3)
            shape = [rng.randint(1, 5) for _ in range(nd)]
            common = rng.choice(((40, 8, 1), (60, 12, 2), (1, 7, 35), (50, 10, 1)))
            stride = [rng.choice((common[k], common[k], rng.randint(0, 40))) for k in range(nd)]
            views.append(buffer.as_strided(shape, stride, rng.randint(0, 60)))
        places = [_addresses(v) for v in views]
        shares = any(len(set(p)) < len(p) for p in places) or len(set().union(*places)) < sum(len(set(p)) for p in places)
        seen[shares] += 1
        if shares:
            _refused(views)
        else:
            _taken(views)
    assert min(seen) > 500


def test_many_columns():
    """Hundreds of columns of one tensor are compared in order, not each with each."""
    widths = [1 + k % 9 for k in range(600)]
    b = torch.zeros(50, sum(widths))
    columns = list(b.split(widths, 1))
    calls = []
    meet = gradients._meet
    gradients._meet = lambda *a: calls.append(1) or meet(*a)
    try:
        _taken(columns)
        assert not calls
        _refused([*columns, b[:, 7:8]])
    finally:
        gradients._meet = meet
