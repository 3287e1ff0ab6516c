"""clip_gradients has no forward derivative: tensors with a tangent are refused, and none is lost."""
import pytest
import torch
from torch.autograd import forward_ad

import torch_gsplat_bridge_fast as gs


def _refused(make, device):
    def dual(v):
        return forward_ad.make_dual(torch.full((4,), v, device=device), torch.ones(4, device=device))

    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="not in forward mode"):
            make(dual)


CALLS = [lambda d, plain: gs.clip_gradients([d(2.0)], 1.0), lambda d, plain: gs.clip_gradients([plain, None, d(2.0)], 1.0),
         lambda d, plain: gs.clip_gradients([d(2.0)], 1.0, out=[plain]),
         lambda d, plain: gs.clip_gradients([plain], 1.0, out=[d(0.0)])]


@pytest.mark.parametrize("call", CALLS)
def test_refused(call):
    _refused(lambda d: call(d, torch.full((4,), 2.0)), "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("call", CALLS)
def test_refused_on_the_device(gpu, call):
    plain = torch.full((4,), 2.0, device=gpu)
    _refused(lambda d: call(d, plain), gpu)
    assert bool((plain == 2.0).all())


@pytest.mark.gpu
def test_plain_tensors_within_a_level(gpu):
    with forward_ad.dual_level():
        t = torch.full((4,), 2.0, device=gpu)
        assert float(gs.clip_gradients([t], 1.0)) == 4.0 and bool((t == 0.5).all())
