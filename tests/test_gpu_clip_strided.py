"""clip_gradients of strided tensors on the GPU: refused before anything is written where they share memory, and scaled
where they only lie between one another's values."""
import pytest
import torch

import torch_gsplat_bridge_fast as gs
from oracle import decoders_reference as R

pytestmark = pytest.mark.gpu


def test_refused_before_anything_is_written(gpu):
    one, wide = torch.full((3,), 2.0, device=gpu), torch.ones(4, 6, device=gpu)
    for g, out in (([one, torch.ones(1, device=gpu).expand(5)], None), ([one, wide[:, :3], wide[:, 2:5]], None),
                   ([one, wide[:, :3], wide[1]], None), ([wide[:, :3]], [wide[:, 1:4]]),
                   ([one, torch.ones(4, 3, device=gpu)], [one, torch.ones(3, device=gpu).expand(4, 3)])):
        with pytest.raises(ValueError, match="must not share memory"):
            gs.clip_gradients(g, 0.5, out=out)
    assert bool((one == 2.0).all()) and bool((wide == 1.0).all())


def test_columns_and_rows_between_one_another(gpu):
    wide = torch.randn(50, 12, generator=torch.Generator().manual_seed(1))
    for cut in (lambda t: [t[:, 5:9], t[:, :5], t[:, 9:]], lambda t: [t[::2, :7], t[1::2, :7], t[:, 7:]]):
        for into in (False, True):
            on = wide.to(gpu)
            grads = cut(on)
            out = cut(torch.zeros_like(on)) if into else grads
            (norm, bound), want = R.clip([t.cpu() for t in grads], 3.0)
            R.check(gs.clip_gradients(grads, 3.0, out=out if into else None), (norm, bound), "norm")
            for o, w in zip(out, want):
                R.check(o, w, "out")
