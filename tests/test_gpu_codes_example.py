"""examples/train_coded_scene.py with more codes than 16 bits hold: what is stored names the codes of the last step."""
import importlib.util
import os

import pytest
import torch

import torch_gsplat_bridge_fast as gs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("codes,dtype", [(300, torch.int16), (1 << 15, torch.int16), (40000, torch.int32), (70000, torch.int32)])
def test_stored_codes(gpu, codes, dtype, monkeypatch):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_coded_scene.py")
    spec = importlib.util.spec_from_file_location("train_coded_scene", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    chosen = []

    def lookup(c, *a):
        chosen.append(c)
        return lookup_codes(c, *a)
    lookup_codes = gs.lookup_codes
    monkeypatch.setattr(gs, "lookup_codes", lookup)
    _, stored = example.train(steps=2, splats=2000, codes=codes, size=32)
    assert stored["codes"].dtype == dtype
    assert torch.equal(stored["codes"].to(torch.int32), chosen[-1])
    assert codes <= 300 or int(chosen[-1].max()) > codes // 2
