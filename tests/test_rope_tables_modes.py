"""Tables of scaled positions that were first asked for in inference mode: a training pass behind it uses them too."""
import pytest
import torch

from tests.test_rotary_tangents import _stand_in
from trimkv_b200 import apply_rotary, ops
from trimkv_b200.positions import RotaryPlan

KINDS = {"default": {}, "linear": dict(factor=2.0), "llama3": dict(factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0), "yarn": dict(factor=4.0),
         "longrope": dict(short_factor=[1.0] * 4, long_factor=[2.0] * 4), "dynamic": dict(factor=2.0)}


def _check(kind, device):
    plan = RotaryPlan(8, 1e4, dict(KINDS[kind], rope_type=kind, original_max_position_embeddings=64), 128)
    pos = torch.arange(200, device=device)[None]
    with torch.inference_mode():
        first, scale = plan.on(pos.device, pos)
    freq, again = plan.on(pos.device, pos)
    assert torch.equal(first, freq) and scale == again and not freq.is_inference()
    q = torch.randn(1, 2, 200, 8, device=device, requires_grad=True)
    out, _ = apply_rotary(q, None, pos, freq, scale=scale)
    back, = torch.autograd.grad(out, q, torch.ones_like(out))
    assert bool(back.isfinite().all())


@pytest.mark.parametrize("kind", list(KINDS))
def test_tables_first_made_in_inference_mode(kind, monkeypatch):
    monkeypatch.setattr(ops, "rotary", _stand_in)
    _check(kind, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
def test_tables_first_made_in_inference_mode_on_the_gpu(kind):
    _check(kind, "cuda")
