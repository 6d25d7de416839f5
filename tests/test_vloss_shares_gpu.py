"""Gradients of the CUDA-core forms where ignored tokens would leave room for more shares of dx than the launch has blocks for."""
import pytest
import torch

from tests.test_vloss_gpu import BF, HF, SF, _check, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,t,v,h,keep", [
    (SF, 300, 32000, 4098, 0.7), (BF, 300, 32000, 4098, 0.4), (HF, 600, 32000, 4098, 0.5), (SF, 1500, 50257, 1001, 0.1), (BF, 1500, 32000, 1001, 0.1),
    (BF, 1500, 32000, 1001, 1.0)])
def test_widths_that_are_not_whole_vectors(dtype, t, v, h, keep):
    _check(*_inputs(t, v, h, dtype, keep=keep, seed=5), reduction="mean")


@pytest.mark.parametrize("dtype", [BF, SF])
def test_a_weight_between_vectors(dtype):
    x, w, y = _inputs(300, 32000, 4104, dtype, keep=0.5, seed=6)
    store = torch.empty(w.numel() + 1, dtype=dtype, device="cuda")
    held = store[1:].view_as(w)
    held.copy_(w)
    assert held.data_ptr() % 16
    _check(x, held, y, reduction="mean")


def test_few_tokens_of_a_wide_fp32_head():
    """A few rows, in pieces of 512 columns: the form of up to 32 tokens."""
    x, w, y = _inputs(16, 6368, 51432, SF, seed=7, sharp=False)
    y[7:] = -100
    _check(x, w, y, reduction="mean")
