"""Gradients after a wait ran out: with the plan's mark set (by the host: nothing waits), nothing that is returned may be taken for a gradient."""
import pytest
import torch

from tests.test_vloss_gpu import BF, HF, SF, _inputs
from trimkv_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,t,v,h", [(BF, 300, 9000, 128), (HF, 3, 700, 264), (SF, 300, 5000, 128), (SF, 8, 3001, 64), (BF, 40, 500, 33)])
@pytest.mark.parametrize("want_dx,want_dw", [(True, True), (False, True), (True, False)])
def test_marked_gradients_are_nan(dtype, t, v, h, want_dx, want_dw):
    x, w, y = _inputs(t, v, h, dtype, keep=0.8)
    y[0] = 1
    _, _, plan = ops.vloss_forward(x, w, y, -100, 1)
    grad = torch.ones((), device="cuda")
    for mark in (0, 1):
        plan[2] = mark
        for got in ops.vloss_backward(x, w, plan, grad, 1, want_dx, want_dw):
            if got is not None:
                rows = got if got.shape[0] == v else got[y >= 0]
                assert bool((rows.isnan() if mark else rows.isfinite()).all())
