"""linear_cross_entropy refuses status words that a kernel could not write."""
import pytest
import torch

from trimkv_b200 import _lib, linear_cross_entropy, ops


def _call(status, device="cpu"):
    x, w = torch.zeros(3, 8, device=device), torch.zeros(5, 8, device=device)
    return linear_cross_entropy(x, w, torch.zeros(3, dtype=torch.int64, device=device), status=status)


@pytest.mark.parametrize("status", [torch.zeros(1, dtype=torch.int64), torch.zeros(1), torch.zeros(0, dtype=torch.int32),
                                    torch.zeros(1, dtype=torch.int32, device="meta")])
def test_refused(status):
    with pytest.raises(ValueError):
        _call(status)


def test_a_status_beside_the_rows_passes():
    with pytest.raises(_lib.TrimKVNativeError):                # as far as the CPU goes
        _call(ops.new_status("cpu"))


@pytest.mark.gpu
def test_a_status_on_the_cpu_is_refused():
    with pytest.raises(ValueError):
        _call(ops.new_status("cpu"), "cuda")
    status = ops.new_status("cuda")
    assert bool(_call(status, "cuda").isfinite()) and ops.read_status(status) == 0
