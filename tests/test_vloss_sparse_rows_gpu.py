"""Logits whose sums are exact, or of one sign: what is put back for the tensor cores' cuts is a mean, and bounded."""
import pytest
import torch

from tests.test_vloss_gpu import BF, HF, SF
from trimkv_b200 import linear_cross_entropy

pytestmark = pytest.mark.gpu


def _loss_is_the_logit(x, w):
    """Two words, the label's all zeros: loss = log(exp(s) + 1), and what that is in 64 bits."""
    y = torch.ones(x.shape[0], dtype=torch.int64, device="cuda")
    both = torch.stack([w, torch.zeros_like(w)])
    return linear_cross_entropy(x, both, y, reduction="none").double(), torch.logsumexp(x.double() @ both.double().t(), 1)


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("t", [3, 64])
@pytest.mark.parametrize("h", [64, 1024, 4096])
@pytest.mark.parametrize("elements", [1, 8])
def test_rows_with_few_elements(dtype, t, h, elements):
    g = torch.Generator(device="cuda").manual_seed(h + t)
    x = torch.zeros(t, h, device="cuda")
    at = torch.rand(t, h, generator=g, device="cuda").argsort(1)[:, :elements]
    x.scatter_(1, at, 4 + 4 * torch.rand(t, elements, generator=g, device="cuda"))
    w = 0.5 + torch.rand(h, generator=g, device="cuda")
    got, want = _loss_is_the_logit(x.to(dtype), w.to(dtype))
    # at most 16 stages' mean cut put back, 4 additions each, 2^-24 / (4 ln 2) of the logit; then the few roundings of an fp32 loss: the logit, its
    # difference from the maximum, the sum and its logarithm, and (fp32) parts of a product that are left out
    put_back = 64 * 0.36067376 * 2.0 ** -24
    assert bool(((got - want).abs() <= (put_back + 6 * 2.0 ** -24) * want).all())


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("h", [64, 1024, 4096])
def test_rows_of_one_sign(dtype, h):
    g = torch.Generator(device="cuda").manual_seed(h)
    x = 0.5 + torch.rand(64, h, generator=g, device="cuda")
    w = (0.5 + torch.rand(h, generator=g, device="cuda")) * (40 / h)
    got, want = _loss_is_the_logit(x.to(dtype), w.to(dtype))
    # 16 stages of 4 products of 16, groups of four of which may be cut by 2^-23 of the sum; sums of them added in fp32
    assert bool(((got - want).abs() <= (256 * 2.0 ** -23 + h / 1024 * 2.0 ** -24 + 6 * 2.0 ** -24) * want).all())
