"""Gradients of the weight over very many tokens, all of whose products have one sign: what the tensor cores cut from a sum does not add up."""
import pytest
import torch

from trimkv_b200 import linear_cross_entropy

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [1 << 15, (1 << 21) - 77])
def test_sums_of_one_sign(t):
    v, h, dtype = 64, 64, torch.float16
    g = torch.Generator(device="cuda").manual_seed(t)
    x = (0.5 + 0.5 * torch.rand(t, h, generator=g, device="cuda")).to(dtype)
    w = (0.05 * torch.randn(v, h, generator=g, device="cuda")).to(dtype).requires_grad_()
    y = torch.zeros(t, dtype=torch.int64, device="cuda")
    dw, = torch.autograd.grad(linear_cross_entropy(x, w, y, reduction="sum"), w, torch.tensor(64.0 / t, device="cuda"))
    p = torch.softmax(x.double() @ w.detach().double().t(), 1)
    want = (64.0 / t) * (p.t() @ x.double())[1:]                 # of the words that are no label: sums of positive products
    half = 2.0 ** -11
    # dL and dw are rounded to fp16; a sum in TMEM takes 16 products a time, 4 times in each of up to 64 stages, and may cut every group of four of
    # them by 2^-23 of itself; the sums are added in fp32; p is off by what a logit below 2^2 is, 64 products of 2^-23, and a few roundings of
    # its exponent
    cut = 64 * 4 * 4 * 2.0 ** -23 + t / 4096 * 2.0 ** -24
    off = (dw[1:].double() - want).abs() / want
    assert float(off.max()) <= 2 * half * 1.01 + cut + 2 * (64 * 2.0 ** -23 * 4 + 2.0 ** -20)
    # roundings of many entries go either way: the mean over all words and columns keeps only what goes one way, of 4032 roundings 2^-11 / 60
    assert abs(float(((dw[1:].double() - want) / want).mean())) <= half / 16 + cut
