"""expert_balance (csrc/tkv_moe_balance.cu) against the formula in 64 bits."""
import pytest
import torch

from trimkv_b200 import expert_balance

pytestmark = pytest.mark.gpu


def _want(z, choice, valid):
    z = z.detach().double()
    live = torch.ones(z.shape[0], dtype=torch.bool, device=z.device) if valid is None else valid
    E, n, k = z.shape[1], int(live.sum()), choice.shape[1]
    picked = choice[live].long()
    picked = picked[(picked >= 0) & (picked < E)]
    counts = torch.bincount(picked, minlength=E)
    f = counts.double() / max(1, n * k)
    p = torch.softmax(z[live], 1)
    loss = E * (f * p.sum(0) / max(1, n)).sum()
    dz = torch.zeros_like(z)
    dz[live] = E / max(1, n) * p * (f - (p * f).sum(1, keepdim=True))
    return loss, counts.int(), dz


def _check(z, choice, valid=None, grad=1.0):
    z = z.requires_grad_()
    loss, counts = expert_balance(z, choice, valid)
    assert loss.dtype == torch.float32 and loss.shape == () and counts.dtype == torch.int32
    dz, = torch.autograd.grad(loss, z, torch.tensor(grad, device="cuda"))
    want, hits, dwant = _want(z.reshape(-1, z.shape[-1]), choice.reshape(-1, choice.shape[-1]), None if valid is None else valid.reshape(-1))
    E = z.shape[-1]
    assert torch.equal(counts, hits)
    # p = exp(z - max) / sum: an argument rounded to 2^-24 of |z - max| <= 40, an exponential and a division of 2 units each, a sum of E
    # positive numbers in fp32 (log2 E + E / 32 roundings): below rel = 2^-24 (40 + 8 + 48); sums over a warp's tokens likewise.
    rel = 2.0 ** -24 * (96 + z.numel() // E // 16)
    assert abs(float(loss.detach()) - float(want)) <= float(want) * rel + 1e-12
    f_most = float(hits.double().max()) / max(1, choice.numel())
    n = int(valid.sum()) if valid is not None else z.numel() // E
    size = E / max(1, n) * abs(grad) * torch.softmax(z.detach().double(), -1) * max(f_most, 0) * 2
    scale = float(choice.numel()) / max(1, n * choice.shape[-1])               # f counts valid tokens only
    tol = size * scale * rel + dwant.view_as(z).abs() * abs(grad) * torch.finfo(z.dtype).eps * 0.51 + torch.finfo(z.dtype).smallest_normal
    assert dz.dtype == z.dtype
    assert bool(((dz.double() - dwant.view_as(z) * grad).abs() <= tol).all())


@pytest.mark.parametrize("tokens", [1, 31, 32, 33, 65, 1000, 6000])
@pytest.mark.parametrize("experts,top", [(1, 1), (8, 2), (31, 3), (33, 6), (60, 4), (128, 8), (160, 6), (257, 40), (1024, 64)])
def test_sizes(tokens, experts, top):
    g = torch.Generator(device="cuda").manual_seed(tokens * 2000 + experts)
    z = 3 * torch.randn(tokens, experts, generator=g, device="cuda")
    choice = z.topk(min(top, experts), 1).indices
    _check(z, choice.int(), grad=0.5)
    _check(z.detach(), choice, torch.rand(tokens, generator=g, device="cuda") < 0.7)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_types_and_shapes(dtype):
    z = (2 * torch.randn(3, 50, 40, device="cuda")).to(dtype)
    _check(z, torch.randint(0, 40, (3, 50, 4), device="cuda"), torch.rand(3, 50, device="cuda") < 0.5)


def test_strides():
    wide = torch.randn(100, 80, device="cuda")
    _check(wide[:, 8:40], torch.randint(0, 32, (100, 9), device="cuda")[:, 3:6])
    _check(wide.t()[:, ::2], torch.randint(0, 50, (4, 80), device="cuda").t(), (torch.rand(80, 2, device="cuda") < 0.5)[:, 1])


def test_masked_rows_are_not_read_and_no_tokens():
    z = torch.randn(64, 16, device="cuda")
    valid = torch.arange(64, device="cuda") % 3 > 0
    choice = torch.randint(0, 16, (64, 2), device="cuda")
    clean = expert_balance(z, choice, valid)
    z[~valid], choice[~valid] = float("nan"), -7
    dirty = expert_balance(z.requires_grad_(), choice, valid)
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])
    assert not bool(torch.autograd.grad(dirty[0], z)[0].isnan().any())
    loss, counts = expert_balance(z, choice, torch.zeros_like(valid))
    assert float(loss.detach()) == 0.0 and not bool(counts.any())
    assert not bool(torch.autograd.grad(loss, z)[0].any())
    loss, counts = expert_balance(z[:0], choice[:0])
    assert float(loss.detach()) == 0.0 and counts.shape == (16,) and not bool(counts.any())
    assert torch.autograd.grad(loss, z)[0].shape == z.shape


def test_choices_outside_and_twice():
    z = torch.randn(40, 8, device="cuda")
    choice = torch.randint(-3, 12, (40, 5), device="cuda")
    choice[:, 1] = choice[:, 0]
    _check(z, choice)
    _check(z.detach(), choice.int() * 0 + 3)


def test_even_use_is_one_and_equal_inputs_give_equal_bits():
    z = torch.zeros(4096, 64, device="cuda")
    choice = (torch.arange(4096 * 2, device="cuda") % 64).view(4096, 2)
    loss, counts = expert_balance(z, choice)
    assert abs(float(loss.detach()) - 1.0) <= 2.0 ** -20 and bool((counts == 128).all())
    z = torch.randn(30000, 128, device="cuda", requires_grad=True)
    choice = z.topk(8, 1).indices
    first = expert_balance(z, choice)
    g = torch.autograd.grad(first[0], z)[0]
    for _ in range(3):
        again = expert_balance(z, choice)
        assert torch.equal(first[0], again[0]) and torch.equal(g, torch.autograd.grad(again[0], z)[0])


def test_gradient_against_differences():
    z = torch.randn(6, 5, device="cuda", requires_grad=True)
    choice = torch.randint(0, 5, (6, 2), device="cuda")
    d, = torch.autograd.grad(expert_balance(z, choice)[0], z)
    h = 2.0 ** -5
    for i in range(z.numel()):
        step = torch.zeros(z.numel(), device="cuda")
        step[i] = h
        with torch.no_grad():
            up, down = (float(expert_balance(z + s * step.view_as(z), choice)[0]) for s in (1, -1))
        # third derivatives of the loss are below 5 / 6 (p and f at most 1): h^2 of error, and two roundings of a loss below 5 over 2 h
        assert abs((up - down) / (2 * h) - float(d.flatten()[i])) <= h * h + 2 * 5 * 2.0 ** -22 / (2 * h)


def test_captured_and_replayed():
    z, choice = torch.randn(500, 32, device="cuda"), torch.randint(0, 32, (500, 4), device="cuda")
    expert_balance(z, choice)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, counts = expert_balance(z, choice)
    for _ in range(3):
        z.normal_(); choice.random_(0, 32)
        graph.replay()
        want, hits, _ = _want(z, choice, None)
        assert torch.equal(counts, hits) and abs(float(loss.detach()) - float(want)) <= float(want) * 2.0 ** -16
