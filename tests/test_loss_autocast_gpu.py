"""linear_cross_entropy under autocast: operands in its type, gradients in their own, as the product of the logits has it."""
import pytest
import torch

from tests.test_loss_heads import _model
from trimkv_b200 import linear_cross_entropy

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cast", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dx,dw", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float32, torch.float16)])
def test_types(cast, dx, dw):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(50, 72, generator=g, device="cuda").to(dx).requires_grad_()
    w = torch.randn(300, 72, generator=g, device="cuda").mul(0.2).to(dw).requires_grad_()
    y = torch.randint(0, 300, (50,), generator=g, device="cuda")
    with torch.autocast("cuda", cast):
        loss = linear_cross_entropy(x, w, y)
    got = torch.autograd.grad(loss, (x, w))
    a, b = x.detach().to(cast).requires_grad_(), w.detach().to(cast).requires_grad_()
    want = linear_cross_entropy(a, b, y)
    assert torch.equal(loss, want)
    for p, q, t in zip(got, torch.autograd.grad(want, (a, b)), (dx, dw)):
        assert p.dtype == t and torch.equal(p, q.to(t))
    if dx != dw:                                                   # and nothing is cast without it
        with pytest.raises(TypeError):
            linear_cross_entropy(x, w, y)
    with torch.autocast("cuda", cast, enabled=False), torch.no_grad():
        assert dx != dw or not torch.equal(linear_cross_entropy(x, w, y), want)


def test_a_decoder_under_autocast():
    """fp32 parameters: the loss is that of the product in bf16, whose logits the same call returns rounded to bf16 (2^-8 of numbers below 2^3)."""
    model = _model().cuda()
    ids = torch.randint(1, 131, (2, 17), generator=torch.Generator().manual_seed(5)).cuda()
    with torch.autocast("cuda", torch.bfloat16):
        out = model(input_ids=ids, labels=ids)
    z = out.logits.detach().double()[:, :-1].flatten(0, 1)
    assert out.loss.dtype == torch.float32
    assert abs(float(out.loss.detach()) - float(torch.nn.functional.cross_entropy(z, ids[:, 1:].flatten()))) <= 2 * 2.0 ** -8 * 8
    out.loss.backward()
    assert all(p.grad is None or (p.grad.dtype == torch.float32 and bool(p.grad.isfinite().all())) for p in model.parameters())
    assert model.lm_head.weight.grad is not None
