"""apply_rotary in forward mode: tangents are turned like what they belong to, whether or not the other input has one."""
import pytest
import torch
from torch.autograd import forward_ad

from trimkv_b200 import apply_rotary, ops
from trimkv_b200.positions import split_frequencies


def _plain(x, positions, freq, layout, inverse, scale):
    """[B, H, S, D] in 64 bits."""
    angle = positions.double()[:, None, :, None] * freq.double().sum(1) * (-1.0 if inverse else 1.0)
    n, y = freq.shape[0], x.double().clone()
    at = (slice(0, n), slice(n, 2 * n)) if layout == 0 else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    a, b = x.double()[..., at[0]], x.double()[..., at[1]]
    y[..., at[0]] = scale * (a * angle.cos() - b * angle.sin())
    y[..., at[1]] = scale * (b * angle.cos() + a * angle.sin())
    return y


def _stand_in(q, k, positions, freq, layout, inverse, scale):
    """As a kernel: it sees numbers, no tangents and no graph."""
    return tuple(None if x is None else _plain(forward_ad.unpack_dual(x).primal.detach(), positions, freq, layout, inverse, scale).to(x.dtype)
                 for x in (q, k))


def _case(device, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k, tq, tk = (torch.randn(2, h, 5, 12, generator=g).to(device, dtype) for h in (3, 2, 3, 2))
    positions = torch.randint(0, 5000, (2, 5), generator=g).to(device)
    return q, k, tq, tk, positions, split_frequencies(1e4 ** (-torch.arange(4, dtype=torch.float64) / 4)).to(device)


def _check(device, dtype, tol):
    for layout, name in enumerate(("half", "pairs")):
        q, k, tq, tk, positions, freq = _case(device, dtype)
        want_q, want_k = (_plain(t, positions, freq, layout, False, 1.3) for t in (tq, tk))
        for with_q, with_k in ((True, True), (True, False), (False, True)):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), forward_ad.dual_level():
                    a = forward_ad.make_dual(q, tq) if with_q else q
                    b = forward_ad.make_dual(k, tk) if with_k else k
                    out = [forward_ad.unpack_dual(t) for t in apply_rotary(a, b, positions, freq, layout=name, scale=1.3)]
                for had, got, want, x in ((with_q, out[0], want_q, q), (with_k, out[1], want_k, k)):
                    assert bool(((got.primal.double() - _plain(x, positions, freq, layout, False, 1.3)).abs() <= tol).all())
                    if had:
                        assert bool(((got.tangent.double() - want).abs() <= tol).all())
                    else:
                        assert got.tangent is None or not bool(got.tangent.any())
        with forward_ad.dual_level():                                  # queries alone
            got, none = apply_rotary(forward_ad.make_dual(q, tq), None, positions, freq, layout=name, scale=1.3)
            assert none is None and bool(((forward_ad.unpack_dual(got).tangent.double() - want_q).abs() <= tol).all())
        # a gradient through a tangent, and tangents of what has a gradient
        q, tq = q.requires_grad_(), tq.requires_grad_()
        with forward_ad.dual_level():
            got = forward_ad.unpack_dual(apply_rotary(forward_ad.make_dual(q, tq), k, positions, freq, layout=name, scale=1.3)[0])
            up = torch.ones_like(got.tangent)
            back = torch.autograd.grad(got.tangent, tq, up)[0]
        assert bool(((back.double() - _plain(up, positions, freq, layout, True, 1.3)).abs() <= tol).all())


def test_tangents_are_turned(monkeypatch):
    """The operator's own path, the kernel replaced by the formula."""
    monkeypatch.setattr(ops, "rotary", _stand_in)
    _check("cpu", torch.float32, 8 * 2.0 ** -21)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tangents_are_turned_by_the_kernel(dtype):
    # numbers below 8: angles to 2^-21, a product and a sum in fp32, one rounding
    _check("cuda", dtype, 8 * (2.0 ** -21 + torch.finfo(dtype).eps / 2))
