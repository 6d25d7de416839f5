"""apply_rotary (csrc/tkv_rotary.cu) against the formula in 64 bits: layouts, parts of heads, types, strides, positions, gradients."""
import math

import pytest
import torch

from trimkv_b200 import apply_rotary

pytestmark = pytest.mark.gpu


def _table(pairs, base=500000.0):
    f = base ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1))
    hi = f.float()
    return torch.stack([hi, (f - hi.double()).float()], 1).cuda()


def _want(x, positions, freq, layout, scale, back=False):
    """The turned values in 64 bits, and |a| + |b| of the pair (what errors of sine and cosine are multiplied with)."""
    x = x.double()
    n = freq.shape[0]
    angle = positions.double()[:, None, :, None] * freq.double().sum(1)
    c, s = angle.cos() * scale, angle.sin() * scale * (-1 if back else 1)
    y, size = x.clone(), torch.zeros_like(x)
    at = (slice(0, n), slice(n, 2 * n)) if layout == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    a, b = x[..., at[0]], x[..., at[1]]
    y[..., at[0]], y[..., at[1]] = a * c - b * s, b * c + a * s
    size[..., at[0]] = size[..., at[1]] = (a.abs() + b.abs()) * scale
    return y, size


def _close(got, want, size):
    # The part of a turn is rounded to fp32 (at most 2^-26 of a turn: 2 pi 2^-26 < 2^-23 in the angle), sine and cosine are good to 2 units
    # (2^-23 below 1), products and sum round thrice (3 2^-24): below 2^-21 of |a| + |b|.  Then one rounding to the type, or its smallest step.
    tol = size * 2.0 ** -21 + want.abs() * (torch.finfo(got.dtype).eps / 2) * 1.001 + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    assert got.shape == want.shape
    assert bool(((got.double() - want).abs() <= tol).all()), float(((got.double() - want).abs() - tol).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "pairs"])
@pytest.mark.parametrize("dim,pairs", [(128, 64), (128, 32), (96, 12), (80, 40), (80, 10), (64, 8), (66, 33), (7, 3), (2, 1), (64, 0), (256, 128)])
def test_sizes(dtype, layout, dim, pairs):
    g = torch.Generator(device="cuda").manual_seed(dim * 1000 + pairs)
    for b, hq, hkv, s in ((1, 1, 1, 1), (3, 4, 2, 5), (2, 5, 1, 301)):
        q, k = (torch.randn(b, s, h, dim, generator=g, device="cuda").to(dtype).transpose(1, 2) for h in (hq, hkv))
        pos = torch.randint(0, 100000, (b, s), generator=g, device="cuda")
        freq = _table(pairs)
        q2, k2 = apply_rotary(q, k, pos, freq, layout=layout, scale=1.25)
        assert q2.dtype == k2.dtype == dtype
        for got, x in ((q2, q), (k2, k)):
            _close(got, *_want(x, pos, freq, layout, 1.25))
            assert torch.equal(got[..., 2 * pairs:], x[..., 2 * pairs:])           # the rest is copied
            assert got.transpose(1, 2).is_contiguous()


@pytest.mark.parametrize("tokens", [148 * 16 - 1, 148 * 16, 148 * 32 + 3])
def test_several_tokens_per_cta(tokens):
    x = torch.randn(1, tokens, 3, 64, device="cuda").bfloat16().transpose(1, 2)
    pos, freq = torch.arange(tokens, device="cuda"), _table(16)
    for layout in ("half", "pairs"):
        got, none = apply_rotary(x, None, pos, freq, layout=layout)
        assert none is None
        _close(got, *_want(x, pos[None], freq, layout, 1.0))


def test_far_positions():
    """Positions far beyond fp32's whole numbers; the oracle's 64-bit product is exact to 2^-53 of an angle of at most 2^40 (2^-13),
    so frequencies are powers of two here, whose products are exact."""
    pos = torch.tensor([0, 1, 2 ** 24 + 1, 2 ** 31 - 1, 2 ** 31 + 7, 2 ** 40 + 3, -5, -(2 ** 33) - 1], device="cuda")
    f = torch.tensor([1.0, 0.5, 2.0 ** -10, 2.0 ** -20], device="cuda")
    freq = torch.stack([f, torch.zeros_like(f)], 1).contiguous()
    x = torch.randn(1, 2, 8, 8, device="cuda")
    got, _ = apply_rotary(x, None, pos, freq)
    # 64-bit reduction: position * f in turns is rounded to 2^-53 of up to 2^38 turns
    y, size = _want(x, pos[None], freq, "half", 1.0)
    off = (pos.double().abs() * 2.0 ** -52 * 2 * math.pi)[None, None, :, None]
    assert bool(((got.double() - y).abs() <= size * (2.0 ** -21 + off) + y.abs() * 2.0 ** -24).all())


@pytest.mark.parametrize("kind", ["int32", "one row", "flat", "strided", "expanded"])
def test_positions_forms(kind):
    b, s = 3, 17
    pos = torch.randint(0, 5000, (b, s), device="cuda")
    if kind in ("one row", "flat", "expanded"):
        pos = pos[:1].expand(b, s)
    given = {"int32": lambda: pos.int(), "one row": lambda: pos[:1], "flat": lambda: pos[0], "expanded": lambda: pos,
             "strided": lambda: torch.stack([pos, pos * 0], -1)[..., 0]}[kind]()
    q, k = torch.randn(b, 4, s, 32, device="cuda"), torch.randn(b, 2, s, 32, device="cuda")
    for got, x in zip(apply_rotary(q, k, given, _table(16)), (q, k)):
        _close(got, *_want(x, pos, _table(16), "half", 1.0))


def test_strides():
    """Slices of a fused projection (every alignment), heads first, a broadcast head, and elements that are not consecutive."""
    b, s, d = 2, 9, 32
    freq, pos = _table(16), torch.arange(9, device="cuda")
    for dtype in (torch.bfloat16, torch.float32):
        for shift in (0, 1, 2, 4, 8):
            u = torch.randn(b, s, 3 * d + shift, device="cuda").to(dtype)
            q = u[..., shift:shift + 2 * d].unflatten(-1, (2, d)).transpose(1, 2)
            k = u[..., shift + 2 * d:].unflatten(-1, (1, d)).transpose(1, 2)
            for got, x in zip(apply_rotary(q, k, pos, freq), (q, k)):
                _close(got, *_want(x, pos[None].expand(b, s), freq, "half", 1.0))
    heads_first = torch.randn(b, 3, s, d, device="cuda")
    shared = torch.randn(b, 1, s, d, device="cuda").expand(b, 4, s, d)
    apart = torch.randn(b, 2, s, 2 * d, device="cuda")[..., ::2]
    for x in (heads_first, shared, apart, torch.randn(b, s, d, 2, device="cuda").permute(0, 3, 1, 2)):
        got, _ = apply_rotary(x, None, pos, freq, layout="pairs")
        _close(got, *_want(x, pos[None].expand(b, s), freq, "pairs", 1.0))


def test_nothing_to_do():
    freq = _table(4)
    for q in (torch.zeros(0, 2, 3, 8), torch.zeros(2, 2, 0, 8), torch.zeros(2, 0, 3, 8)):
        q = q.cuda()
        got, _ = apply_rotary(q, None, torch.zeros(q.shape[2], dtype=torch.int64, device="cuda"), freq)
        assert got.shape == q.shape


def test_input_is_left_and_values_pass():
    """The inputs keep their values; infinities and NaN stay within their pair and the copied part."""
    x = torch.randn(1, 1, 2, 16, device="cuda")
    x[0, 0, 0, 3], x[0, 0, 1, 15] = float("nan"), float("inf")
    keep = x.clone()
    got, _ = apply_rotary(x, None, torch.arange(2, device="cuda"), _table(4))
    assert torch.equal(x.nan_to_num(), keep.nan_to_num())
    bad = ~torch.isfinite(got)
    want = torch.zeros_like(bad)
    want[0, 0, 0, 3] = want[0, 0, 0, 7] = want[0, 0, 1, 15] = True
    assert torch.equal(bad, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout,dim,pairs", [("half", 64, 32), ("half", 48, 12), ("pairs", 64, 32), ("pairs", 20, 5)])
def test_gradient_is_the_turn_back(dtype, layout, dim, pairs):
    b, s = 2, 33
    q = torch.randn(b, 4, s, dim, device="cuda").to(dtype).requires_grad_()
    k = torch.randn(b, 1, s, dim, device="cuda").to(dtype).requires_grad_()
    pos, freq = torch.randint(0, 9999, (b, s), device="cuda"), _table(pairs)
    q2, k2 = apply_rotary(q, k.expand(b, 2, s, dim), pos, freq, layout=layout, scale=0.75)
    gq, gk = torch.randn_like(q2), torch.randn_like(k2)
    dq, dk = torch.autograd.grad((q2, k2), (q, k), (gq, gk))
    _close(dq, *_want(gq, pos, freq, layout, 0.75, back=True))
    # the keys' gradient is the sum over the heads that share them, rounded as the two parts are and once more
    parts, size = _want(gk, pos, freq, layout, 0.75, back=True)
    half = torch.finfo(dtype).eps / 2
    want, each = parts.sum(1, keepdim=True), parts.abs().sum(1, keepdim=True)
    assert bool(((dk.double() - want).abs() <= size.sum(1, keepdim=True) * 2.0 ** -21 + each * 2.01 * half + want.abs() * half * 1.01 + 1e-7).all())


def test_gradients_asked_of_one_side_only():
    q, k = (torch.randn(1, 2, 5, 16, device="cuda") for _ in range(2))
    pos, freq = torch.arange(5, device="cuda"), _table(8)
    k.requires_grad_()
    q2, k2 = apply_rotary(q, k, pos, freq)
    assert torch.autograd.grad(k2.sum(), k)[0].shape == k.shape
    q.requires_grad_()
    q2, k2 = apply_rotary(q, k, pos, freq)
    dq, = torch.autograd.grad(q2[..., 3].sum(), q)                 # a gradient with strides of its own, the keys' left out
    want, size = _want(torch.zeros_like(q).index_fill(3, torch.tensor([3], device="cuda"), 1.0), pos[None], freq, "half", 1.0, back=True)
    _close(dq, want, size)
    with torch.no_grad():
        assert not apply_rotary(q, k, pos, freq)[0].requires_grad


def test_gradient_against_differences():
    q = torch.randn(1, 2, 3, 12, device="cuda", requires_grad=True)
    pos, freq, w = torch.tensor([3, 70, 900], device="cuda"), _table(4), torch.randn(1, 2, 3, 12, device="cuda")
    f = lambda x: float((apply_rotary(x, None, pos, freq, scale=1.5)[0].double() * w.double()).sum())  # noqa: E731
    d, = torch.autograd.grad((apply_rotary(q, None, pos, freq, scale=1.5)[0] * w).sum(), q)
    for i in range(0, q.numel(), 5):
        step = torch.zeros(q.numel(), device="cuda")
        step[i] = 0.5
        step = step.view_as(q)
        with torch.no_grad():
            slope = f(q + step) - f(q - step)                      # linear: differences over a whole 1.0 are exact but for fp32 roundings
        assert abs(slope - float(d.flatten()[i])) <= 72 * 4 * 2.0 ** -22


def test_captured_and_replayed_with_other_inputs():
    q, k = torch.randn(2, 4, 1, 64, device="cuda").bfloat16(), torch.randn(2, 2, 1, 64, device="cuda").bfloat16()
    pos, freq = torch.tensor([[3], [4]], device="cuda"), _table(32)
    apply_rotary(q, k, pos, freq)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q2, k2 = apply_rotary(q, k, pos, freq)
    for i in range(3):
        q.normal_(); k.normal_(); pos.add_(1000 * i)
        graph.replay()
        torch.cuda.synchronize()
        for got, x in ((q2, q), (k2, k)):
            _close(got, *_want(x, pos, freq, "half", 1.0))


def test_another_stream():
    side = torch.cuda.Stream()
    q, pos, freq = torch.randn(1, 8, 2048, 128, device="cuda").bfloat16(), torch.arange(2048, device="cuda"), _table(64)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = apply_rotary(q * 1, None, pos, freq)
    torch.cuda.current_stream().wait_stream(side)
    _close(got, *_want(q, pos[None], freq, "half", 1.0))


def test_gradient_of_the_gradient():
    q = torch.randn(1, 2, 4, 16, device="cuda", requires_grad=True)
    pos, freq, g = torch.arange(4, device="cuda"), _table(8), torch.randn(1, 2, 4, 16, device="cuda", requires_grad=True)
    d, = torch.autograd.grad(apply_rotary(q, None, pos, freq, scale=0.5)[0], q, g, create_graph=True)
    v = torch.randn_like(q)
    back, = torch.autograd.grad(d, g, v)                            # of a linear map: the map itself
    _close(back, *_want(v, pos[None], freq, "half", 0.5))


def test_offsets_beyond_32_bits():
    """More than 2^31 elements of queries: tokens on either side of the border, and the last."""
    heads, dim, tokens = 64, 256, 131072 + 50                          # 2^17 tokens are 2^31 elements
    q = torch.empty(1, tokens, heads, dim, device="cuda", dtype=torch.bfloat16).normal_().transpose(1, 2)
    pos, freq = torch.arange(tokens, device="cuda"), _table(64)
    got, _ = apply_rotary(q, None, pos, freq)
    for s in (slice(0, 3), slice(131072 - 3, 131072 + 3), slice(tokens - 2, tokens)):
        _close(got[:, :, s], *_want(q[:, :, s], pos[None, s], freq, "half", 1.0))
