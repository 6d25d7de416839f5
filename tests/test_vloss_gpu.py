"""linear_cross_entropy (csrc/tkv_vloss*.cu) against the formula in 64 bits: sizes around the tiles, types, ignored tokens, strides,
reductions, gradients."""
import pytest
import torch
import torch.nn.functional as F

from trimkv_b200 import linear_cross_entropy, ops

pytestmark = pytest.mark.gpu

BF, HF, SF = torch.bfloat16, torch.float16, torch.float32


def _inputs(t, v, h, dtype, keep=1.0, seed=0, sharp=True):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + t * 31 + v)
    w = (torch.randn(v, h, generator=g, device="cuda") * h ** -0.5).to(dtype)
    x = torch.randn(t, h, generator=g, device="cuda")
    y = torch.randint(0, v, (t,), generator=g, device="cuda")
    if sharp:                                                    # some tokens nearly certain of their label
        x += 8 * torch.rand(t, 1, generator=g, device="cuda") ** 3 * w[y].float()
    live = torch.rand(t, generator=g, device="cuda") < keep
    return x.to(dtype), w, torch.where(live, y, torch.full_like(y, -100))


def _want(x, w, y, grad):
    """Losses, gradients and, for the tolerances, |dL| |w| and |dL| |x| in 64 bits; grad [T] of every token's loss."""
    x, w, live = x.detach().double(), w.detach().double(), y >= 0
    at = y.clamp_min(0)
    logp = torch.log_softmax(x @ w.t(), 1)
    loss = torch.where(live, -logp.gather(1, at[:, None])[:, 0], 0.0)
    d = logp.exp()
    p = d.clone()
    d.scatter_add_(1, at[:, None], -torch.ones_like(d[:, :1]))
    g = (grad.double() * live)[:, None]
    d, size = d * g, (p * g.abs())                               # errors of a logit act on p, not on p - 1
    return loss, d @ w, d.t() @ x, (d.abs() @ w.abs(), d.abs().t() @ x.abs()), (size @ w.abs(), size.t() @ x.abs())


def _within(got, want, tol):
    """Off by at most tol.  Rounding to nearest turns what is beyond the largest number and half its unit into an infinity (fp16: beyond
    65504 + 16), so an infinity is right where the formula's value, tol further out, is beyond that."""
    top = torch.finfo(got.dtype).max
    border = top * (1 + torch.finfo(got.dtype).eps / 4)
    beyond = got.isinf() & (want.abs() + tol >= border) & (got.sign() == want.sign())
    return bool((((got.double() - want).abs() <= tol) | beyond).all())


def _check(x, w, y, reduction="none", grad=None):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    t, h, v = x.shape[0], x.shape[1], w.shape[0]
    n = int((y >= 0).sum())
    loss = linear_cross_entropy(x, w, y, reduction=reduction)
    assert loss.dtype == torch.float32
    if grad is None:
        grad = torch.randn(t, device="cuda") if reduction == "none" else torch.tensor(0.7, device="cuda")
    dx, dw = torch.autograd.grad(loss, (x, w), grad)
    each = grad if reduction == "none" else grad.expand(t) / (max(n, 1) if reduction == "mean" else 1)
    want, ex, ew, (mx, mw), (px, pw) = _want(x, w, y, each)
    half = torch.finfo(x.dtype).eps / 2
    # A logit is h products added in fp32 in some order (an accumulator may cut instead of rounding): h 2^-23 of the sum of |x w|.
    logit = h * 2.0 ** -23 * float((x.detach().double().abs() @ w.detach().double().abs().t()).max()) if t else 0.0
    # Base-2 exponents, their sum over v, the logarithm: roundings of numbers up to |lse| log2(e), 2^-23 each, a few of them.
    soft = 2 * logit + 2.0 ** -20 * (2 + float(want.max()) if t else 0)
    if reduction == "none":
        assert loss.shape == y.shape
        assert bool(((loss.double() - want).abs() <= soft).all())
        assert not bool(loss[y < 0].any())
    elif n:
        total = want.sum() / (n if reduction == "mean" else 1)
        assert abs(float(loss.detach()) - float(total)) <= soft * (1 if reduction == "mean" else n) + abs(float(total)) * 2.0 ** -23
    # dL: p off by soft, then rounded to the inputs' type (fp32: kept), then sums of v or t products in fp32, then one rounding.
    kept = 0.0 if x.dtype == SF else half * 1.01
    tiny = torch.finfo(x.dtype).smallest_normal
    tol_x = px * (2 * soft) + mx * (kept + (v + h) * 2.0 ** -23) + ex.abs() * half * 1.01 + tiny
    tol_w = pw * (2 * soft) + mw * (kept + (t + h) * 2.0 ** -23) + ew.abs() * half * 1.01 + tiny
    # fp16: what dL loses below its smallest normal number, 2^-25 beside a largest of at least 2^13
    if x.dtype == HF and t:
        lost = 2.0 ** -38 * float(each.abs().max())
        tol_x = tol_x + lost * w.detach().double().abs().sum(0)
        tol_w = tol_w + lost * x.detach().double()[y >= 0].abs().sum(0)
    # A weight exp(s - lse) below 2^-126, the smallest normal fp32 number, may be taken as 0 (and the smaller parts that an fp32 number of
    # that size is made of): dL is then off by at most 2 * 2^-126 of the row's gradient, a gradient by that times the sum of |w| or |x|.
    under = 2.0 ** -125 * each.double().abs() * (y >= 0)
    tol_x = tol_x + under[:, None] * w.detach().double().abs().sum(0)
    tol_w = tol_w + (under[:, None] * x.detach().double().abs()).sum(0)
    assert dx.dtype == x.dtype and dw.dtype == w.dtype
    assert _within(dx, ex, tol_x) and _within(dw, ew, tol_w)
    assert not bool(dx[y < 0].any())
    return loss, dx, dw


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("t", [1, 2, 127, 128, 129, 257])
@pytest.mark.parametrize("v,h", [(1, 8), (7, 64), (127, 72), (129, 128), (256, 64), (257, 200), (1000, 264), (4099, 136)])
def test_sizes(dtype, t, v, h):
    _check(*_inputs(t, v, h, dtype, keep=0.8))


@pytest.mark.parametrize("dtype", [BF, SF])
@pytest.mark.parametrize("h", [1, 3, 33, 100])
def test_odd_widths(dtype, h):
    _check(*_inputs(70, 300, h, dtype, keep=0.9))


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("keep", [1.0, 0.5, 0.02])
def test_reductions_and_ignored_tokens(dtype, reduction, keep):
    _check(*_inputs(600, 1500, 192, dtype, keep=keep, seed=3), reduction=reduction)


@pytest.mark.parametrize("dtype", [BF, HF, SF])
def test_pieces_of_the_vocabulary(dtype):
    """More vocabulary than a piece, and a last piece that is not whole."""
    _check(*_inputs(2100, 17003, 64, dtype, keep=0.95), reduction="mean")


def test_gradients_of_very_different_size():
    """Gradients of rows from 1e-6 to 1e6 times one another keep their digits in bf16; in fp16 as many as its range leaves."""
    for dtype in (BF, HF):
        x, w, y = _inputs(300, 900, 64, dtype)
        _check(x, w, y, grad=torch.exp2(torch.linspace(-20, 20, 300, device="cuda")))
        _check(x, w, y, grad=torch.zeros(300, device="cuda"))
        _check(x, w, y, reduction="sum", grad=torch.tensor(1e-30 if dtype == BF else 1e-2, device="cuda"))


@pytest.mark.parametrize("dtype", [BF, SF])
def test_nothing_of_ignored_tokens_gets_anywhere(dtype):
    x, w, y = _inputs(200, 700, 64, dtype, keep=0.6)
    first = _check(x, w, y, reduction="mean")
    x[y < 0] = float("nan")
    x, w = x.requires_grad_(), w.requires_grad_()
    loss = linear_cross_entropy(x, w, y)
    dx, dw = torch.autograd.grad(loss, (x, w), torch.tensor(0.7, device="cuda"))
    assert torch.equal(loss, first[0]) and torch.equal(dx, first[1]) and torch.equal(dw, first[2])


@pytest.mark.parametrize("dtype", [BF, SF])
def test_all_ignored_and_no_tokens(dtype):
    for t in (0, 1, 300):
        x, w, y = _inputs(t, 500, 64, dtype, keep=0.0)
        x, w = x.requires_grad_(), w.requires_grad_()
        for reduction in ("none", "sum", "mean"):
            loss = linear_cross_entropy(x, w, y, reduction=reduction)
            dx, dw = torch.autograd.grad(loss, (x, w), torch.ones_like(loss))
            assert not bool(dx.any()) and not bool(dw.any()) and dx.shape == x.shape
            assert bool(loss.isnan()) if reduction == "mean" else not bool(loss.any())


@pytest.mark.parametrize("dtype", [BF, SF])
def test_labels_outside_the_vocabulary(dtype):
    x, w, y = _inputs(130, 300, 64, dtype)
    y[5], y[77] = 300, -1
    status = ops.new_status("cuda")
    x, w = x.requires_grad_(), w.requires_grad_()
    loss = linear_cross_entropy(x, w, y, reduction="none", status=status)
    assert ops.read_status(status) == 3
    bad = torch.zeros(130, dtype=torch.bool, device="cuda")
    bad[5] = bad[77] = True
    assert torch.equal(loss.isnan(), bad)
    dx, dw = torch.autograd.grad(loss, (x, w), torch.ones(130, device="cuda"))
    assert not bool(dx[bad].any()) and bool(dw.isfinite().all())
    y[bad] = -100
    clean = linear_cross_entropy(x, w, y, reduction="none")
    assert torch.equal(clean[~bad], loss[~bad])
    assert torch.equal(torch.autograd.grad(clean, w, torch.ones(130, device="cuda"))[0], dw)
    assert bool(linear_cross_entropy(x, w, torch.where(bad, 999, y)).isnan())
    other = linear_cross_entropy(x, w, torch.where(bad, 7777, y), ignore_index=7777, reduction="none")
    assert torch.equal(other, clean)


@pytest.mark.parametrize("dtype", [BF, SF])
def test_strides_and_shapes(dtype):
    x, w, y = _inputs(120, 400, 64, dtype)
    wide = torch.zeros(120, 200, dtype=dtype, device="cuda")
    for shift in (0, 1, 8):                                       # rows apart, and off the 16-byte boundary
        wide[:, shift:shift + 64] = x
        _check(wide[:, shift:shift + 64], w, y)
    base = linear_cross_entropy(x, w, y, reduction="none")
    assert torch.equal(linear_cross_entropy(x.view(4, 30, 64), w, y.view(4, 30), reduction="none"), base.view(4, 30))
    assert torch.equal(linear_cross_entropy(x.t().contiguous().t(), w.t().contiguous().t(), y.int(), reduction="none"), base)
    assert torch.equal(linear_cross_entropy(x[7], w, y[7], reduction="none"), linear_cross_entropy(x[7:8], w, y[7:8], reduction="none")[0])
    same = x[:1].expand(50, 64)                                   # rows zero apart
    assert torch.equal(linear_cross_entropy(same, w, y[:1].expand(50), reduction="none"), linear_cross_entropy(same.contiguous(), w, y[:1].repeat(50), reduction="none"))


@pytest.mark.parametrize("dtype", [BF, SF])
def test_one_gradient_only(dtype):
    x, w, y = _inputs(150, 600, 64, dtype, keep=0.9)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    both = torch.autograd.grad(linear_cross_entropy(xg, wg, y), (xg, wg))
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(xg, w, y), xg)[0], both[0])
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(x, wg, y), wg)[0], both[1])
    expanded = torch.autograd.grad(linear_cross_entropy(xg, w, y, reduction="none").sum(), xg)[0]   # a gradient of stride 0
    assert torch.equal(expanded, torch.autograd.grad(linear_cross_entropy(xg, w, y, reduction="none"), xg, torch.ones(150, device="cuda"))[0])


def test_large_logits_and_certain_tokens():
    """Logits in the thousands (maxima are taken before exponents), and a token whose probability of its label is 1."""
    x, w, y = _inputs(64, 500, 64, SF)
    _check(x * 300, w, y)
    x = w[y] * 500
    loss = linear_cross_entropy(x, w, y, reduction="none")
    want = F.cross_entropy(x.double() @ w.double().t(), y, reduction="none")
    assert bool(((loss.double() - want).abs() <= 64 * 2.0 ** -23 * 500 * 4).all())


@pytest.mark.parametrize("dtype", [BF, SF])
def test_gradient_against_differences(dtype):
    x, w, y = _inputs(20, 90, 16, dtype, sharp=False)
    x, w = x.requires_grad_(), w.requires_grad_()
    dx, dw = torch.autograd.grad(linear_cross_entropy(x, w, y, reduction="sum"), (x, w))
    f = lambda a, b: float(F.cross_entropy(a.double() @ b.double().t(), y, reduction="sum"))  # noqa: E731
    half = torch.finfo(dtype).eps / 2
    h = 2.0 ** -8
    with torch.no_grad():
        for i in range(0, x.numel(), 37):
            step = torch.zeros(x.numel(), device="cuda", dtype=torch.float64)
            step[i] = h
            slope = (f(x.double() + step.view_as(x), w) - f(x.double() - step.view_as(x), w)) / (2 * h)
            size = float(w.double().abs()[:, i % 16].max()) * 2      # sum over v of |dL| is at most 2
            assert abs(slope - float(dx.flatten()[i])) <= size * (half * 1.02 + 2.0 ** -16) + abs(slope) * half + h * h * 10


def test_equal_inputs_give_equal_bits():
    x, w, y = _inputs(1000, 3000, 128, BF, keep=0.9)
    first = _check(x, w, y, grad=torch.ones(1000, device="cuda"))
    for _ in range(3):
        for a, b in zip(first, _check(x, w, y, grad=torch.ones(1000, device="cuda"))):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,t", [(BF, 3), (BF, 300), (SF, 40)])
def test_captured_and_replayed_with_other_inputs(dtype, t):
    """A training pass in a graph: other rows, another number of ignored tokens at every replay."""
    x, w, y = _inputs(t, 700, 64, dtype)
    x, w = x.requires_grad_(), w.requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(linear_cross_entropy(x, w, y), (x, w))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = linear_cross_entropy(x, w, y)
        dx, dw = torch.autograd.grad(loss, (x, w))
    for seed, keep in ((1, 1.0), (2, 0.3), (3, 0.9)):
        x2, w2, y2 = _inputs(t, 700, 64, dtype, keep=keep, seed=seed)
        y2[0] = 5
        with torch.no_grad():
            x.copy_(x2); w.copy_(w2); y.copy_(y2)
        graph.replay()
        torch.cuda.synchronize()
        eager = linear_cross_entropy(x, w, y)
        ex, ew = torch.autograd.grad(eager, (x, w))
        assert torch.equal(loss, eager) and torch.equal(dx, ex) and torch.equal(dw, ew)


def test_two_streams_at_once():
    a, b = (_inputs(500, 2000, 128, BF, seed=s) for s in (1, 2))
    want = [linear_cross_entropy(*z, reduction="none") for z in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, z in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i] = linear_cross_entropy(*z, reduction="none")
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_no_gradient_of_the_gradient():
    x, w, y = _inputs(10, 90, 16, SF)
    x.requires_grad_()
    dx, = torch.autograd.grad(linear_cross_entropy(x, w, y), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_offsets_beyond_32_bits():
    """More than 2^31 elements of weight (and of its gradient): what the last words and the first ones give."""
    v, h = 140000, 16384
    g = torch.Generator(device="cuda").manual_seed(0)
    w = torch.empty(v, h, device="cuda", dtype=BF).normal_(0, h ** -0.5, generator=g).requires_grad_()
    x = torch.randn(3, h, generator=g, device="cuda").to(BF).requires_grad_()
    y = torch.tensor([v - 1, 0, v - 77], device="cuda")
    loss = linear_cross_entropy(x, w, y, reduction="none")
    with torch.no_grad():
        s = torch.cat([x.double() @ w[i:i + 20000].double().t() for i in range(0, v, 20000)], 1)
        want = F.cross_entropy(s, y, reduction="none")
        assert bool(((loss.double() - want).abs() <= h * 2.0 ** -23 * 6 + 2.0 ** -16).all())
    dx, dw = torch.autograd.grad(loss.sum(), (x, w))
    with torch.no_grad():
        d = torch.softmax(s, 1)
        d[torch.arange(3), y] -= 1
        for rows in (slice(0, 40), slice(v - 100, v), slice(131072 - 20, 131072 + 20)):          # 131072 * 16384 = 2^31
            t = d[:, rows].t() @ x.double()
            size = d[:, rows].abs().t() @ x.double().abs()
            assert bool(((dw[rows].double() - t).abs() <= size * 2.0 ** -7 + 1e-30).all())
        ex = sum(d[:, i:i + 20000] @ w[i:i + 20000].double() for i in range(0, v, 20000))
        assert float((dx.double() - ex).norm()) <= 2.0 ** -7 * float(ex.norm())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("t", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("v,h", [(1, 8), (3, 248), (4, 256), (5, 264), (31, 520), (33, 2048), (9000, 1000), (40000, 512), (700, 4096), (70, 16384)])
def test_a_handful_of_tokens(dtype, t, v, h):
    """Logits on the CUDA cores where a handful of tokens has not too many columns: rows, runs of columns and words that end inside a
    warp's four; every second token ignored too."""
    x, w, y = _inputs(t, v, h, dtype)
    loss, _, _ = _check(x, w, y)
    half = torch.where(torch.arange(t, device="cuda") % 2 == 0, torch.full_like(y, -100), y)
    again, _, _ = _check(x, w, half)
    assert torch.equal(again[1::2], loss[1::2])                  # a token's loss does not depend on its neighbours'


@pytest.mark.parametrize("dtype", [BF, HF])
def test_a_handful_of_tokens_of_odd_places(dtype):
    x, w, y = _inputs(4, 1000, 256, dtype)
    want = linear_cross_entropy(x, w, y, reduction="none")
    wide = torch.full((4, 300), float("nan"), device="cuda", dtype=dtype)
    wide[:, 3:259] = x
    assert torch.equal(linear_cross_entropy(wide[:, 3:259], w, y, reduction="none"), want)
    x[2, 5] = float("nan")                                       # one token's NaN is its own
    got = linear_cross_entropy(x, w, y, reduction="none")
    assert torch.equal(got.isnan(), torch.tensor([False, False, True, False], device="cuda")) and torch.equal(got[[0, 1, 3]], want[[0, 1, 3]])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("t,v,h", [(1, 4000, 64), (3, 50, 200), (60, 9000, 136), (256, 30000, 72)])
def test_the_label_entry_loses_nothing(dtype, reduction, t, v, h):
    """The label's entry of dL counts in full: no rounding of it to 16 bits in dx, nor, up to 256 tokens of which no 32 words have more than
    eight as their labels, in dw.  Every other entry is rounded once, sums and the last rounding are those of _check."""
    x, w, y = _inputs(t, v, h, dtype)
    if t > 8:
        y = torch.arange(t, device="cuda") * 7 % v
        assert int(torch.bincount(y // 32).max()) <= 8
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    grad = 0.5 + torch.rand(t, device="cuda") if reduction == "none" else torch.tensor(0.7, device="cuda")
    dx, dw = torch.autograd.grad(linear_cross_entropy(xg, wg, y, reduction=reduction), (xg, wg), grad)
    g = (grad if reduction == "none" else grad.expand(t) / t).double()[:, None]
    xd, wd = x.double(), w.double()
    p = torch.softmax(xd @ wd.t(), 1)
    own = torch.zeros_like(p).scatter_(1, y[:, None], 1.0)
    d, others = (p - own) * g, p * (1 - own) * g
    half = torch.finfo(dtype).eps / 2
    logit = h * 2.0 ** -23 * float((xd.abs() @ wd.abs().t()).max())
    soft = 2 * logit + 2.0 ** -20 * (2 + float(-p.gather(1, y[:, None]).log().min()))
    for got, want, size, rounded, whole, n in ((dx, d @ wd, (p * g) @ wd.abs(), others @ wd.abs(), d.abs() @ wd.abs(), v),
                                               (dw, d.t() @ xd, (p * g).t() @ xd.abs(), others.t() @ xd.abs(), d.abs().t() @ xd.abs(), t)):
        tol = size * 2 * soft + rounded * half * 1.01 + whole * (n + h) * 2.0 ** -23 + want.abs() * half * 1.01 + torch.finfo(dtype).smallest_normal
        if dtype == HF:                                          # entries below fp16's smallest normal number, beside a largest of at least 2^13
            tol = tol + 2.0 ** -38 * float(g.max()) * (wd if n == v else xd).abs().sum(0)
        assert bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("t", [40, 256, 300])
def test_one_label_for_all(dtype, t):
    x, w, y = _inputs(t, 600, 136, dtype)
    _check(x, w, torch.full_like(y, 77))
    _check(x, w, 64 + y % 32)


@pytest.mark.parametrize("t", [33, 50, 64, 65])
def test_some_tokens_of_a_large_fp32_head(t):
    x, w, y = _inputs(t, 131072 + 7, 1024, SF, keep=0.9)
    loss, dx, _ = _check(x, w, y)
    wide = torch.zeros(t, 1027, device="cuda")
    wide[:, 1:1025] = x                                          # rows of another alignment: another form
    logit = 1024 * 2.0 ** -23 * float((x.double().abs() @ w.double().abs().t()).max())
    again = linear_cross_entropy(wide[:, 1:1025], w, y, reduction="none")
    assert bool(((again - loss).abs() <= 2 * (2 * logit + 2.0 ** -20 * (2 + float(loss.detach().max())))).all())


@pytest.mark.parametrize("dtype,t,v,h", [(BF, 1, 5000, 2048), (HF, 4, 9000, 2048), (BF, 5, 9000, 2048), (BF, 300, 9000, 2048), (SF, 20, 5000, 1024),
                                         (SF, 40, 131072, 1024), (SF, 70, 5000, 1024)])
def test_nearly_certain_tokens(dtype, t, v, h):
    """Logits near 60 and 1 - p from 1e-5 to 1e-2: g (p - 1) of the label is as exact as the sum of the other words' p, whichever forms of the
    products the forward and the backward pass took: their differences of 2^-20 of a logit act on the p of other words alone."""
    g = torch.Generator(device="cuda").manual_seed(t + v)
    w = (torch.randn(v, h, generator=g, device="cuda") * h ** -0.5).to(dtype)
    y = torch.randint(0, v, (t,), generator=g, device="cuda")
    rest = 10 ** (-5 + 3 * torch.rand(t, generator=g, device="cuda"))
    base = torch.rand(t, h, generator=g, device="cuda") * w[y].float().sign() * 0.6       # products of one sign: what a cut is worst for
    x = base
    for _ in range(6):                                           # along w[y] until the label has the probability wanted
        s = x.to(dtype).double() @ w.double().t()
        others = torch.logsumexp(s.scatter(1, y[:, None], -float("inf")), 1)
        gap = -torch.log(rest.double()) - (s.gather(1, y[:, None])[:, 0] - others)
        x = x + (gap / (w[y].double() ** 2).sum(1))[:, None].float() * w[y].float()
    x = x.to(dtype)
    xd, wd = x.double(), w.double()
    p = torch.softmax(xd @ wd.t(), 1)
    own = torch.zeros_like(p).scatter_(1, y[:, None], 1.0)
    tail = (p * (1 - own)).sum(1)
    assert float(tail.max()) < 0.05 and float(tail.min()) > 1e-7
    xg = x.clone().requires_grad_()
    dx = torch.autograd.grad(linear_cross_entropy(xg, w, y, reduction="sum"), xg)[0]
    want = -tail[:, None] * wd[y] + (p * (1 - own)) @ wd
    half = torch.finfo(dtype).eps / 2
    logit = h * 2.0 ** -23 * float((xd.abs() @ wd.abs().t()).max())
    soft = 2 * logit + 2.0 ** -20
    # the label's entry: the others' sum, off by soft, and p itself, a few roundings of numbers up to 1; the other entries: soft and one rounding
    tol = (tail * 2 * soft + 2.0 ** -21)[:, None] * wd[y].abs() + (p * (1 - own)) @ wd.abs() * (2 * soft + half * 1.01) + want.abs() * half * 1.01
    tol = tol + torch.finfo(dtype).smallest_normal + (2.0 ** -38 * wd.abs().sum(0) if dtype == HF else 0)
    assert bool(((dx.double() - want).abs() <= tol).all()), float(((dx.double() - want).abs() / tol).max())
