"""Operators of an adaptation or scoring pass through a decoder, as cases that can be timed: sizes, inputs, one pass, what it cannot
do without, and what it should give.

  * ``rotary``: queries and keys turned by their positions, in halves or in neighbouring pairs, the whole head or its first part, with
    the frequencies of long-context checkpoints; training passes turn the gradients back;
  * ``loss``: softmax cross entropy of hidden rows against a large vocabulary straight from the head's weight, for scoring (a number
    per token) and for training (gradients of the rows and, unless the head is frozen, of the weight);
  * ``balance``: how evenly a router spreads its tokens over the experts, as a loss with its gradient, and the tokens of each expert.

Sizes are those of the repository's benchmark (width 2048, vocabulary 151936, heads of 128) and what lies around them.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
IGNORE = -100


# ---------------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # A chat with one user: one token's queries and keys of a layer.  Latency.
        dict(name="rotary 1 token", kind="rotary", batch=1, tokens=1, heads=16, kv_heads=8, dim=128, rot=128, layout="half",
             scale=1.0, start=4100, train=False, dtype="bf16"),
        # One token of 64 requests, half of the head turned.
        dict(name="rotary 64 requests part", kind="rotary", batch=64, tokens=1, heads=32, kv_heads=8, dim=128, rot=64, layout="pairs",
             scale=1.0, start=30000, train=False, dtype="f16"),
        # A layer of a long prompt, far out, with the scale that goes with stretched frequencies.
        dict(name="rotary 8192 tokens", kind="rotary", batch=1, tokens=8192, heads=32, kv_heads=8, dim=128, rot=128, layout="half",
             scale=1.19, start=122880, train=False, dtype="bf16"),
        # Training, there and back, an odd length.
        dict(name="rotary training 4 x 2731", kind="rotary", batch=4, tokens=2731, heads=16, kv_heads=8, dim=128, rot=64,
             layout="pairs", scale=1.0, start=0, train=True, dtype="f16"),
        # The log probability of one given token (a choice scored while decoding): the weight is read once.
        dict(name="loss 1 token", kind="loss", tokens=1, width=2048, vocab=151936, keep=1.0, train="", reduction="none", dtype="bf16"),
        # Scoring a prompt.
        dict(name="loss scoring 1500", kind="loss", tokens=1500, width=2048, vocab=151936, keep=1.0, train="", reduction="none",
             dtype="bf16"),
        # A training step's loss, the head trained too.  The largest case.
        dict(name="loss training 8192", kind="loss", tokens=8192, width=2048, vocab=151936, keep=1.0, train="xw", reduction="mean",
             dtype="bf16"),
        # Answers only: most tokens are prompt or padding and count for nothing; the head is frozen.
        dict(name="loss answers of 6000 frozen head", kind="loss", tokens=6000, width=4096, vocab=32768, keep=0.4, train="x",
             reduction="mean", dtype="f16"),
        # A short batch and a vocabulary of odd size.
        dict(name="loss training 777 odd", kind="loss", tokens=777, width=1024, vocab=50257, keep=0.9, train="xw", reduction="sum",
             dtype="bf16"),
        # A model kept in 32 bits.
        dict(name="loss training 300 f32", kind="loss", tokens=300, width=1024, vocab=32768, keep=0.9, train="xw", reduction="mean",
             dtype="f32"),
        # The router of a small batch ...
        dict(name="balance 64", kind="balance", tokens=64, experts=32, top=6, keep=1.0, dtype="f32"),
        # ... and of a training batch with padding.
        dict(name="balance 65536", kind="balance", tokens=65536, experts=128, top=8, keep=0.85, dtype="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("rotary", "rotary", "loss", "loss", "loss", "balance"))
    if kind == "rotary":
        kv = rng.choice((1, 2, 4, 8))
        dim = rng.choice((64, 80, 96, 128, 128, 256))
        rot = rng.choice((dim, dim, dim // 2, dim // 4))
        batch, tokens = _log(rng, 1, 64), 1
        if rng.random() < 0.7:
            batch = rng.choice((1, 1, 2, 4))
            tokens = _log(rng, 2, 16384 // batch)
        return dict(kind=kind, batch=batch, tokens=tokens, heads=kv * rng.choice((1, 2, 4)), kv_heads=kv, dim=dim, rot=rot,
                    layout=rng.choice(("half", "pairs")), scale=rng.choice((1.0, 1.0, 1.19)), start=_log(rng, 1, 1 << 20),
                    train=rng.random() < 0.5, dtype=rng.choice(("bf16", "bf16", "f16", "f32")))
    if kind == "balance":
        experts = rng.choice((8, 16, 60, 64, 128, 160, 256))
        return dict(kind=kind, tokens=_log(rng, 1, 65536), experts=experts, top=rng.choice((1, 2, 4, 6, 8)),
                    keep=rng.choice((1.0, 0.85, 0.3)), dtype=rng.choice(("f32", "f32", "bf16")))
    dtype = rng.choice(("bf16", "bf16", "bf16", "f16", "f32"))
    train = rng.choice(("", "x", "xw", "xw"))
    width = 8 * _log(rng, 64, 512)
    vocab = _log(rng, 8000, 200000)
    room = 8192 * 2048 * 151936 * (1.0 if dtype != "f32" else 0.03) / (width * vocab)
    return dict(kind=kind, tokens=_log(rng, 1, max(2, min(8192, int(room)))), width=width, vocab=vocab,
                keep=rng.choice((1.0, 0.9, 0.4)), train=train, reduction=rng.choice(("mean", "sum", "none")), dtype=dtype)


# ------------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape, dtype, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype).mul_(scale)


def _table(pairs):
    """Frequencies of a base of 500000 as a high and a low part, the low ones stretched by eight as long-context checkpoints do."""
    f = 500000.0 ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1))
    f = torch.where(f * 8192 < 2 * math.pi, f / 8, f)
    hi = f.float()
    return torch.stack([hi, (f - hi.double()).float()], 1).to(DEV)


def prepare(case, seed):
    c, g = case, _gen(seed)
    dt = TYPES[c["dtype"]]
    if c["kind"] == "rotary":
        b, s, d = c["batch"], c["tokens"], c["dim"]
        # as the projections leave them: token-major, seen as [batch, heads, tokens, dim]
        q, k, gq, gk = (_randn(g, b, s, n, d, dtype=dt).transpose(1, 2) for n in (c["heads"], c["kv_heads"]) * 2)
        first = torch.randint(0, 64, (b, 1), generator=g, device=DEV) + c["start"]
        st = dict(case=c, q=q, k=k, positions=first + torch.arange(s, device=DEV), freq=_table(c["rot"] // 2))
        if c["train"]:
            st.update(q=q.requires_grad_(), k=k.requires_grad_(), gq=gq, gk=gk)
        return st
    t = c["tokens"]
    live = torch.rand(t, generator=g, device=DEV) < c["keep"]
    if c["kind"] == "balance":
        tilt = torch.randn(c["experts"], generator=g, device=DEV)      # some experts are liked better
        z = (_randn(g, t, c["experts"], dtype=torch.float32) + tilt).to(dt)
        choice = z.float().topk(c["top"], 1).indices.to(torch.int32)
        return dict(case=c, logits=z.requires_grad_(), choice=choice, valid=live)
    w = _randn(g, c["vocab"], c["width"], dtype=dt, scale=0.02)
    x = _randn(g, t, c["width"], dtype=dt)
    labels = torch.randint(0, c["vocab"], (t,), generator=g, device=DEV)
    sure = 12 * torch.rand(t, 1, generator=g, device=DEV) ** 2 / (0.0004 * c["width"])
    x += (sure * w[labels].float()).to(dt)                             # some tokens are nearly certain, most are not
    labels = torch.where(live, labels, torch.full_like(labels, IGNORE))
    return dict(case=c, hidden=x.requires_grad_("x" in c["train"]), weight=w.requires_grad_("w" in c["train"]), labels=labels,
                grad=torch.rand(t, generator=g, device=DEV) if c["reduction"] == "none" else torch.ones((), device=DEV))


# --------------------------------------------------------------------------------------------------------------------- a pass
def _turn(x, cos, sin, layout):
    """x [b, heads, tokens, dim] in 32 bits or more; cos, sin [b, 1, tokens, pairs]."""
    n = cos.shape[-1]
    part, rest = x[..., :2 * n], x[..., 2 * n:]
    if layout == "half":
        a, b = part[..., :n], part[..., n:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b = part[..., 0::2], part[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)


def _rotary(st):
    c = st["case"]
    if own:
        from trimkv_b200 import apply_rotary
        if not c["train"]:
            return apply_rotary(st["q"], st["k"], st["positions"], st["freq"], layout=c["layout"], scale=c["scale"])
        q, k = apply_rotary(st["q"], st["k"], st["positions"], st["freq"], layout=c["layout"], scale=c["scale"])
        dq, dk = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["gq"], st["gk"]))
        return q.detach(), k.detach(), dq, dk
    with torch.no_grad():
        angle = st["positions"].double()[:, None, :, None] * st["freq"].double().sum(1)      # far positions need the bits
        cos, sin = (angle.cos() * c["scale"]).float(), (angle.sin() * c["scale"]).float()
        out = [_turn(st[n].float(), cos, sin, c["layout"]).to(st[n].dtype) for n in ("q", "k")]
        if c["train"]:
            out += [_turn(st[n].float(), cos, -sin, c["layout"]).to(st[n].dtype) for n in ("gq", "gk")]
        return tuple(out)


def _loss(st):
    c, x, w, labels = st["case"], st["hidden"], st["weight"], st["labels"]
    if own:
        from trimkv_b200 import linear_cross_entropy
        loss = linear_cross_entropy(x, w, labels, ignore_index=IGNORE, reduction=c["reduction"])
        if not c["train"]:
            return loss
        return (loss.detach(),) + torch.autograd.grad(loss, [t for t in (x, w) if t.requires_grad], st["grad"])
    with torch.no_grad():
        x32, w32 = x.float(), w.float()
        live = labels != IGNORE
        at = labels.clamp_min(0)[:, None]
        s = x32 @ w32.t()
        top = s.amax(1, keepdim=True)
        mine = s.gather(1, at)
        s.sub_(top).exp_()
        total = s.sum(1, keepdim=True)
        each = torch.where(live, (total.log() + top - mine)[:, 0], 0.0)
        n = live.sum()
        out = [{"none": each, "sum": each.double().sum().float(), "mean": (each.double().sum() / n).float()}[c["reduction"]]]
        if c["train"]:
            g = st["grad"] * live
            g = g / n.clamp_min(1) if c["reduction"] == "mean" else g
            s.mul_((g / total[:, 0])[:, None])
            s.scatter_add_(1, at, -g[:, None])
            if "x" in c["train"]:
                out.append((s @ w32).to(x.dtype))
            if "w" in c["train"]:
                out.append((s.t() @ x32).to(w.dtype))
        return tuple(out) if c["train"] else out[0]


def _balance(st):
    z, choice, valid = st["logits"], st["choice"], st["valid"]
    if own:
        from trimkv_b200 import expert_balance
        loss, counts = expert_balance(z, choice, valid)
        return loss.detach(), counts, torch.autograd.grad(loss, z)[0]
    with torch.no_grad():
        t, e = z.shape
        p = z.float()
        p = (p - p.amax(1, keepdim=True)).exp()
        p = p / p.sum(1, keepdim=True)
        counts = torch.zeros(e, dtype=torch.int32, device=z.device)
        counts.index_add_(0, choice.flatten().long(), valid[:, None].expand_as(choice).flatten().to(torch.int32))
        n = valid.sum().double()
        f = counts.double() / (n * choice.shape[1]).clamp_min(1)
        mean = (p.double() * valid[:, None]).sum(0) / n.clamp_min(1)
        f32 = f.float()
        dz = p * (f32 - (p * f32).sum(1, keepdim=True)) * (valid[:, None] * (e / n.clamp_min(1)).float())
        return (e * (f * mean).sum()).float(), counts, dz.to(z.dtype)


def run(state):
    return {"rotary": _rotary, "loss": _loss, "balance": _balance}[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------------------------ what cannot be avoided
def work(case):
    c, size = case, SIZE[case["dtype"]]
    if c["kind"] == "rotary":
        rows = c["batch"] * c["tokens"]
        values = rows * (c["heads"] + c["kv_heads"]) * c["dim"] * (2 if c["train"] else 1)
        return {"bytes": 2 * values * size + 8 * rows + 4 * c["rot"], "flops": 3 * values}
    t = c["tokens"]
    if c["kind"] == "balance":
        return {"bytes": 2 * t * c["experts"] * size + t * (4 * c["top"] + 1) + 4 * c["experts"], "flops": 10 * t * c["experts"]}
    n = max(1, round(t * c["keep"]))
    ways = 1 + len(c["train"])
    x, w = t * c["width"] * size, c["vocab"] * c["width"] * size
    return {"bytes": x + w + 12 * t + (x if "x" in c["train"] else 0) + (w if "w" in c["train"] else 0),
            "flops": 2 * n * c["width"] * c["vocab"] * ways}


# ------------------------------------------------------------------------------------------------------------- the definition
def _exact_rotary(c, st):
    theta = st["positions"].double().unsqueeze(1).unsqueeze(-1) * (st["freq"][:, 0].double() + st["freq"][:, 1].double())
    turn = torch.polar(torch.full_like(theta, c["scale"]), theta)
    out = []
    for name in ("q", "k") + (("gq", "gk") if c["train"] else ()):
        x, r = st[name].detach().double(), c["rot"]
        y = x.clone()
        if c["layout"] == "half":
            z = torch.complex(x[..., :r // 2], x[..., r // 2:r]) * (turn if name[0] != "g" else turn.conj())
            y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
        else:
            z = torch.complex(x[..., 0:r:2], x[..., 1:r:2]) * (turn if name[0] != "g" else turn.conj())
            y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
        out.append(y)
    return tuple(out)


def _exact_loss(c, st):
    x, w, labels, grad = st["hidden"].detach(), st["weight"].detach().double(), st["labels"], st["grad"].double()
    live = labels != IGNORE
    n = int(live.sum())
    g = (grad if grad.dim() else grad.expand(len(labels))) * live / (n if c["reduction"] == "mean" else 1)
    each = torch.zeros(len(labels), dtype=torch.float64, device=DEV)
    dx = torch.zeros(*x.shape, dtype=torch.float64, device=DEV)
    dw = torch.zeros_like(w) if "w" in c["train"] else None
    for rows in torch.nonzero(live)[:, 0].split(1024):
        xr, yr = x[rows].double(), labels[rows]
        logp = torch.log_softmax(xr @ w.t(), 1)
        each[rows] = -logp[torch.arange(len(rows), device=DEV), yr]
        if c["train"]:
            d = logp.exp_()
            d[torch.arange(len(rows), device=DEV), yr] -= 1
            d *= g[rows, None]
            dx[rows] = d @ w
            if dw is not None:
                dw.addmm_(d.t(), xr)
    value = each if c["reduction"] == "none" else each.sum() / (n if c["reduction"] == "mean" else 1)
    if not c["train"]:
        return value
    return (value,) + ((dx,) if "x" in c["train"] else ()) + ((dw,) if dw is not None else ())


def _exact_balance(c, st):
    z = st["logits"].detach().double()[st["valid"]].requires_grad_()
    n, e = z.shape
    hits = torch.zeros(n, e, dtype=torch.float64, device=DEV).scatter_add_(
        1, st["choice"][st["valid"]].long(), torch.ones(n, c["top"], dtype=torch.float64, device=DEV))
    loss = e * (hits.sum(0) / max(1, n * c["top"]) * torch.softmax(z, 1).sum(0) / max(1, n)).sum()
    dz = torch.zeros(c["tokens"], e, dtype=torch.float64, device=DEV)
    dz[st["valid"]] = torch.autograd.grad(loss, z)[0]
    return loss.detach(), None, dz


def exact(case, seed):
    st = prepare(case, seed)
    return {"rotary": _exact_rotary, "loss": _exact_loss, "balance": _exact_balance}[case["kind"]](case, st)
