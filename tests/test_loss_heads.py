"""The loss of forward(labels=...) where the LM head is more than its weight: that of the logits which the same call returns."""
import pytest
import torch
import torch.nn.functional as F
from torch import nn
from torch.nn.utils import parametrize

import trimkv_b200 as t
from tests.host_emulation import on_device
from trimkv_b200 import modeling_trimkv
from trimkv_b200.losses import logits_cross_entropy


def _model(dtype=torch.float32):
    kw = dict(vocab_size=131, hidden_size=128, intermediate_size=64, num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=1, head_dim=64,
              retention_gate_intermediate_size=32, compress_memory=False, rope_parameters=dict(rope_type="default", rope_theta=1e4),
              attn_implementation="sdpa", tie_word_embeddings=False, pad_token_id=0, eos_token_id=None, bos_token_id=None)
    torch.manual_seed(2)
    model = t.TrimKVLlamaForCausalLM(t.TrimKVLlamaConfig(**kw))
    with torch.no_grad():
        for p in model.parameters():
            if p.dim() > 1:
                p.normal_(0, p.shape[-1] ** -0.5)
    return model.to(dtype)


class Adapter(nn.Module):
    """A low-rank addition beside a head, with a name of its own for everything."""

    def __init__(self, head):
        super().__init__()
        self.head, self.weight = head, head.weight
        self.down, self.up = nn.Linear(head.in_features, 4, bias=False), nn.Linear(4, head.out_features, bias=False)

    def forward(self, x):
        return self.head(x) + self.up(self.down(x))


class Doubled(nn.Module):
    def forward(self, w):
        return 2 * w


def _bias(model):
    head = nn.Linear(model.config.hidden_size, model.config.vocab_size, bias=True)
    head.weight = model.lm_head.weight
    nn.init.normal_(head.bias, std=2.0)
    model.set_output_embeddings(head)


def _replaced(model):
    plain = model.lm_head.forward
    model.lm_head.forward = lambda x: plain(x) * 1.5


CHANGES = {
    "bias": _bias, "adapter": lambda m: m.set_output_embeddings(Adapter(m.lm_head)),
    "parametrization": lambda m: parametrize.register_parametrization(m.lm_head, "weight", Doubled()),
    "hook": lambda m: m.lm_head.register_forward_hook(lambda mod, args, out: out * 0.5),
    "hook before": lambda m: m.lm_head.register_forward_pre_hook(lambda mod, args: (args[0] * 3.0,)), "replaced": _replaced}


class OnePass:
    """Stands in for a cache on the CPU, for a pass over everything at once."""

    def get_seq_length(self, layer_idx=0):
        return 0

    def update(self, k, v, retention_weights, cache_position, layer_idx, extra):
        return k, v, retention_weights, None, {}


def _check(model, tol):
    device = model.device
    more = dict(past_key_values=OnePass()) if device.type == "cpu" else {}
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(1, 131, (2, 17), generator=g).to(device)
    labels = ids.clone()
    labels[0, :6] = -100
    calls = []
    model.lm_head.register_forward_hook(lambda *a: calls.append(1) or None)
    out = model(input_ids=ids, labels=labels, **more)
    assert len(calls) == 1
    target = labels[:, 1:].flatten()
    z = out.logits.double()[:, :-1].flatten(0, 1)
    want = F.cross_entropy(z, target)
    assert abs(float(out.loss.detach()) - float(want.detach())) <= tol * float(want.detach())
    params = [p for p in model.parameters() if p.requires_grad]
    got, ref = (torch.autograd.grad(x, params, retain_graph=True, allow_unused=True) for x in (out.loss, want))
    assert sum(a is not None for a in got) > 6
    for a, b in zip(got, ref):
        assert (a is None) == (b is None)
        if a is not None:
            assert float((a.double() - b.double()).norm()) <= 64 * tol * float(b.double().norm()) + 1e-12
    short = model(input_ids=ids, labels=labels, logits_to_keep=2, **more)
    assert torch.equal(short.loss, out.loss) and torch.equal(short.logits, out.logits[:, -2:])
    none = model(input_ids=ids, labels=labels, logits_to_keep=None, **more)
    assert torch.equal(none.loss, out.loss) and none.logits is None
    count = int((target >= 0).sum())
    half = model(input_ids=ids, labels=labels, logits_to_keep=None, num_items_in_batch=2 * count, **more).loss
    assert abs(2 * float(half.detach()) - float(out.loss.detach())) <= 2.0 ** -20 * float(want.detach())
    assert abs(float(model.loss_of(out.last_hidden_state, labels).detach()) - float(out.loss.detach())) <= tol * float(want.detach())


@pytest.mark.parametrize("change", list(CHANGES))
def test_the_loss_is_that_of_the_logits(change):
    model = _model()
    assert model._head_is_its_weight()
    CHANGES[change](model)
    assert not model._head_is_its_weight()
    _check(model, 2.0 ** -18)                       # fp32: a few roundings of numbers up to 2^5


@pytest.mark.gpu
@pytest.mark.parametrize("change", list(CHANGES))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_loss_is_that_of_the_logits_on_the_gpu(change, dtype):
    torch.backends.cuda.matmul.allow_tf32 = False
    model = _model()
    CHANGES[change](model)
    # bf16: the logits of both are the same bf16 numbers; gradients of them are rounded to bf16 once (2^-8)
    _check(model.to("cuda", dtype), 2.0 ** -18 if dtype == torch.float32 else 2.0 ** -14)


def test_a_plain_head_takes_the_weight(monkeypatch):
    seen = []

    def fused(hidden, weight, labels, **how):
        seen.append((hidden.shape, weight.shape, how))
        return hidden.sum()
    monkeypatch.setattr(modeling_trimkv, "linear_cross_entropy", fused)
    model = _model()
    hidden = on_device(torch.zeros(2, 5, 128))
    model.loss_of(hidden, torch.ones(2, 5, dtype=torch.int64))
    assert seen == [((2, 5, 128), (131, 128), dict(ignore_index=-100, reduction="mean"))]


def test_losses_of_logits():
    z = 4 * torch.randn(3, 7, 11, generator=torch.Generator().manual_seed(1))
    y = torch.randint(0, 11, (3, 7), generator=torch.Generator().manual_seed(2))
    y[0, 2:5] = -100
    bad = z.clone()
    bad[0, 2:5] = float("nan")                      # rows that do not count
    for reduction in ("none", "mean", "sum"):
        x = bad.clone().requires_grad_()
        got = logits_cross_entropy(x, y, reduction=reduction)
        ref = z.double().requires_grad_()
        want = F.cross_entropy(ref.flatten(0, 1), y.flatten(), reduction=reduction).view(got.shape)
        assert bool(((got.double() - want).abs() <= 2.0 ** -19 * (1 + want.abs())).all())
        up = torch.rand(got.shape)
        a, b = torch.autograd.grad(got, x, up)[0], torch.autograd.grad(want, ref, up.double())[0]
        assert bool(((a.double() - b).abs() <= 2.0 ** -20).all())
    assert bool(logits_cross_entropy(z, torch.full_like(y, -100)).isnan())
    assert float(logits_cross_entropy(z, torch.full_like(y, -100), reduction="sum")) == 0.0
    y[1, 1], y[2, 2] = 11, -7
    x = z.clone().requires_grad_()
    each = logits_cross_entropy(x, y, reduction="none")
    assert each.isnan().nonzero().tolist() == [[1, 1], [2, 2]]
    dx, = torch.autograd.grad(each[~each.isnan()].sum(), x)
    assert not bool(dx[1, 1].any()) and not bool(dx[2, 2].any()) and bool(dx.isfinite().all())
    y = y.masked_fill((y < 0) | (y > 10), 3)
    assert torch.equal(logits_cross_entropy(z, y, ignore_index=3, reduction="none") == 0, y == 3)
