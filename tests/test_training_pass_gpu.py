"""Positions, experts' balance and vocabulary loss together, as a training or scoring pass through the decoders uses them."""
import pytest
import torch
import torch.nn.functional as F

import trimkv_b200 as t
from trimkv_b200 import modeling_trimkv
from trimkv_b200.feedforward import SparseMLP
from tests import dafovik_cases, lonulix_cases

pytestmark = pytest.mark.gpu

ROPE = {"llama": dict(rope_type="llama3", rope_theta=5e5, factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=64),
        "qwen3": dict(rope_type="yarn", rope_theta=1e6, factor=4.0, original_max_position_embeddings=128),
        "phi3": dict(rope_type="longrope", rope_theta=1e4, short_factor=[1.0 + 0.02 * i for i in range(32)], long_factor=[2.0 + 0.3 * i for i in range(32)],
                     original_max_position_embeddings=48)}


def _model(family, dtype, **more):
    Cfg, Cls = {"qwen3": (t.TrimKVQwen3Config, t.TrimKVQwen3ForCausalLM), "llama": (t.TrimKVLlamaConfig, t.TrimKVLlamaForCausalLM),
                "phi3": (t.TrimKVPhi3Config, t.TrimKVPhi3ForCausalLM)}[family]
    kw = dict(vocab_size=517, hidden_size=128, intermediate_size=192, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=128,
              retention_gate_intermediate_size=32, memory_size=64, buffer_size=16, compress_memory=False, max_position_embeddings=4096,
              rope_parameters=ROPE[family], attn_implementation="sdpa", tie_word_embeddings=False, pad_token_id=0, eos_token_id=None, bos_token_id=None)
    if family == "phi3":
        kw.update(partial_rotary_factor=0.5, hidden_size=512)
    kw.update(more)
    torch.manual_seed(3)
    model = Cls(Cfg(**kw)).to(dtype).cuda()
    with torch.no_grad():
        for p in model.parameters():
            if p.dim() > 1:
                p.normal_(0, p.shape[-1] ** -0.5)
    return model


def _ids(b=2, s=75):
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.randint(1, 517, (b, s), generator=g, device="cuda")
    labels = ids.clone()
    labels[0, :20] = -100
    return ids, labels


def _plain(monkeypatch):
    """The eager rotation for scaled positions too."""
    real = modeling_trimkv.RotaryEmbedding.forward
    monkeypatch.setattr(modeling_trimkv.RotaryEmbedding, "forward", lambda self, x, p: modeling_trimkv.RotaryTables(real(self, x, p)))


def _near(a, b, rel):
    return float((a.double() - b.double()).norm()) <= rel * float(b.double().norm()) + 1e-12


@pytest.mark.parametrize("family", sorted(ROPE))
def test_loss_and_gradients_of_a_pass(family, monkeypatch):
    """fp32: the loss of a pass and every parameter's gradient against the same model with eager rotations and a loss from its logits.
    Both are fp32 passes of the same formulas through two layers, a few hundred roundings of 2^-24 deep: 2^-14 of a gradient's norm."""
    torch.backends.cuda.matmul.allow_tf32 = False
    model = _model(family, torch.float32)
    ids, labels = _ids()
    out = model(input_ids=ids, labels=labels, logits_to_keep=None)
    assert out.logits is None and out.loss.shape == ()
    out.loss.backward()
    got = {n: p.grad for n, p in model.named_parameters() if p.grad is not None}
    model.zero_grad(set_to_none=True)
    _plain(monkeypatch)
    plain = model(input_ids=ids)
    assert plain.loss is None
    loss = F.cross_entropy(plain.logits[:, :-1].flatten(0, 1), labels[:, 1:].flatten())
    loss.backward()
    want = {n: p.grad for n, p in model.named_parameters() if p.grad is not None}
    assert abs(float(out.loss.detach()) - float(loss.detach())) <= 2.0 ** -16 * float(loss.detach())
    assert set(got) == set(want) and any("q_proj" in n or "qkv_proj" in n for n in got)
    for n in want:
        assert _near(got[n], want[n], 2.0 ** -14), n


def test_loss_forms():
    model = _model("llama", torch.bfloat16)
    ids, labels = _ids()
    with torch.no_grad():
        base = model(input_ids=ids, labels=labels)
        logits = base.logits.double()
        want = F.cross_entropy(logits[:, :-1].flatten(0, 1), labels[:, 1:].flatten())
        # the logits were rounded to bf16 (2^-8 of up to max |logit|), the loss was taken from unrounded ones
        tol = 2.0 ** -8 * float(logits.abs().max()) * 2
        assert abs(float(base.loss) - float(want)) <= tol
        kept = model(input_ids=ids, labels=labels, logits_to_keep=3)
        assert kept.logits.shape == (2, 3, 517) and torch.equal(kept.loss, base.loss)
        count = int((labels[:, 1:] >= 0).sum())
        by = model(input_ids=ids, labels=labels, logits_to_keep=None, num_items_in_batch=2 * count).loss
        assert abs(float(by) * 2 - float(base.loss)) <= 2.0 ** -20 * float(base.loss)
        moved = F.pad(labels[:, 1:], (0, 1), value=-100)
        assert torch.equal(model(input_ids=ids, labels=labels, shift_labels=moved, logits_to_keep=None).loss, base.loss)
        assert torch.equal(model(input_ids=ids, shift_labels=moved, logits_to_keep=None).loss, base.loss)
    with torch.inference_mode():
        assert torch.equal(model(input_ids=ids, labels=labels, logits_to_keep=None).loss, base.loss)
    with torch.no_grad():
        assert torch.equal(model(input_ids=ids).logits, base.logits) and model(input_ids=ids).loss is None
        other = model(input_ids=ids, labels=labels.masked_fill(labels < 0, 7), logits_to_keep=None, ignore_index=7).loss
        assert bool(other.isfinite())


@pytest.mark.parametrize("family", sorted(ROPE))
def test_decoding_with_scaled_positions(family):
    """A prompt, then token by token through the cache and its kernels, against one pass over everything (bf16).  Where the cache's keys were
    turned by the kernel and the queries by tables in bf16, a score is off by a rounding or two of 2^-8 of its size."""
    model = _model(family, torch.bfloat16, attn_implementation="tkv_b200").eval()
    ids, _ = _ids(2, 60)
    at = 40 if family == "phi3" else 52                            # longrope: all of the pass within or beyond the original length
    if family == "phi3":
        ids = ids[:, :47]
    with torch.inference_mode():
        whole = model(input_ids=ids).logits.float()
        cache = model.new_cache()
        first = model(input_ids=ids[:, :at], past_key_values=cache).logits.float()
        assert float((first - whole[:, :at]).norm()) <= 0.03 * float(whole[:, :at].norm())
        for i in range(at, ids.shape[1]):
            step = model(input_ids=ids[:, i:i + 1], past_key_values=cache).logits.float()
            assert float((step[:, 0] - whole[:, i]).norm()) <= 0.05 * float(whole[:, i].norm()), i


def test_fused_step_with_scaled_positions():
    model = _model("llama", torch.bfloat16, attn_implementation="tkv_b200", hidden_act="silu").eval()
    ids, _ = _ids(2, 50)
    with torch.inference_mode():
        a, b = model.new_cache(), model.new_cache()
        for cache in (a, b):
            model(input_ids=ids, past_key_values=cache)
        for i in range(4):
            nxt = ids[:, i:i + 1]
            model.config.fused_decode_step = False
            plain = model(input_ids=nxt, past_key_values=a).logits.float()
            model.config.fused_decode_step = True
            fused = model(input_ids=nxt, past_key_values=b).logits.float()
            assert float((plain - fused).norm()) <= 0.05 * float(plain.norm()), i


def test_the_kernel_for_the_default_embedding_on_request():
    """``fused_rotary``: near the default path (which rounds the tables and every product to bf16), which itself stays as it was."""
    plain = _model("llama", torch.bfloat16, rope_parameters=dict(rope_type="default", rope_theta=5e5))
    ids, _ = _ids()
    with torch.no_grad():
        a = plain(input_ids=ids).logits
        assert plain.model.rotary_emb(a, torch.arange(4, device="cuda")[None]).turn is None
        plain.config.fused_rotary = True
        assert plain.model.rotary_emb(a, torch.arange(4, device="cuda")[None]).turn is not None
        b = plain(input_ids=ids).logits
    assert float((a.float() - b.float()).norm()) <= 0.03 * float(a.float().norm()) and not torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("identity", [0, 2])
def test_balance_of_a_routed_layer(dtype, identity):
    torch.manual_seed(5)
    mlp = SparseMLP(64, 32, experts=8 - identity, top=3, identity=identity).cuda()
    mlp.reset_parameters(0.3)
    mlp = mlp.to(dtype)
    x = torch.randn(300, 64, device="cuda", dtype=dtype, requires_grad=True)
    valid = torch.rand(300, device="cuda") < 0.8
    loss, counts = mlp.balance(x, valid)
    _, _, _, offsets = mlp.route(x[valid].detach())
    real = 8 - identity
    assert torch.equal(counts[:real], offsets[1:] - offsets[:-1]) and int(counts.sum()) == 3 * int(valid.sum())
    gr, gx = torch.autograd.grad(loss, (mlp.router, x))
    n = int(valid.sum())
    z = x.detach()[valid].double() @ mlp.router.detach().double().t()
    p = torch.softmax(z, 1)
    f = counts.double() / (3 * n)
    assert abs(float(loss.detach()) - float(8 * (f * p.mean(0)).sum())) <= 2.0 ** -18
    dz = 8 / n * p * (f - (p * f).sum(1, keepdim=True))
    assert _near(gr, dz.t() @ x.detach()[valid].double(), 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -18)
    full = torch.zeros(300, 64, device="cuda", dtype=torch.float64)
    full[valid] = dz @ mlp.router.detach().double()
    assert _near(gx, full, 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -18)
    with torch.no_grad():
        quiet = mlp.balance(x, valid)
    assert torch.equal(quiet[1], counts)


def test_all_of_them_in_one_training_pass(monkeypatch):
    """Scaled positions, vocabulary loss and the balance of a router that reads the decoder's hidden rows, padding left out: the sum's
    gradients against a pass without any of the kernels (fp32; the same tolerance as above)."""
    torch.backends.cuda.matmul.allow_tf32 = False
    model = _model("llama", torch.float32)
    router = SparseMLP(128, 64, experts=6, top=2).cuda()
    router.reset_parameters(0.3)
    ids, labels = _ids()
    valid = torch.ones_like(ids, dtype=torch.bool)
    valid[1, 60:] = False
    labels = labels.masked_fill(~valid, -100)
    out = model(input_ids=ids, labels=labels, logits_to_keep=None)
    balance, counts = router.balance(out.last_hidden_state.flatten(0, 1), valid.flatten())
    (out.loss + 0.05 * balance).backward()
    named = list(model.named_parameters()) + [("router", router.router)]
    got = {n: p.grad.clone() for n, p in named if p.grad is not None}
    for _, p in named:
        p.grad = None
    _plain(monkeypatch)
    plain = model(input_ids=ids)
    z = F.linear(plain.last_hidden_state.flatten(0, 1), router.router)[valid.flatten()]
    n = z.shape[0]
    aux = 6 * (counts / (2.0 * n) * torch.softmax(z, 1).mean(0)).sum()
    loss = F.cross_entropy(plain.logits[:, :-1].flatten(0, 1), labels[:, 1:].flatten()) + 0.05 * aux
    loss.backward()
    assert abs(float((out.loss + 0.05 * balance).detach()) - float(loss.detach())) <= 2.0 ** -16 * float(loss.detach())
    for n, p in named:
        if p.grad is not None:
            assert _near(got[n], p.grad, 2.0 ** -14), n


@pytest.mark.parametrize("design", ["lonulix", "dafovik"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_loss_of_the_hybrid_decoders(design, dtype, tmp_path):
    """Scoring with padding on either side: the loss is that of the logits, which stay as they were."""
    cases, cls = {"lonulix": (lonulix_cases, t.LonulixForCausalLM), "dafovik": (dafovik_cases, t.DafovikForCausalLM)}[design]
    cfg = cases.CONFIGS["mixed"]
    dafovik_cases.write_checkpoint(tmp_path, cfg, cases.random_tensors(cfg))
    model = cls.from_pretrained(str(tmp_path), dtype=dtype).cuda()
    g = torch.Generator(device="cuda").manual_seed(2)
    ids = torch.randint(0, cfg["vocab"], (3, 31), generator=g, device="cuda")
    mask = torch.ones_like(ids)
    mask[1, :9] = 0
    mask[2, 20:] = 0
    labels = ids.clone()
    labels[0, 4:9] = -100
    for m in (None, mask):
        with torch.no_grad():
            logits = model(input_ids=ids, attention_mask=m).logits
            out = model(input_ids=ids, attention_mask=m, labels=labels)
            short = model(input_ids=ids, attention_mask=m, labels=labels, logits_to_keep=None)
            one = model(input_ids=ids, attention_mask=m, labels=labels, logits_to_keep=2)
        target = labels[:, 1:].clone()
        if m is not None:
            target[(m[:, 1:] == 0) | (m[:, :-1] == 0)] = -100
        want = F.cross_entropy(logits[:, :-1].double().flatten(0, 1), target.flatten())
        # fp32 logits of both passes, a hundred products each: 2^-17 of a logit below 2^5
        assert abs(float(out.loss) - float(want)) <= 2.0 ** -12
        assert torch.equal(out.logits, logits) and torch.equal(short.loss, out.loss) and short.logits is None
        assert torch.equal(one.logits, logits[:, -2:])
    single = model(input_ids=ids[:, :1], shift_labels=ids[:, 1:2], logits_to_keep=None)
    assert bool(single.loss.isfinite())
