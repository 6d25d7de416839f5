"""Rotary positions of models that were loaded from a checkpoint: the tables are those of the model that was saved."""
import pytest
import torch

import trimkv_b200 as t

FAMILIES = {"qwen3": (t.TrimKVQwen3Config, t.TrimKVQwen3ForCausalLM), "llama": (t.TrimKVLlamaConfig, t.TrimKVLlamaForCausalLM),
            "phi3": (t.TrimKVPhi3Config, t.TrimKVPhi3ForCausalLM)}
ROPE = {
    "default": dict(rope_type="default", rope_theta=5e5),
    "linear": dict(rope_type="linear", rope_theta=1e4, factor=4.0),
    "llama3": dict(rope_type="llama3", rope_theta=5e5, factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=64),
    "yarn": dict(rope_type="yarn", rope_theta=1e6, factor=4.0, original_max_position_embeddings=128),
    "longrope": dict(rope_type="longrope", rope_theta=1e4, short_factor=[1.0 + 0.02 * i for i in range(32)],
                     long_factor=[2.0 + 0.3 * i for i in range(32)], original_max_position_embeddings=48),
    "dynamic": dict(rope_type="dynamic", rope_theta=1e4, factor=2.0)}
CASES = [("llama", k) for k in ("default", "linear", "llama3", "dynamic")] + [("qwen3", "default"), ("qwen3", "yarn"), ("phi3", "default"), ("phi3", "longrope")]


def _saved(family, kind, path, **more):
    Cfg, Cls = FAMILIES[family]
    kw = dict(vocab_size=97, hidden_size=128, intermediate_size=64, num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=1, head_dim=64,
              retention_gate_intermediate_size=32, compress_memory=False, max_position_embeddings=512, rope_parameters=ROPE[kind],
              attn_implementation="sdpa", tie_word_embeddings=False, pad_token_id=0, eos_token_id=None, bos_token_id=None)
    torch.manual_seed(1)
    model = Cls(Cfg(**dict(kw, **more)))
    model.save_pretrained(path)
    return model, Cls


@pytest.mark.parametrize("family,kind", CASES)
def test_tables_of_a_loaded_model(family, kind, tmp_path):
    model, Cls = _saved(family, kind, tmp_path)
    loaded = Cls.from_pretrained(str(tmp_path), load_trimkv_weights=False)
    x, cpu = torch.zeros(1), torch.device("cpu")
    for pos in (torch.arange(40)[None], torch.arange(700, 720)[None]):
        want, got = model.model.rotary_emb, loaded.model.rotary_emb
        (f0, s0), (f1, s1) = want.plan.on(cpu, pos), got.plan.on(cpu, pos)
        assert torch.equal(f0, f1) and s0 == s1
        for a, b in zip(want(x, pos), got(x, pos)):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("family,kind", CASES)
def test_a_loaded_model_runs(family, kind, tmp_path):
    """The same logits as the model that was saved, bit for bit, for a prompt and a token behind it."""
    more = dict(head_dim=128, hidden_size=256, partial_rotary_factor=0.5) if family == "phi3" else {}
    model, Cls = _saved(family, kind, tmp_path, attn_implementation="tkv_b200", **more)
    loaded = Cls.from_pretrained(str(tmp_path), load_trimkv_weights=False, dtype=torch.bfloat16, attn_implementation="tkv_b200").cuda().eval()
    model = model.to(torch.bfloat16).cuda().eval()
    ids = torch.randint(1, 97, (2, 41), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    with torch.no_grad():
        for m in (model, loaded):
            m.cache = m.new_cache()
        a, b = (m(input_ids=ids[:, :40], past_key_values=m.cache).logits for m in (model, loaded))
        assert bool(a.isfinite().all()) and torch.equal(a, b)
        a, b = (m(input_ids=ids[:, 40:], past_key_values=m.cache).logits for m in (model, loaded))
        assert bool(a.isfinite().all()) and torch.equal(a, b)
