"""Rotary frequencies of long-context checkpoints against transformers' own, and what a plan refuses."""
import math

import pytest
import torch
from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

from trimkv_b200 import TrimKVLlamaConfig
from trimkv_b200.modeling_trimkv import RotaryEmbedding, RotaryTables, apply_rotary_pos_emb, rotate
from trimkv_b200.positions import RotaryPlan

KINDS = {
    "linear": dict(factor=4.0),
    "llama3": dict(factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=8192),
    "yarn": dict(factor=4.0, original_max_position_embeddings=32768),
    "yarn mscale": dict(factor=40.0, original_max_position_embeddings=4096, mscale=0.707, mscale_all_dim=0.9, beta_fast=24.0, beta_slow=2.0),
    "yarn attention": dict(factor=16.0, original_max_position_embeddings=4096, attention_factor=1.3, truncate=False),
    "longrope": dict(short_factor=[1.0 + 0.01 * i for i in range(32)], long_factor=[1.0 + 0.9 * i for i in range(32)],
                     original_max_position_embeddings=4096),
    "longrope factor": dict(short_factor=[1.0] * 32, long_factor=[4.0 + i for i in range(32)], factor=16.0,
                            original_max_position_embeddings=4096, attention_factor=1.19),
    "dynamic": dict(factor=4.0),
}


def _config(kind, **more):
    rope = dict(KINDS[kind], rope_type=kind.split()[0], rope_theta=5e5)
    return TrimKVLlamaConfig(vocab_size=64, hidden_size=128, intermediate_size=64, num_hidden_layers=1, num_attention_heads=2,
                             num_key_value_heads=1, head_dim=64, max_position_embeddings=131072 if kind != "dynamic" else 4096,
                             rope_parameters=rope, **more)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("length", [100, 5000, 100000])
def test_frequencies_are_those_of_transformers(kind, length):
    config = _config(kind)
    plan = RotaryEmbedding(config).plan
    freq, scale = plan.on(torch.device("cpu"), torch.arange(length - 10, length)[None])
    inv, attention = ROPE_INIT_FUNCTIONS[kind.split()[0]](config, torch.device("cpu"), seq_len=length)
    assert freq.dtype == torch.float32 and freq.shape == (32, 2)
    # theirs are made in fp32, a power and a few products: 2^-20 of them
    assert bool(((freq.double().sum(1) - inv.double()).abs() <= inv.double() * 2.0 ** -20).all())
    assert abs(scale - attention) <= 1e-6


def test_default_and_parts():
    plan = RotaryPlan(8, 10000.0)
    freq, scale = plan.on(torch.device("cpu"), torch.arange(3)[None])
    want = 10000.0 ** (-torch.arange(0, 8, 2, dtype=torch.float64) / 8)
    assert scale == 1.0 and bool(((freq.double().sum(1) - want).abs() <= want * 2.0 ** -46).all())
    assert RotaryPlan(0, 10000.0).on(torch.device("cpu"), torch.arange(3)[None])[0].shape == (0, 2)


@pytest.mark.parametrize("dims,parameters,more,error", [
    (8, dict(rope_type="proportional"), {}, NotImplementedError), (7, {}, {}, ValueError), (8, dict(rope_type="linear"), {}, ValueError),
    (8, dict(rope_type="llama3", factor=8.0), {}, ValueError), (8, dict(rope_type="yarn", factor=8.0), {}, ValueError),
    (8, dict(rope_type="longrope", short_factor=[1.0] * 4), dict(max_positions=100), ValueError),
    (8, dict(rope_type="longrope", short_factor=[1.0] * 4, long_factor=[1.0] * 3), dict(max_positions=100), ValueError)])
def test_what_a_plan_refuses(dims, parameters, more, error):
    with pytest.raises(error):
        RotaryPlan(dims, 10000.0, parameters, **more)


@pytest.mark.parametrize("kind", ["llama3", "yarn", "longrope", "dynamic"])
def test_eager_tables(kind):
    """On the CPU the tables of a scaled embedding are cos and sin of 64-bit angles, times the scale, and the rotation uses them."""
    config = _config(kind)
    rot = RotaryEmbedding(config)
    pos = torch.tensor([[0, 7, 4000, 90000]])
    tables = rot(torch.zeros(1, dtype=torch.float32), pos)
    assert isinstance(tables, RotaryTables) and tables.turn is None
    freq, scale = rot.plan.on(torch.device("cpu"), pos)
    angle = pos[..., None].double() * freq.double().sum(1)
    for got, want in zip(tables, (angle.cos(), angle.sin())):
        assert bool(((got.double() - torch.cat([want, want], -1) * scale).abs() <= 2.0 ** -23 * max(1.0, scale)).all())
    q, k = torch.randn(1, 2, 4, 64), torch.randn(1, 1, 4, 64)
    for a, b in zip(rotate(q, k, tables), apply_rotary_pos_emb(q, k, *tables)):
        assert torch.equal(a, b)


def test_the_default_embedding_is_as_it_was():
    config = TrimKVLlamaConfig(vocab_size=64, hidden_size=128, intermediate_size=64, num_hidden_layers=1, num_attention_heads=2,
                               num_key_value_heads=1, head_dim=64, rope_theta=5e5)
    pos = torch.arange(5, 25)[None]
    for dt in (torch.float32, torch.bfloat16):
        cos, sin = RotaryEmbedding(config)(torch.zeros(1, dtype=dt), pos)
        inv = 1.0 / (5e5 ** (torch.arange(0, 64, 2, dtype=torch.int64).float() / 64))
        emb = torch.cat([pos[..., None].float() * inv] * 2, -1)
        assert torch.equal(cos, emb.cos().to(dt)) and torch.equal(sin, emb.sin().to(dt))
    assert math.isclose(RotaryEmbedding(config).plan.base, 5e5)
