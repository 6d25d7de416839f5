"""Which of a configuration's lengths the scaled frequencies go by, against transformers' own embedding of the same configuration."""
import pytest
import torch
from transformers import LlamaConfig
from transformers.models.llama.modeling_llama import LlamaRotaryEmbedding

from trimkv_b200 import TrimKVLlamaConfig
from trimkv_b200.modeling_trimkv import RotaryEmbedding
from trimkv_b200.positions import RotaryPlan

KINDS = {
    "linear": dict(factor=4.0),
    "llama3": dict(factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0),
    "yarn": dict(factor=4.0),
    "longrope": dict(factor=4.0, short_factor=[1.0 + 0.01 * i for i in range(32)], long_factor=[1.0 + 0.9 * i for i in range(32)]),
    "longrope factor": dict(short_factor=[1.0 + 0.01 * i for i in range(32)], long_factor=[1.0 + 0.9 * i for i in range(32)]),
    "dynamic": dict(factor=4.0),
}


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("key,attribute", [(None, None), (4096, None), (None, 4096), (8192, 4096)])
@pytest.mark.parametrize("length", [1000, 5000, 20000])
def test_lengths_are_taken_as_transformers_takes_them(kind, key, attribute, length):
    rope = dict(KINDS[kind], rope_type=kind.split()[0], rope_theta=1e4)
    more = {} if attribute is None else dict(original_max_position_embeddings=attribute)
    if key is not None:
        rope["original_max_position_embeddings"] = key
    kw = dict(vocab_size=64, hidden_size=128, intermediate_size=64, num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=1, head_dim=64,
              max_position_embeddings=16384, **more)
    pos = torch.arange(length - 5, length)[None]
    theirs = LlamaRotaryEmbedding(LlamaConfig(**kw, rope_parameters=dict(rope)))(torch.zeros(1), pos)
    ours = RotaryEmbedding(TrimKVLlamaConfig(**kw, rope_parameters=dict(rope)))(torch.zeros(1), pos)
    # theirs: frequencies in fp32 (a power and a few products, 2^-20 of them) times a position, cosines of that in fp32; scaled by up to 1.5
    for a, b in zip(ours, theirs):
        assert float((a - b).abs().max()) <= 1.5 * (length * 2.0 ** -20 + 2.0 ** -20)


def test_dynamic_without_a_longest_position():
    """Nothing else to go by: the key counts."""
    p = dict(rope_type="dynamic", factor=2.0, original_max_position_embeddings=100)
    assert RotaryPlan(8, 1e4, p).original == 100 and RotaryPlan(8, 1e4, p, 300).original == 300
    with pytest.raises(ValueError):
        RotaryPlan(8, 1e4, dict(rope_type="dynamic", factor=2.0))
