"""One column of labelled tokens where the mask leaves some requests out: only the others take part in the step."""
from types import SimpleNamespace

import pytest
import torch
import torch.nn.functional as F

import trimkv_b200 as t
from tests import dafovik_cases, lonulix_cases
from trimkv_b200.modeling_hybrid import HybridForCausalLM


@pytest.mark.parametrize("mask,steps", [(None, (None, None, 3)), ([[1], [1], [1]], (None, None, 3)), ([[1], [0], [1]], ([1, 1], [0, 2], 2))])
def test_which_requests_take_part(mask, steps):
    seen = []

    def packed_hidden(ids, cache, lengths, rows):
        seen.append((lengths, rows, len(ids)))
        return torch.zeros(len(ids), 4)
    model = SimpleNamespace(packed_hidden=packed_hidden, head=lambda n: n, _loss_of_packed=lambda normed, live, labels, kw: normed.sum())
    ids = torch.tensor([[3], [4], [5]])
    out = HybridForCausalLM.forward(model, input_ids=ids, attention_mask=None if mask is None else torch.tensor(mask),
                                    past_key_values=SimpleNamespace(_batch=3), shift_labels=ids)
    assert seen == [steps] and out.logits.shape == (3, 1, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("design", ["lonulix", "dafovik"])
def test_the_other_request_stays_where_it_was(design, tmp_path):
    cases, cls = {"lonulix": (lonulix_cases, t.LonulixForCausalLM), "dafovik": (dafovik_cases, t.DafovikForCausalLM)}[design]
    cfg = cases.CONFIGS["mixed"]
    dafovik_cases.write_checkpoint(tmp_path, cfg, cases.random_tensors(cfg))
    model = cls.from_pretrained(str(tmp_path), dtype=torch.float32).cuda()
    ids = torch.randint(0, cfg["vocab"], (2, 9), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    scored, packed = model.new_cache(), model.new_cache()
    with torch.no_grad():
        for cache in (scored, packed):
            model(input_ids=ids[:, :5], past_key_values=cache)
        out = model(input_ids=ids[:, 5:6], attention_mask=torch.tensor([[1], [0]], device="cuda"), past_key_values=scored, shift_labels=ids[:, 6:7])
        alone = model.forward_packed(ids[0, 5:6], packed, [1], [0])
        assert torch.equal(out.logits[0], alone) and not bool(out.logits[1].any())
        want = F.cross_entropy(alone.double(), ids[0, 6:7])
        assert abs(float(out.loss) - float(want)) <= 2.0 ** -12      # fp32 logits below 2^5 of a hundred products: 2^-17 each
        assert scored._len == packed._len
        after = [model(input_ids=ids[:, 7:8], past_key_values=cache).logits for cache in (scored, packed)]
        assert torch.equal(*after)
