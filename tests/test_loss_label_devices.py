"""Labels that are still on the CPU, as a data loader gives them, with a model on the GPU."""
import pytest
import torch

import trimkv_b200 as t
from tests import dafovik_cases
from tests.test_loss_heads import _model

pytestmark = pytest.mark.gpu


def test_labels_on_the_cpu():
    model = _model().cuda()
    ids = torch.randint(1, 131, (2, 9), generator=torch.Generator().manual_seed(5))
    want = model(input_ids=ids.cuda(), labels=ids.cuda()).loss
    assert torch.equal(model(input_ids=ids.cuda(), labels=ids).loss, want)
    moved = torch.nn.functional.pad(ids[:, 1:], (0, 1), value=-100)
    assert torch.equal(model(input_ids=ids.cuda(), shift_labels=moved).loss, want)


@pytest.mark.parametrize("padded", [False, True])
def test_labels_on_the_cpu_of_a_hybrid_decoder(padded, tmp_path):
    cfg = dafovik_cases.CONFIGS["mixed"]
    dafovik_cases.write_checkpoint(tmp_path, cfg, dafovik_cases.random_tensors(cfg))
    model = t.DafovikForCausalLM.from_pretrained(str(tmp_path), dtype=torch.float32).cuda()
    ids = torch.randint(0, cfg["vocab"], (2, 9), generator=torch.Generator().manual_seed(5))
    mask = torch.ones_like(ids).cuda()
    mask[1, 5:] = 0 if padded else 1
    with torch.no_grad():
        want = model(input_ids=ids.cuda(), attention_mask=mask, labels=ids.cuda()).loss
        assert torch.equal(model(input_ids=ids.cuda(), attention_mask=mask, labels=ids).loss, want)
        moved = torch.nn.functional.pad(ids[:, 1:], (0, 1), value=-100)
        a, b = (model(input_ids=ids.cuda(), attention_mask=mask, shift_labels=x).loss for x in (moved, moved.cuda()))
        assert torch.equal(a, b)
