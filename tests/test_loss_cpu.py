"""forward(labels=...) where the kernels do not run: on the CPU, and in 64 bits, the loss is that of the logits."""
import pytest
import torch
import torch.nn.functional as F

from tests.test_loss_heads import OnePass, _check, _model


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2.0 ** -18), (torch.float64, 2.0 ** -40), (torch.bfloat16, 2.0 ** -14)])
def test_a_pass_with_labels(dtype, tol):
    _check(_model(dtype), tol)


def test_a_pass_with_labels_already_moved():
    model = _model()
    ids = torch.randint(1, 131, (2, 9), generator=torch.Generator().manual_seed(5))
    with torch.no_grad():
        out = model(input_ids=ids, shift_labels=ids, past_key_values=OnePass(), ignore_index=int(ids[0, 0]))
        want = F.cross_entropy(out.logits.double().flatten(0, 1), ids.flatten(), ignore_index=int(ids[0, 0]))
    assert abs(float(out.loss) - float(want)) <= 2.0 ** -18 * float(want)


@pytest.mark.gpu
def test_a_pass_in_64_bits():
    """On the GPU too, with a stand-in for the cache, whose kernels take no 64-bit rows."""
    model = _model(torch.float64).cuda()
    ids = torch.randint(1, 131, (2, 9), generator=torch.Generator().manual_seed(5)).cuda()
    with torch.no_grad():
        out = model(input_ids=ids, labels=ids, past_key_values=OnePass())
        want = F.cross_entropy(out.logits[:, :-1].flatten(0, 1), ids[:, 1:].flatten())
    assert abs(float(out.loss) - float(want)) <= 2.0 ** -40 * float(want)
