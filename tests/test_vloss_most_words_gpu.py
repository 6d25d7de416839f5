"""The largest vocabularies that the entry points take, in every form."""
import pytest

from tests.test_vloss_gpu import BF, SF, _check, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("v", [65535 * 128, 65535 * 128 + 1, 1 << 23])
@pytest.mark.parametrize("dtype,t,h", [(BF, 2, 3), (SF, 2, 1), (SF, 3, 8), (BF, 6, 8)])
def test_many_words(dtype, t, h, v):
    _check(*_inputs(t, v, h, dtype, seed=9), reduction="mean")
