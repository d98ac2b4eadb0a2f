"""The 8-bit linear layer inside autograd, where it is not called in the plain way."""
import pytest
import torch
from torch.autograd import forward_ad

from test_block_e8m0_gpu import _data

pytestmark = pytest.mark.gpu


def test_forward_mode_tangents_are_refused(qlib, dev):
    """And a dual level in which these tensors have no tangent changes nothing."""
    from qgemm_b200.linear import fp8_linear
    x, w = _data(9, 256, torch.bfloat16, dev, 1), _data(40, 256, torch.bfloat16, dev, 2)
    want = fp8_linear(x, w)
    with forward_ad.dual_level():
        for pair in ((forward_ad.make_dual(x, torch.ones_like(x)), w), (x, forward_ad.make_dual(w, torch.ones_like(w)))):
            with pytest.raises(qlib.QgemmError) as e:
                fp8_linear(*pair)
            assert e.value.status == qlib.ERR_UNSUPPORTED
        assert torch.equal(fp8_linear(x, w), want)
