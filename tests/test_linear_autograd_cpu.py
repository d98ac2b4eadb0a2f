"""What the 8-bit linear layer does about autograd before it touches a GPU."""
import pytest
import torch
from torch.autograd import forward_ad


@pytest.mark.parametrize("of", ["x", "weight", "x of a packed weight"])
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_tangents_are_refused(qlib, of, grad):
    from qgemm_b200.linear import PackedWeight, fp8_linear
    x, w = torch.ones(4, 128), torch.ones(32, 128)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        if of == "weight":
            w = forward_ad.make_dual(w, torch.ones_like(w))
        else:
            x = forward_ad.make_dual(x, torch.ones_like(x))
        if of == "x of a packed weight":
            w = PackedWeight(w.to(torch.float8_e4m3fn), torch.ones(1, 1).to(torch.float8_e8m0fnu))
        with pytest.raises(qlib.QgemmError) as e:
            fp8_linear(x, w)
    assert e.value.status == qlib.ERR_UNSUPPORTED
