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


def test_saved_tensors_come_back_as_the_kernels_take_them():
    from qgemm_b200.linear import _as_saved
    g = torch.Generator().manual_seed(1)
    codes = torch.randint(0, 120, (130, 77), generator=g, dtype=torch.uint8).view(torch.float8_e4m3fn)  # padding lost
    scale = torch.randint(0, 255, (2, 1), generator=g, dtype=torch.uint8).view(torch.float8_e8m0fnu).t()
    wide = torch.randint(0, 255, (1000,), generator=g, dtype=torch.uint8)
    moved = wide[3 - wide.data_ptr() % 16:][:900]  # 3 bytes past a boundary
    buffer, (c, s) = _as_saved(moved, (codes, scale))
    assert buffer.data_ptr() % 16 == 0 and torch.equal(buffer, moved)
    assert c.data_ptr() % 16 == 0 and c.stride() == (80, 1) and torch.equal(c.view(torch.uint8), codes.view(torch.uint8))
    assert s.is_contiguous() and torch.equal(s.view(torch.uint8), scale.view(torch.uint8))
    for kept in (_as_saved(buffer, (c, s)), _as_saved(buffer, ())):  # what fits is not copied
        assert kept[0] is buffer and (kept[1] is None or kept[1][0] is c)
    assert _as_saved(None, None) == (None, None)
