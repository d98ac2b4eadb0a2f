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


def _mark(t):
    from qgemm_b200.linear import _STREAM, _leaf_node, _node
    return _leaf_node(_node(t)).metadata.get(_STREAM)


class _Layer(torch.autograd.Function):
    """Stands in for the layer: a node whose inputs are x and the weight."""
    @staticmethod
    def forward(ctx, x, w):
        return x @ w.t()

    @staticmethod
    def backward(ctx, dy):
        return None, None


def _call(stream, capturing, x, w):
    from qgemm_b200.linear import _note_nodes, _probe_nodes
    if stream:
        _probe_nodes(capturing, x, w)
    y = _Layer.apply(x, w)
    _note_nodes(y, stream)
    return y


def _refusal(qlib, x, w):
    """The status of a refused capture (the error itself would keep its frames' tensors alive)."""
    try:
        _call(7, True, x, w)
    except qlib.QgemmError as e:
        return e.status


def test_leaf_nodes_are_found_through_casts_and_transposes(qlib):
    from qgemm_b200.linear import _leaf_node, _node
    w = torch.ones(4, 4, requires_grad=True)
    keep = w * 2
    own = _leaf_node(_node(w))
    for t in (w, w.t(), w.to(torch.bfloat16), w.t().to(torch.bfloat16), w.view(2, 8).t().half().t()):
        assert _leaf_node(_node(t)) is own
    two = w + torch.ones(4, 4, requires_grad=True)
    far = w.t().t().t().t().t()
    assert _leaf_node(_node(two)) is None and _leaf_node(_node(far)) is None
    del keep


def test_captures_beside_default_stream_graphs(qlib):
    """Streams as numbers: 0 is the default one. A refusal as long as the earlier graph lives, for the leaf itself, for a cast
    or a transpose of it, and for a leaf that another operation's graph holds besides."""
    x, w = torch.ones(2, 4), torch.ones(4, 4, requires_grad=True)
    for weight in (lambda: w, lambda: w.to(torch.bfloat16).float(), lambda: w.t()):
        alive = _call(0, False, x, weight())
        for again in (weight, lambda: w):
            assert _refusal(qlib, x, again()) == qlib.ERR_UNSUPPORTED
        del alive
        _call(7, True, x, weight())
    regulariser = w.square().sum()
    alive = _call(0, False, x, w)
    assert _refusal(qlib, x, w) == qlib.ERR_UNSUPPORTED
    del regulariser, alive
    xg = torch.ones(2, 4, requires_grad=True)
    alive = _call(0, False, xg, w)
    assert _refusal(qlib, xg, torch.ones(4, 4, requires_grad=True)) == qlib.ERR_UNSUPPORTED
    del alive
    _call(7, True, xg, w)


def test_captures_beside_graphs_of_other_streams(qlib):
    """A node that a call on another stream made stays that stream's whatever uses it later; one that only other operations
    made says nothing, so a capture goes on, until a default-stream call has met it."""
    x, w = torch.ones(2, 4), torch.ones(4, 4, requires_grad=True)
    first = _call(5, False, x, w)
    assert _mark(w) == 5
    second = _call(0, False, x, w)
    assert _mark(w) == 5
    third = _call(7, True, x, w)
    del first, second
    assert _mark(w) == 5
    del third
    assert _mark(w) is None
    held = _call(7, True, x, w)  # a capture's own
    alive = _call(0, False, x, w)
    _call(7, True, x, w)
    del held, alive
    other = w.square()
    captured = _call(7, True, x, w)
    assert _mark(w) is None
    alive = _call(0, False, x, w)
    assert _mark(w) == 0
    del captured, alive, other
