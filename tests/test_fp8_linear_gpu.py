"""The 8-bit linear layer: forward and backward run together, against the layer's formula in 64 bits, with gradients also
against differences; captured into a graph; over micro-batches; with a packed weight.

Tolerance of each product: as derived in test_block_e8m0_gpu.py. Quantised operands are bit-exact on either side."""
import math

import pytest
import torch

from block_reference import quantize, values
from test_block_e8m0_gpu import _assert_close, _data

pytestmark = pytest.mark.gpu


def _q(x, square=False):
    return values(*quantize(x, square))


def _formula(x, w, dy):
    """[(value, sum of magnitudes, summed length)] of y, dx, dw in 64 bits."""
    dev = x.device
    xq, wq = _q(x), _q(w, True)
    along, across, xt = _q(dy), _q(dy.t()), _q(xq.t())
    pairs = [(xq, wq.t(), w.shape[1]), (along, wq, w.shape[0]), (across, xt.t(), x.shape[0])]
    return [((a.to(dev) @ b.to(dev)), (a.abs().to(dev) @ b.abs().to(dev)), k) for a, b, k in pairs]


@pytest.mark.parametrize("tokens,fin,fout", [(1, 256, 128), (7, 1040, 520), (200, 129, 77), (333, 640, 1040), (2100, 520, 2200)])
@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16),
                                          (torch.float16, torch.float16), (torch.float32, torch.float32)])
def test_layer_matches_its_formula(qlib, dev, tokens, fin, fout, dtype, wdtype):
    from qgemm_b200.linear import fp8_linear
    x = _data(tokens, fin, dtype, dev, 1, 0.5).requires_grad_(True)
    w = (_data(fout, fin, torch.float32, dev, 2, 0.2) / math.sqrt(fin)).to(wdtype).requires_grad_(True)
    dy = (_data(tokens, fout, torch.float32, dev, 3, 0.5) * 0.1).to(dtype)
    y = fp8_linear(x, w)
    assert y.dtype == dtype
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert dx.dtype == dtype and dw.dtype == wdtype
    for got, (ref, mags, k) in zip((y, dx, dw), _formula(x, w, dy)):
        _assert_close(got.detach(), ref, mags, k, got.dtype)
    rc, st = qlib.device_status()
    assert rc == 0, st


def test_gradients_against_differences(qlib, dev):
    """On values the codes hold exactly (small whole numbers, steps that stay so) the layer is a plain product, and a
    difference quotient along any direction of such steps is exact: sum(dy * (f(x + d) - f(x))) = sum(dx * d)."""
    from qgemm_b200.linear import fp8_linear
    g = torch.Generator().manual_seed(4)
    whole = lambda r, c, lo, hi: torch.randint(lo, hi, (r, c), generator=g).float().to(dev)  # noqa: E731
    tokens, fin, fout = 150, 200, 260
    x, w, dy = whole(tokens, fin, -3, 4), whole(fout, fin, -3, 4), whole(tokens, fout, -3, 4)
    ex, ew = whole(tokens, fin, -1, 2), whole(fout, fin, -1, 2)
    x.requires_grad_(True)
    w.requires_grad_(True)
    dx, dw = torch.autograd.grad(fp8_linear(x, w), (x, w), dy)
    with torch.no_grad():
        by_x = (dy.double() * (fp8_linear(x + ex, w) - fp8_linear(x, w)).double()).sum()
        by_w = (dy.double() * (fp8_linear(x, w + ew) - fp8_linear(x, w)).double()).sum()
    assert float(by_x) == float((dx.double() * ex.double()).sum())
    assert float(by_w) == float((dw.double() * ew.double()).sum())


def test_only_the_gradients_asked_for(qlib, dev):
    from qgemm_b200.linear import fp8_linear, fp8_linear_backward, fp8_linear_forward
    x, w = _data(70, 256, torch.bfloat16, dev, 1), _data(130, 256, torch.float32, dev, 2)
    dy = _data(70, 130, torch.bfloat16, dev, 3)
    y, saved = fp8_linear_forward(x, w)
    dx, dw = fp8_linear_backward(dy, saved)
    for need_x, need_w in ((True, False), (False, True)):
        xi, wi = x.clone().requires_grad_(need_x), w.clone().requires_grad_(need_w)
        out = fp8_linear(xi, wi)
        assert torch.equal(out, y)
        out.backward(dy)
        assert (xi.grad is not None) == need_x and (wi.grad is not None) == need_w
        if need_x:
            assert torch.equal(xi.grad, dx)
        if need_w:
            assert torch.equal(wi.grad, dw)
    with torch.no_grad():
        assert torch.equal(fp8_linear(x.requires_grad_(True), w), y)


def test_shapes_layouts_and_broadcast_gradients(qlib, dev):
    """Leading dimensions of any number, a transposed x, and y.sum(), whose gradient is one value broadcast."""
    from qgemm_b200.linear import fp8_linear
    x, w = _data(60, 256, torch.bfloat16, dev, 1), _data(130, 256, torch.bfloat16, dev, 2)
    y = fp8_linear(x, w)
    assert torch.equal(fp8_linear(x.view(3, 4, 5, 256), w), y.view(3, 4, 5, 130))
    assert torch.equal(fp8_linear(x[0], w), y[0])
    xt = x.t().contiguous().t()
    assert torch.equal(fp8_linear(xt, w), y)
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    fp8_linear(a, b).sum().backward()
    c, d = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    fp8_linear(c, d).backward(torch.ones_like(y))
    assert torch.equal(a.grad, c.grad) and torch.equal(b.grad, d.grad)
    empty = fp8_linear(x[:0].clone().requires_grad_(True), b)
    assert empty.shape == (0, 130)
    b.grad = None
    empty.sum().backward()
    assert bool((b.grad == 0).all())


def test_micro_batches_add_up(qlib, dev):
    from qgemm_b200.linear import fp8_linear_backward, fp8_linear_forward
    w = _data(200, 384, torch.float32, dev, 2, 0.5)
    total = torch.zeros(200, 384, device=dev)
    want = torch.zeros(200, 384, dtype=torch.float64, device=dev)
    mags = want.clone()
    for i, tokens in enumerate((64, 1, 130)):
        x, dy = _data(tokens, 384, torch.bfloat16, dev, 10 + i, 0.5), _data(tokens, 200, torch.bfloat16, dev, 20 + i, 0.5)
        _, saved = fp8_linear_forward(x, w, need_dx=False)
        dx, dw = fp8_linear_backward(dy, saved, dw=total, accumulate=True)
        assert dx is None and dw is total
        ref, m, _ = _formula(x, w, dy)[2]
        want += ref
        mags += m + want.abs()
    _assert_close(total, want, mags, 256, torch.float32)


def test_packed_weight(qlib, dev):
    from qgemm_b200.linear import fp8_linear, pack_weight
    x, w = _data(5, 512, torch.float16, dev, 1, 0.3), _data(300, 512, torch.float16, dev, 2, 0.3)
    y = fp8_linear(x, w)
    p = pack_weight(w)
    assert p.codes_t is None and torch.equal(fp8_linear(x, p), y)
    xi, xj = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    with pytest.raises(qlib.QgemmError):
        fp8_linear(xi, p)
    dy = torch.ones_like(y)
    fp8_linear(xi, pack_weight(w, backward=True)).backward(dy)
    fp8_linear(xj, w).backward(dy)
    assert torch.equal(xi.grad, xj.grad)


def test_checkpoint_restores_the_activation(qlib, dev):
    from qgemm_b200.linear import fp8_linear_forward
    x, w = _data(90, 512, torch.bfloat16, dev, 1), _data(64, 512, torch.bfloat16, dev, 2)
    _, saved = fp8_linear_forward(x, w)
    codes, scale = saved.x
    assert codes.element_size() == 1 and codes.shape == x.shape
    back = qlib.dequantize_block(codes, scale, torch.bfloat16)
    assert torch.equal(back.cpu(), _q(x).to(torch.float32).to(torch.bfloat16))


def test_checkpoint_of_no_tokens_and_none_kept(qlib, dev):
    from qgemm_b200.linear import fp8_linear_forward
    x, w = _data(5, 512, torch.bfloat16, dev, 1), _data(130, 512, torch.bfloat16, dev, 2)
    codes, scale = fp8_linear_forward(x[:0], w, need_dx=False)[1].x
    assert codes.shape == (0, 512) and scale.shape == (4, 0)
    assert fp8_linear_forward(x, w, need_dw=False)[1].x is None


def _captured(step):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    return graph, held


@pytest.mark.parametrize("autograd", [True, False])
def test_captured_step_replays_on_new_inputs(qlib, dev, autograd):
    """Forward and backward in one graph, replayed on other values; without autograd also while an eager graph of the same
    leaves is alive."""
    from qgemm_b200.linear import fp8_linear, fp8_linear_backward, fp8_linear_forward
    x = _data(140, 384, torch.bfloat16, dev, 1, 0.5).requires_grad_(True)
    w = _data(260, 384, torch.float32, dev, 2, 0.5).requires_grad_(True)
    dy = _data(140, 260, torch.bfloat16, dev, 3, 0.5)

    def step():
        if autograd:
            y = fp8_linear(x, w)
            return (y.detach(), *torch.autograd.grad(y, (x, w), dy))
        y, saved = fp8_linear_forward(x, w)
        return (y, *fp8_linear_backward(dy, saved))

    alive = None if autograd else fp8_linear(x, w)
    graph, held = _captured(step)
    for seed in (5, 6):
        with torch.no_grad():
            x.copy_(_data(140, 384, torch.bfloat16, dev, seed, 0.5))
            w.copy_(_data(260, 384, torch.float32, dev, seed + 1, 0.5))
            dy.copy_(_data(140, 260, torch.bfloat16, dev, seed + 2, 0.5))
        graph.replay()
        for got, want in zip(held, step()):
            assert torch.equal(got, want)
    del alive


def test_capture_beside_a_living_graph_is_refused(qlib, dev):
    from qgemm_b200.linear import fp8_linear
    x = _data(20, 256, torch.bfloat16, dev, 1)
    w = _data(40, 256, torch.float32, dev, 2).requires_grad_(True)
    alive = fp8_linear(x, w)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(qlib.QgemmError):
        with torch.cuda.graph(graph):
            fp8_linear(x, w)
    alive.sum().backward()  # and nothing is broken by it
    assert w.grad.shape == w.shape
    want = w.grad.clone()
    del alive
    w.grad = None
    _captured(lambda: fp8_linear(x, w).sum().backward())[0].replay()
    w.grad.zero_()
    graph, _ = _captured(lambda: fp8_linear(x, w).sum().backward())
    w.grad.zero_()
    graph.replay()
    assert torch.equal(w.grad, want)


def test_capture_beside_a_graph_of_another_side_stream(qlib, dev):
    """Only the default stream's graphs hinder a capture."""
    from qgemm_b200.linear import fp8_linear
    x = _data(20, 256, torch.bfloat16, dev, 1)
    w = _data(40, 256, torch.float32, dev, 2).requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = fp8_linear(x, w)
        want, = torch.autograd.grad(fp8_linear(x, w).sum(), w)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got, = torch.autograd.grad(fp8_linear(x, w).sum(), w)
        got.zero_()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    del alive


def test_two_streams_at_once(qlib, dev):
    """The operators share no scratch: layers on two streams, nothing ordering them, each get their own results."""
    from qgemm_b200.linear import fp8_linear
    sets = []
    for i in range(2):
        x, w = _data(300 + i, 1024, torch.bfloat16, dev, 30 + i, 0.5), _data(900, 1024, torch.bfloat16, dev, 40 + i, 0.5)
        sets.append((x, w, fp8_linear(x, w)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(fp8_linear(sets[i][0], sets[i][1]))
    torch.cuda.synchronize()
    for i in range(2):
        for y in outs[i]:
            assert torch.equal(y, sets[i][2])


def test_layer_refusals(qlib, dev):
    from qgemm_b200.linear import fp8_linear, fp8_linear_backward, fp8_linear_forward, pack_weight
    x, w = torch.ones(4, 64, device=dev), torch.ones(32, 64, device=dev)
    with pytest.raises(qlib.QgemmError):
        fp8_linear(x[:, :32], w)
    with pytest.raises(qlib.QgemmError):
        fp8_linear(x.double(), w)
    with pytest.raises(qlib.QgemmError):
        fp8_linear(x, w.to(torch.int8))
    with pytest.raises(qlib.QgemmError):
        fp8_linear(x.cpu(), w)
    with pytest.raises(qlib.QgemmError):
        pack_weight(w[0])
    y, saved = fp8_linear_forward(x, w)
    with pytest.raises(qlib.QgemmError):
        fp8_linear_backward(y[:2], saved)
    with pytest.raises(qlib.QgemmError):
        fp8_linear_backward(y, saved, accumulate=True)
    with pytest.raises(qlib.QgemmError):
        fp8_linear_backward(y, saved, dw=torch.zeros(32, 64, device=dev, dtype=torch.bfloat16), accumulate=True)
    with pytest.raises(qlib.QgemmError):
        fp8_linear_backward(y, saved, dw=torch.zeros(31, 64, device=dev))


def test_broadcast_input_gets_the_sum_of_its_gradients(qlib, dev):
    from qgemm_b200.linear import fp8_linear
    base, w = _data(1, 256, torch.float32, dev, 1), _data(130, 256, torch.float32, dev, 2)
    dy = _data(9, 130, torch.float32, dev, 3)
    b = base.clone().requires_grad_(True)
    fp8_linear(b.expand(9, 256), w).backward(dy)
    full = base.expand(9, 256).clone().requires_grad_(True)
    fp8_linear(full, w).backward(dy)
    assert torch.equal(b.grad, full.grad.sum(0, keepdim=True))
    # one weight in two layers of one graph
    x, u = _data(20, 130, torch.float32, dev, 4, 0.5), _data(130, 130, torch.float32, dev, 5, 0.5).requires_grad_(True)
    y = fp8_linear(x, u)
    z = fp8_linear(y, u)
    z.sum().backward()
    first = y.detach().requires_grad_(True)
    v = u.detach().clone().requires_grad_(True)
    fp8_linear(first, v).sum().backward()
    t = u.detach().clone().requires_grad_(True)
    fp8_linear(x, t).backward(first.grad)
    assert torch.equal(u.grad, v.grad + t.grad) or torch.equal(u.grad, t.grad + v.grad)


def test_backward_twice_and_on_another_thread(qlib, dev):
    import threading

    from qgemm_b200.linear import fp8_linear
    x, w = _data(33, 256, torch.bfloat16, dev, 1).requires_grad_(True), _data(140, 256, torch.bfloat16, dev, 2).requires_grad_(True)
    dy = _data(33, 140, torch.bfloat16, dev, 3)
    y = fp8_linear(x, w)
    one = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    two = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    got = []
    t = threading.Thread(target=lambda: got.extend(torch.autograd.grad(y, (x, w), dy)))
    t.start()
    t.join()
    for a, b, c in zip(one, two, got):
        assert torch.equal(a, b) and torch.equal(a, c)
