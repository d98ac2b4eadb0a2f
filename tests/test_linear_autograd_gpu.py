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


def test_overwritten_tensors_are_noticed(qlib, dev):
    """Every call that writes into a caller's tensor counts as a change of it in place."""
    from qgemm_b200.linear import fp8_linear, fp8_linear_backward, fp8_linear_forward, pack_weight
    x, w = _data(40, 256, torch.bfloat16, dev, 1), _data(40, 256, torch.float32, dev, 2)
    q, s, qt, st = qlib.quantize_block(x, form="both")
    back, c, dw = torch.zeros(40, 256, device=dev), torch.zeros(40, 40, device=dev), torch.zeros(40, 256, device=dev)
    y, saved = fp8_linear_forward(x, w)
    calls = [((q, s), lambda: qlib.quantize_block(x, out=(q, s))),
             ((q, s, qt, st), lambda: qlib.quantize_block(x, form="both", out=(q, s, qt, st))),
             ((qt, st), lambda: qlib.requantize_block(q, s, out=(qt, st))),
             ((back,), lambda: qlib.dequantize_block(q, s, out=back)),
             ((c,), lambda: qlib.fp8_block_mm_e8m0(q, q, s, s, c)),
             ((c,), lambda: qlib.fp8_block_mm_e8m0(q, q, s, s, c, accumulate=True)),
             ((dw,), lambda: fp8_linear_backward(y, saved, dw=dw)),
             ((dw,), lambda: fp8_linear_backward(y, saved, dw=dw, accumulate=True))]
    for tensors, call in calls:
        before = [t._version for t in tensors]
        call()
        assert all(t._version > b for t, b in zip(tensors, before))
    with torch.inference_mode():
        qlib.dequantize_block(q, s, out=back)
        qlib.dequantize_block(q, s, out=torch.zeros(40, 256, device=dev))  # a tensor without a version
    p = torch.ones(40, 256, device=dev, requires_grad=True)
    z = (p * back).sum()  # keeps `back` for p's gradient
    qlib.dequantize_block(q, s, out=back)
    with pytest.raises(RuntimeError):
        z.backward()
    packed = pack_weight(w, backward=True)
    xi = x.clone().requires_grad_(True)
    y = fp8_linear(xi, packed)
    qlib.quantize_block(w, square=True, form="both", out=(packed.codes, packed.scale, packed.codes_t, packed.scale_t))
    with pytest.raises(RuntimeError):
        y.sum().backward()


def _unaligned(t):
    """An equal tensor three bytes past a boundary, without the original's padding."""
    buf = torch.empty(t.numel() * t.element_size() + 16, dtype=torch.uint8, device=t.device)
    flat = buf[3:3 + t.numel() * t.element_size()]
    flat.copy_(t.contiguous().view(-1).view(torch.uint8))
    return flat.view(t.dtype).view(t.shape)


@pytest.mark.parametrize("out_features", [128, 130])
@pytest.mark.parametrize("packed", [False, True])
def test_saved_tensor_hooks(qlib, dev, out_features, packed):
    """Saved tensors kept on the host, or anywhere else on the device, until the backward pass."""
    from qgemm_b200.linear import fp8_linear, pack_weight
    x, w = _data(33, 200, torch.bfloat16, dev, 1), _data(out_features, 200, torch.float32, dev, 2)
    dy = _data(33, out_features, torch.bfloat16, dev, 3)

    def gradients():
        xi, wi = x.clone().requires_grad_(True), w.clone().requires_grad_(not packed)
        y = fp8_linear(xi, pack_weight(wi, backward=True) if packed else wi)
        return xi, wi, y

    xi, wi, y = gradients()
    y.backward(dy)
    want = (xi.grad, wi.grad)
    for hooks in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.save_on_cpu(pin_memory=True),
                  torch.autograd.graph.saved_tensors_hooks(_unaligned, lambda t: t)):
        with hooks:
            xi, wi, y = gradients()
        y.backward(dy)
        assert torch.equal(xi.grad, want[0])
        assert packed or torch.equal(wi.grad, want[1])


def test_recomputed_in_the_backward_pass(qlib, dev):
    from torch.utils.checkpoint import checkpoint

    from qgemm_b200.linear import fp8_linear
    x, w = _data(33, 200, torch.bfloat16, dev, 1), _data(130, 200, torch.float32, dev, 2)
    got = []
    for again in (False, True):
        xi, wi = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        y = checkpoint(fp8_linear, xi, wi, use_reentrant=False) if again else fp8_linear(xi, wi)
        y.square().sum().backward()
        got.append((y.detach(), xi.grad, wi.grad))
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("need_dx,need_dw", [(True, True), (False, True), (True, False)])
def test_backward_on_another_stream_keeps_what_was_saved(qlib, dev, need_dx, need_dw):
    """The backward pass is queued behind a delay on a second stream and `saved` dropped at once: the forward's stream, which
    takes memory and writes to it meanwhile, must not be given the saved codes' memory."""
    from qgemm_b200.linear import fp8_linear_backward, fp8_linear_forward
    x, w = _data(300, 1024, torch.bfloat16, dev, 1), _data(900, 1024, torch.bfloat16, dev, 2)
    dy = _data(300, 900, torch.bfloat16, dev, 3)
    want = fp8_linear_backward(dy, fp8_linear_forward(x, w, need_dx, need_dw)[1])
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(one):
        saved = fp8_linear_forward(x, w, need_dx, need_dw)[1]
        size = saved.buffer.numel()
    two.wait_stream(one)
    with torch.cuda.stream(two):
        torch.cuda._sleep(100_000_000)  # about 50 ms
        got = fp8_linear_backward(dy, saved)
    del saved
    with torch.cuda.stream(one):
        others = [torch.full((size,), 0x7F, dtype=torch.uint8, device=dev) for _ in range(4)]
    torch.cuda.synchronize()
    for g, r in zip(got, want):
        assert (g is None and r is None) or torch.equal(g, r)
    del others


@pytest.mark.parametrize("weight", ["cast", "transposed"])
def test_capture_beside_a_living_graph_of_a_derived_weight_is_refused(qlib, dev, weight):
    from qgemm_b200.linear import fp8_linear
    x = _data(20, 64, torch.bfloat16, dev, 1)
    w = _data(64, 64, torch.float32, dev, 2).requires_grad_(True)
    derive = {"cast": lambda: w.to(torch.bfloat16), "transposed": lambda: w.t()}[weight]
    alive = fp8_linear(x, derive())
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(qlib.QgemmError) as e:
        with torch.cuda.graph(graph):
            fp8_linear(x, w)
    assert e.value.status == qlib.ERR_UNSUPPORTED
    alive.sum().backward()
    assert w.grad.shape == w.shape


def test_capture_beside_a_side_streams_graph_that_the_default_stream_used_too(qlib, dev):
    """The leaf's node was made by a call on a side stream and is still alive; a later call on the default stream does not
    make it that one's."""
    from qgemm_b200.linear import fp8_linear
    x = _data(20, 256, torch.bfloat16, dev, 1)
    w = _data(40, 256, torch.float32, dev, 2).requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = fp8_linear(x, w)
    torch.cuda.current_stream().wait_stream(side)
    want, = torch.autograd.grad(fp8_linear(x, w).sum(), w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got, = torch.autograd.grad(fp8_linear(x, w).sum(), w)
    got.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    del alive


@pytest.mark.parametrize("tokens", [1, 2, 129])
@pytest.mark.parametrize("fin", [1, 15, 128])
@pytest.mark.parametrize("fout", [1, 17, 129])
def test_smallest_layers(qlib, dev, tokens, fin, fout):
    from test_block_e8m0_gpu import _assert_close
    from test_fp8_linear_gpu import _formula

    from qgemm_b200.linear import fp8_linear
    x, w = (_data(r, fin, torch.float32, dev, r, 0.5).requires_grad_(True) for r in (tokens, fout))
    dy = _data(tokens, fout, torch.float32, dev, 3, 0.5)
    y = fp8_linear(x, w)
    for got, (ref, mags, k) in zip((y, *torch.autograd.grad(y, (x, w), dy)), _formula(x, w, dy)):
        _assert_close(got.detach(), ref, mags, k, torch.float32)


def test_threads_with_streams_of_their_own(qlib, dev):
    """Forward and backward in four threads at once."""
    import threading

    from qgemm_b200.linear import fp8_linear
    sets = [(_data(100 + i, 512, torch.bfloat16, dev, i, 0.5), _data(300, 512, torch.float32, dev, 9 + i, 0.5)) for i in range(4)]

    def step(x, w):
        xi, wi = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        y = fp8_linear(xi, wi)
        return (y.detach(), *torch.autograd.grad(y.sum(), (xi, wi)))

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    got = [[] for _ in sets]

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got[i].append(step(*sets[i]))
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(4):
        assert len(got[i]) == 20
        for outs in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))
