"""Block operators back to back on the same buffers, each kernel starting while the one that writes its operands still runs:
every result equals that of the same calls with the device waited for in between."""
import pytest
import torch

from test_block_e8m0_gpu import _data

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K", [(1, 2048, 4096), (40, 520, 1040), (300, 1024, 2048), (2304, 2176, 640)])
def test_operands_rewritten_between_calls(qlib, dev, M, N, K):
    sets = [(_data(M, K, torch.bfloat16, dev, 50 + i, 1.0), _data(N, K, torch.bfloat16, dev, 60 + i, 1.0)) for i in range(3)]
    a, b = qlib.quantize_block(sets[0][0]), qlib.quantize_block(sets[0][1])
    at = qlib.requantize_block(*a)
    c, back = torch.empty(M, N, device=dev), torch.empty(M, K, dtype=torch.bfloat16, device=dev)

    def step(x, w, between):
        for call in (lambda: qlib.quantize_block(x, out=a), lambda: qlib.quantize_block(w, out=b),
                     lambda: qlib.fp8_block_mm_e8m0(a[0], b[0], a[1], b[1], c), lambda: qlib.requantize_block(*a, out=at),
                     lambda: qlib.dequantize_block(*a, out=back)):
            call()
            between()
        return [t.clone() for t in (c, back, at[0].view(torch.uint8), at[1].view(torch.uint8))]

    want = [step(x, w, torch.cuda.synchronize) for x, w in sets]
    got = [step(x, w, lambda: None) for _ in range(10) for x, w in sets]
    for i, outs in enumerate(got):
        for g, r in zip(outs, want[i % 3]):
            assert torch.equal(g, r), i


@pytest.mark.parametrize("K,settings", [(4096, {"TILE_M": 48}), (4096, {"TILE_M": 64, "TILE_N": 256}), (4096, {"SLICES": 3}),
                                        (896, {"SLICES": 8})])
def test_settings_that_no_form_has_are_set_aside(qlib, dev, monkeypatch, K, settings):
    """The call then takes the form it would have taken without them, recognised by the order of its fp32 sums."""
    a, sa = qlib.quantize_block(_data(64, K, torch.float32, dev, 1))
    b, sb = qlib.quantize_block(_data(520, K, torch.float32, dev, 2))

    def product(**env):
        for name in ("TILE_M", "TILE_N", "SLICES"):
            monkeypatch.delenv("QGEMM_E8M0_" + name, raising=False)
        for name, value in env.items():
            monkeypatch.setenv("QGEMM_E8M0_" + name, str(value))
        qlib.lib().qgemm_reload_env()
        c = torch.empty(64, 520, device=dev)
        qlib.fp8_block_mm_e8m0(a, b, sa, sb, c)
        return c

    try:
        free, one_slice = product(), product(TILE_M=16, SLICES=1)
        assert not torch.equal(free, one_slice)  # or the comparison would show nothing
        assert torch.equal(product(**settings), free)
    finally:
        monkeypatch.undo()
        qlib.lib().qgemm_reload_env()
