"""The block-scaled product at the edges of C and of the scales' range. Tolerances: as derived in test_block_sums_gpu.py for the
sums, half a step of the output type, and half a step of fp16's subnormals."""
import pytest
import torch

from block_reference import E4M3, E8M0, values
from test_block_e8m0_gpu import HALF_STEP, TYPES, VARIANTS, _operands, _product
from test_block_sums_gpu import _bound

pytestmark = pytest.mark.gpu


def _close(c, ref, mags, K):
    tol = _bound(K, mags) + HALF_STEP[c.dtype] * ref.abs() * (1 + 2.0 ** -7)
    if c.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    return bool(((c.double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("tile_m,tile_n,slices", VARIANTS)
@pytest.mark.parametrize("M,N,K", [(33, 300, 1100), (301, 521, 1100), (259, 388, 1040)])
def test_neighbours_of_an_aligned_result_stay(qlib, dev, monkeypatch, tile_m, tile_n, slices, M, N, K):
    """C cut out of a wider matrix such that rows start on vectors, so that the copy engine and vector stores write it: nothing
    beside its N columns or its M rows changes."""
    a, sa, b, sb = _operands(qlib, dev, M, N, K, False, True, M + N, 1.0)
    sa = (sa.view(torch.uint8) - 12).view(E8M0)  # within fp16's range
    ref, mags = _product(a, sa, b, sb)
    for name, value in (("TILE_M", tile_m), ("TILE_N", tile_n), ("SLICES", slices)):
        monkeypatch.setenv("QGEMM_E8M0_" + name, str(value))
    qlib.lib().qgemm_reload_env()
    try:
        for out in TYPES:
            for accumulate in (False, True) if out == torch.float32 else (False,):
                wide = torch.full((M + 300, -(-N // 16) * 16 + 32), 3.0, dtype=out, device=dev)
                c = wide[8:M + 8, 16:N + 16]
                assert c.data_ptr() % 16 == 0 and c.stride(0) * c.element_size() % 16 == 0
                want, m = (ref + 3, mags + 3) if accumulate else (ref, mags)
                qlib.fp8_block_mm_e8m0(a, b, sa, sb, c, accumulate=accumulate)
                assert _close(c, want, m, K), (out, accumulate)
                c.fill_(3.0)
                assert bool((wide == 3).all()), (out, accumulate)
        rc, st = qlib.device_status()
    finally:
        monkeypatch.undo()
        qlib.lib().qgemm_reload_env()
    assert rc == 0, st


@pytest.mark.parametrize("M,N,K", [(1, 300, 640), (64, 520, 1040), (300, 520, 1040), (1100, 1300, 512)])
@pytest.mark.parametrize("side", ["a", "b"])
def test_the_smallest_scale(qlib, dev, M, N, K, side):
    """Scale byte 0, 2^-127, which the quantisers give to tiny blocks, against the largest, 254; and quantised blocks that
    small against plain ones."""
    g = torch.Generator().manual_seed(3)
    a, b = (torch.randint(8, 0x70, (n, -(-K // 16) * 16), generator=g, dtype=torch.uint8).to(dev).view(E4M3)[:, :K] for n in (M, N))
    kb = -(-K // 128)
    low, high = torch.zeros(kb, 1, dtype=torch.uint8), torch.full((kb, 1), 254, dtype=torch.uint8)
    low[::2] = 1
    sa, sb = ((low, high) if side == "a" else (high, low))
    sa, sb = (s.expand(kb, n).contiguous().to(dev).view(E8M0) for s, n in ((sa, M), (sb, N)))
    ref, mags = _product(a, sa, b, sb)
    c = torch.empty(M, N, device=dev)
    qlib.fp8_block_mm_e8m0(a, b, sa, sb, c)
    assert _close(c, ref, mags, K)
    tiny, plain = (torch.randn(n, K, generator=g).to(dev) for n in (M, N))
    q, s = qlib.quantize_block(tiny * 2.0 ** -122)
    w, ws = qlib.quantize_block(plain * 2.0 ** 60)
    assert int(s.view(torch.uint8).max()) <= 1
    ref, mags = _product(q, s, w, ws)
    qlib.fp8_block_mm_e8m0(q, w, s, ws, c)
    assert _close(c, ref, mags, K)


@pytest.mark.parametrize("tile_m,tile_n,slices", VARIANTS)
@pytest.mark.parametrize("K", [1025, 1031, 1100, 1151])
def test_codes_behind_the_last_of_a_row_do_not_count(qlib, dev, monkeypatch, tile_m, tile_n, slices, K):
    """K that ends inside a 16-byte unit, with NaN codes behind it in every row and in rows behind the last."""
    M, N = 33, 150
    a, sa, b, sb = _operands(qlib, dev, M, N, K, False, True, K, 1.0)
    ref, mags = _product(a, sa, b, sb)
    padded = []
    for t in (a, b):
        buf = torch.full((t.shape[0] + 260, -(-K // 16) * 16 + 16), 0x7F, dtype=torch.uint8, device=dev).view(E4M3)
        view = buf[:t.shape[0], :K]
        view.view(torch.uint8).copy_(t.view(torch.uint8))
        padded.append(view)
    for name, value in (("TILE_M", tile_m), ("TILE_N", tile_n), ("SLICES", slices)):
        monkeypatch.setenv("QGEMM_E8M0_" + name, str(value))
    qlib.lib().qgemm_reload_env()
    try:
        c = torch.empty(M, N, device=dev)
        qlib.fp8_block_mm_e8m0(*padded, sa, sb, c)
        rc, st = qlib.device_status()
    finally:
        monkeypatch.undo()
        qlib.lib().qgemm_reload_env()
    assert rc == 0, st
    assert _close(c, ref, mags, K)


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("N", [249, 252, 255, 257, 300, 383])
def test_a_row_of_nan_stays_in_its_columns(qlib, dev, monkeypatch, out, N):
    """The last columns where they end inside a 16-byte unit, with a NaN row, accumulating and not, next to numbers."""
    M, K = 300, 256
    a, sa, b, sb = _operands(qlib, dev, M, N, K, False, False, N, 0.2)
    a.view(torch.uint8)[7] = 0x7F
    monkeypatch.setenv("QGEMM_E8M0_TILE_M", "256")
    monkeypatch.setenv("QGEMM_E8M0_SLICES", "1")
    qlib.lib().qgemm_reload_env()
    try:
        for accumulate in (False, True) if out == torch.float32 else (False,):
            wide = torch.full((M + 2, 416), 3.0, dtype=out, device=dev)
            c = wide[1:M + 1, 16:N + 16]
            qlib.fp8_block_mm_e8m0(a, b, sa, sb, c, accumulate=accumulate)
            assert bool(torch.isnan(c[7]).all()) and not bool(torch.isnan(c[:7]).any())
            c.fill_(3.0)
            assert bool((wide == 3).all())
    finally:
        monkeypatch.undo()
        qlib.lib().qgemm_reload_env()


@pytest.mark.parametrize("rows,cols", [(1, 129), (127, 250), (129, 131), (257, 385), (300, 1001), (385, 119)])
@pytest.mark.parametrize("square", [False, True])
def test_neighbours_of_aligned_codes_and_values_stay(qlib, dev, rows, cols, square):
    """Codes and restored values cut out of wider matrices whose rows start on vectors."""
    x = torch.randn(rows, cols, generator=torch.Generator().manual_seed(rows)).to(dev)
    want = qlib.quantize_block(x, square=square, form="both")

    def cut(r, c):
        buf = torch.full((r + 2, -(-c // 16) * 16 + 32), 0x55, dtype=torch.uint8, device=dev)
        return buf, buf.view(E4M3)[1:r + 1, 16:c + 16]

    def untouched(buf, view):
        view.view(torch.uint8 if buf.dtype == torch.uint8 else buf.dtype).fill_(0x55)
        return bool((buf == 0x55).all())

    (qb, q), (tb, qt) = cut(rows, cols), cut(cols, rows)
    s, st = torch.empty_like(want[1]), torch.empty_like(want[3])
    for source in (x, x.bfloat16()):
        ref = qlib.quantize_block(source, square=square, form="both")
        qlib.quantize_block(source, square=square, form="both", out=(q, s, qt, st))
        for got, r in zip((q, s, qt, st), ref):
            assert torch.equal(got.view(torch.uint8), r.view(torch.uint8))
        assert untouched(qb, q) and untouched(tb, qt)
    if not square:
        ref = qlib.requantize_block(want[0], want[1])
        qlib.requantize_block(want[0], want[1], out=(qt, st))
        assert torch.equal(qt.view(torch.uint8), ref[0].view(torch.uint8)) and untouched(tb, qt)
    for out in TYPES:
        buf = torch.full((rows + 2, -(-cols // 16) * 16 + 32), 0x55, dtype=out, device=dev)
        back = buf[1:rows + 1, 16:cols + 16]
        qlib.dequantize_block(want[0], want[1], out=back)
        assert torch.equal(back, qlib.dequantize_block(want[0], want[1], out)) and untouched(buf, back)
