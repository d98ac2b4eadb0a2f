"""Block quantisation with power-of-two scales, the 8-bit checkpoint's two ways back, and the product of such operands,
against 64-bit references.

Quantised results are compared bit for bit: the scale follows from a comparison and x * 2^-E is exact, so a code has one
rounding, which both sides make to nearest even. The product's tolerance: the tensor core adds K/32 groups of exact products
(two 4-bit significands) to a fp32 sum, at most one fp32 step, 2^-23, of the running magnitude lost per group and at most
another 2^-23 where the group's products are aligned to one another; S <= 8 slices are added on top. So |error| <=
(2 * ceil(K/32) + 8) * 2^-23 * sum |a b|, plus half a step of the output type."""
import math

import pytest
import torch

from block_reference import E4M3, E8M0, bytes_of, quantize, values

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _data(rows, cols, dtype, dev, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp2(torch.randn(rows, 1, generator=g) * spread)
    return x.to(dtype).to(dev)


def _check_forms(qlib, x, square, forms=("row", "column", "both")):
    q_ref, s_ref = quantize(x, square)
    qt_ref, st_ref = quantize(x.t(), square)
    for form in forms:
        out = qlib.quantize_block(x, square=square, form=form)
        if form != "column":
            assert torch.equal(bytes_of(out[1]), s_ref), form
            assert torch.equal(bytes_of(out[0]), q_ref), form
        if form != "row":
            assert torch.equal(bytes_of(out[-1]), st_ref), form
            assert torch.equal(bytes_of(out[-2]), qt_ref), form


SIZES = [(1, 1), (1, 7168), (5, 16), (128, 128), (127, 129), (129, 127), (300, 520), (257, 1000), (1000, 3)]


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("square", [False, True])
def test_quantize_block_is_exact(qlib, dev, rows, cols, dtype, square):
    _check_forms(qlib, _data(rows, cols, dtype, dev, rows * 7 + cols), square)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("square", [False, True])
def test_quantize_block_reads_and_writes_strided(qlib, dev, dtype, square):
    """Odd offsets and leading dimensions on either side; what lies around the matrices stays as it was."""
    wide = _data(260, 411, dtype, dev, 5)
    x = wide[3:250, 7:340]  # 247 x 333, not on a vector boundary
    rows, cols = x.shape
    q_ref, s_ref = quantize(x, square)
    qt_ref, st_ref = quantize(x.t(), square)
    qb = torch.full((rows + 2, cols + 13), 0x55, dtype=torch.uint8, device=dev)
    tb = torch.full((cols + 2, rows + 9), 0x55, dtype=torch.uint8, device=dev)
    q, qt = qb.view(E4M3)[1:rows + 1, 5:cols + 5], tb.view(E4M3)[1:cols + 1, 3:rows + 3]
    s = torch.empty(s_ref.shape, dtype=E8M0, device=dev)
    st = torch.empty(st_ref.shape, dtype=E8M0, device=dev)
    got = qlib.quantize_block(x, square=square, form="both", out=(q, s, qt, st))
    assert got[0].data_ptr() == q.data_ptr()
    assert torch.equal(bytes_of(q), q_ref) and torch.equal(bytes_of(s), s_ref)
    assert torch.equal(bytes_of(qt), qt_ref) and torch.equal(bytes_of(st), st_ref)
    for buf, view in ((qb, q), (tb, qt)):
        view.view(torch.uint8).fill_(0x55)
        assert bool((buf == 0x55).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("square", [False, True])
def test_quantize_block_special_values(qlib, dev, dtype, square):
    """Zeros, infinities, NaN, the type's largest and smallest values, and maxima on and next to 448 * 2^e."""
    x = _data(384, 640, dtype, dev, 11, 1.0)
    fi = torch.finfo(dtype)
    x[0:128, 0:128] = 0
    x[1, 130] = float("inf")
    x[2, 260] = float("nan")
    x[3, 390] = -float("inf")
    x[130, 0:128] = fi.max
    x[131, 5] = fi.smallest_normal
    x[260:384, 128:256] = torch.finfo(dtype).tiny / 4  # subnormals
    x[200, 256:384] = 0
    x[200, 300] = 448.0
    x[201, 256:384] = 0
    x[201, 300] = 448.0 * (1 + fi.eps)
    x[202, 256:384] = 0
    x[202, 300] = -0.875
    x[256:384, 512:640] = -fi.max
    _check_forms(qlib, x, square)


def test_quantize_block_empty(qlib, dev):
    for rows, cols in ((0, 256), (256, 0), (0, 0)):
        for form in ("row", "column", "both"):
            out = qlib.quantize_block(torch.empty(rows, cols, device=dev), form=form)
            assert out[0].shape == ((rows, cols) if form != "column" else (cols, rows))


@pytest.mark.parametrize("rows,cols", SIZES + [(640, 384)])
@pytest.mark.parametrize("spread", [0.5, 3.0, 8.0])
def test_requantize_block_is_exact(qlib, dev, rows, cols, spread):
    """Rows near one another, at the limit of fp16 arithmetic (2^15 apart), and far beyond it."""
    q, s = qlib.quantize_block(_data(rows, cols, torch.float32, dev, 3 * rows + cols, spread))
    qt_ref, st_ref = quantize(values(q, s).t())
    qt, st = qlib.requantize_block(q, s)
    assert torch.equal(bytes_of(st), st_ref) and torch.equal(bytes_of(qt), qt_ref)


@pytest.mark.parametrize("shift", [0, 1, 14, 15, 16, 17])
@pytest.mark.parametrize("base", [0, 16, 120, 238])
def test_requantize_block_at_the_edges(qlib, dev, base, shift):
    """Scales exactly `shift` powers of two apart down to the smallest and up to the largest byte; columns of zeros, of
    the smallest codes alone, of 448 and next to it, of negative zeros, and one NaN code."""
    g = torch.Generator().manual_seed(7)
    codes = torch.randint(0, 256, (300, 400), generator=g, dtype=torch.uint8)
    codes[codes & 0x7F == 0x7F] = 0x7E
    codes[:, 5] = 0
    codes[:, 6] = 0x80
    codes[:, 7] = torch.randint(0, 2, (300,), generator=g, dtype=torch.uint8)  # 0 or 2^-9
    codes[:, 8] = 0x01
    codes[:, 9] = 0x08  # 2^-6
    codes[:, 10] = 0x07
    codes[:, 130] = 0xFE
    codes[3:9] = 0
    codes[200, 390] = 0x7F
    scale = (base + torch.randint(0, shift + 1, (4, 300), generator=g)).clamp(max=254).to(torch.uint8)
    scale[:, 0], scale[:, 1] = base, min(base + shift, 254)
    qt_ref, st_ref = quantize(values(codes, scale).t())
    qt, st = qlib.requantize_block(codes.to(dev).view(E4M3), scale.to(dev).view(E8M0))
    assert torch.equal(bytes_of(st), st_ref)
    assert torch.equal(bytes_of(qt), qt_ref)


def test_requantize_and_dequantize_every_code_and_scale(qlib, dev):
    """All 256 codes (NaN among them) under all 256 scale bytes: rows of one scale, columns of one code, so that a
    column's block meets 128 neighbouring scales."""
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1).contiguous()
    scale = torch.arange(256, dtype=torch.uint8).repeat(2, 1).contiguous()
    q, s = codes.to(dev).view(E4M3), scale.to(dev).view(E8M0)
    ref = values(codes, scale)
    qt_ref, st_ref = quantize(ref.t())
    qt, st = qlib.requantize_block(q, s)
    assert torch.equal(bytes_of(st), st_ref)
    assert torch.equal(bytes_of(qt), qt_ref)
    # single rows: each scale alone, down to 2^-127 and up to 2^127
    for e in (0, 1, 7, 8, 9, 127, 246, 253, 254):
        one = torch.full((2, 1), e, dtype=torch.uint8)
        qt_ref, st_ref = quantize(values(codes[:1], one).t())
        qt, st = qlib.requantize_block(q[:1], one.to(dev).view(E8M0))
        assert torch.equal(bytes_of(st), st_ref), e
        assert torch.equal(bytes_of(qt), qt_ref), e
    for dtype in TYPES:
        got = qlib.dequantize_block(q, s, dtype).cpu()
        want = ref.to(torch.float32).to(dtype)  # the first step is exact, or overflows as the second would
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        ok = ~torch.isnan(want)
        assert torch.equal(got[ok], want[ok])


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("square", [False, True])
def test_dequantize_block_is_exact(qlib, dev, rows, cols, dtype, square):
    q, s = qlib.quantize_block(_data(rows, cols, torch.float32, dev, rows + cols), square=square)
    got = qlib.dequantize_block(q, s, dtype)
    assert torch.equal(got.cpu(), values(q, s).to(torch.float32).to(dtype))
    buf = torch.full((rows, cols + 5), 7.0, dtype=dtype, device=dev)
    qlib.dequantize_block(q, s, out=buf[:, 3:cols + 3])
    assert torch.equal(buf[:, 3:cols + 3], got)
    assert bool((buf[:, :3] == 7).all()) and bool((buf[:, cols + 3:] == 7).all())


# ------------------------------------------------------------------------------------------------ the product
def _operands(qlib, dev, M, N, K, a_square, b_square, seed, spread=2.0):
    a, sa = qlib.quantize_block(_data(M, K, torch.float32, dev, seed, spread), square=a_square)
    b, sb = qlib.quantize_block(_data(N, K, torch.float32, dev, seed + 1, spread), square=b_square)
    return a, sa, b, sb


def _product(a, sa, b, sb):
    """(reference, sum of magnitudes) in 64 bits, on the GPU for speed."""
    av, bv = values(a, sa).to(a.device), values(b, sb).to(a.device)
    return (av @ bv.t()), (av.abs() @ bv.abs().t())


def _assert_close(got, ref, mags, K, dtype):
    tol = (2 * math.ceil(K / 32) + 8) * 2.0 ** -23 * mags + HALF_STEP[dtype] * ref.abs() * (1 + 2.0 ** -7)
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half a step of its subnormals
    err = (got.double() - ref).abs()
    worst = float((err - tol).max())
    assert worst <= 0, f"error {float(err.max())} exceeds its bound by {worst}"


PRODUCTS = [(1, 128, 128), (1, 7168, 2048), (2, 1, 1), (3, 17, 129), (16, 256, 640), (17, 520, 384), (33, 1000, 1040),
            (64, 2048, 4096), (100, 200, 520), (128, 384, 256), (130, 77, 256), (300, 520, 1040), (520, 1100, 1536),
            (1024, 2048, 640), (2100, 2300, 900)]


@pytest.mark.parametrize("M,N,K", PRODUCTS)
@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("a_square,b_square", [(False, True), (False, False), (True, False)])
def test_product_matches_64_bits(qlib, dev, M, N, K, out, a_square, b_square):
    a, sa, b, sb = _operands(qlib, dev, M, N, K, a_square, b_square, M + N + K)
    ref, mags = _product(a, sa, b, sb)
    if out == torch.float16:  # keep within its range: scaled down exactly, by a power of two
        down = 2.0 ** math.ceil(math.log2(max(float(ref.abs().max()), 1.0) / 2.0 ** 14))
        sa = (sa.view(torch.uint8) - int(math.log2(down))).view(E8M0)
        ref, mags = ref / down, mags / down
    c = torch.full((M, N), float("nan"), dtype=out, device=dev)
    qlib.fp8_block_mm_e8m0(a, b, sa, sb, c)
    _assert_close(c, ref, mags, K, out)
    again = torch.zeros_like(c)
    qlib.fp8_block_mm_e8m0(a, b, sa, sb, again)
    assert torch.equal(c, again)
    rc, st = qlib.device_status()
    assert rc == 0, st


VARIANTS = [(tm, 128, s) for tm in (16, 32, 64) for s in (1, 2, 4, 8)] + [(256, 256, 1), (256, 128, 1), (256, 128, 2)]


@pytest.mark.parametrize("tile_m,tile_n,slices", VARIANTS)
@pytest.mark.parametrize("M,N,K", [(1, 40, 1100), (300, 520, 1400), (777, 900, 1025)])
def test_every_kernel_form(qlib, dev, monkeypatch, tile_m, tile_n, slices, M, N, K):
    """Each tile and slice count the library has, whatever it would choose: same product, sums and neighbours kept."""
    a, sa, b, sb = _operands(qlib, dev, M, N, K, False, False, M + K)
    ref, mags = _product(a, sa, b, sb)
    old = torch.randn(M, N, device=dev)
    monkeypatch.setenv("QGEMM_E8M0_TILE_M", str(tile_m))
    monkeypatch.setenv("QGEMM_E8M0_TILE_N", str(tile_n))
    monkeypatch.setenv("QGEMM_E8M0_SLICES", str(slices))
    qlib.lib().qgemm_reload_env()
    try:
        c16 = torch.empty(M, N, dtype=torch.bfloat16, device=dev)
        qlib.fp8_block_mm_e8m0(a, b, sa, sb, c16)
        wide = torch.full((M + 1, N + 9), 3.0, device=dev)
        c = wide[:M, 4:N + 4]
        c.copy_(old)
        qlib.fp8_block_mm_e8m0(a, b, sa, sb, c, accumulate=True)
        rc, st = qlib.device_status()
    finally:
        monkeypatch.undo()
        qlib.lib().qgemm_reload_env()
    assert rc == 0, st
    _assert_close(c16, ref, mags, K, torch.bfloat16)
    _assert_close(c, ref + old.double(), mags + old.abs().double(), K, torch.float32)
    assert bool((wide[:, :4] == 3).all()) and bool((wide[:, N + 4:] == 3).all()) and bool((wide[M] == 3).all())


@pytest.mark.parametrize("M,N,K", [(1, 300, 384), (64, 2048, 1000), (300, 520, 1040), (777, 2048, 4001), (2304, 2176, 384)])
def test_product_accumulates(qlib, dev, M, N, K):
    a, sa, b, sb = _operands(qlib, dev, M, N, K, False, False, M + N)
    ref, mags = _product(a, sa, b, sb)
    old = torch.randn(M, N, device=dev) * float(ref.abs().mean())
    c = old.clone()
    qlib.fp8_block_mm_e8m0(a, b, sa, sb, c, accumulate=True)
    _assert_close(c, ref + old.double(), mags + old.abs().double(), K, torch.float32)
    wide = torch.full((M, N + 7), 3.0, device=dev)  # no vector boundary anywhere, and neighbours to leave alone
    c = wide[:, 3:N + 3]
    c.copy_(old)
    qlib.fp8_block_mm_e8m0(a, b, sa, sb, c, accumulate=True)
    _assert_close(c, ref + old.double(), mags + old.abs().double(), K, torch.float32)
    assert bool((wide[:, :3] == 3).all()) and bool((wide[:, N + 3:] == 3).all())


@pytest.mark.parametrize("M,N,K", [(16, 512, 512), (300, 512, 256), (512, 512, 16384), (2048, 2048, 128)])
def test_accumulating_takes_tiny_numbers_as_zeros(qlib, dev, M, N, K):
    """On every way to C alike: vectors, rows, TMA. 2^-126 itself and what is larger stay."""
    zeros = lambda r: torch.zeros(r, K, device=dev)  # noqa: E731
    (a, sa), (b, sb) = qlib.quantize_block(zeros(M)), qlib.quantize_block(zeros(N), square=True)
    old = torch.randint(0, 4, (M, N), device=dev)
    held = torch.tensor([2.0 ** -126, 2.0 ** -127, -2.0 ** -149, -3.5], device=dev)
    want = torch.tensor([2.0 ** -126, 0.0, 0.0, -3.5], device=dev)[old]
    for off in (0, 1):
        c = torch.empty(M * N + 4, device=dev)[off:off + M * N].view(M, N)
        c.copy_(held[old])
        qlib.fp8_block_mm_e8m0(a, b, sa, sb, c, accumulate=True)
        assert torch.equal(c, want)


@pytest.mark.parametrize("M,N,K", [(5, 300, 384), (300, 520, 1040), (2100, 2300, 256)])
@pytest.mark.parametrize("out", TYPES)
def test_product_strided(qlib, dev, M, N, K, out):
    """Operands cut out of wider matrices, C at an odd offset."""
    a, sa, b, sb = _operands(qlib, dev, M, N, K, False, True, 3)
    wa = torch.zeros(M + 1, (K // 16 + 4) * 16, dtype=torch.uint8, device=dev).view(E4M3)
    wb = torch.zeros(N + 1, (K // 16 + 5) * 16, dtype=torch.uint8, device=dev).view(E4M3)
    wa.view(torch.uint8).fill_(0x7F)  # NaN all around
    wb.view(torch.uint8).fill_(0x7F)
    va, vb = wa[1:, 16:16 + K], wb[1:, 32:32 + K]
    va.view(torch.uint8).copy_(a.view(torch.uint8))
    vb.view(torch.uint8).copy_(b.view(torch.uint8))
    wide = torch.full((M + 2, N + 7), 3.0, dtype=out, device=dev)
    c = wide[1:M + 1, 5:N + 5]
    down = 2.0 ** 20 if out == torch.float16 else 1.0
    sa = (sa.view(torch.uint8) - int(math.log2(down))).view(E8M0)
    qlib.fp8_block_mm_e8m0(va, vb, sa, sb, c)
    ref, mags = _product(a, sa, b, sb)
    _assert_close(c, ref, mags, K, out)
    c.fill_(3.0)
    assert bool((wide == 3).all())


def test_product_scales_far_apart(qlib, dev):
    """Scale bytes over the whole range whose products cancel out, one element of each K block at a time."""
    M, N, K = 130, 140, 1024
    a = torch.zeros(M, K, dtype=torch.uint8)
    b = torch.zeros(N, K, dtype=torch.uint8)
    g = torch.Generator().manual_seed(2)
    kb = K // 128
    at = torch.randint(0, 128, (kb,), generator=g) + torch.arange(kb) * 128
    a[:, at] = torch.randint(8, 120, (M, kb), generator=g, dtype=torch.uint8)
    b[:, at] = torch.randint(8, 120, (N, kb), generator=g, dtype=torch.uint8)
    ea = torch.randint(1, 254, (kb, 1), generator=g)
    sa = (ea + torch.zeros(kb, M, dtype=torch.int64)).to(torch.uint8)
    sb = (254 - ea + torch.randint(-3, 4, (kb, N), generator=g)).clamp(1, 254).to(torch.uint8)
    a, b, sa, sb = a.to(dev).view(E4M3), b.to(dev).view(E4M3), sa.to(dev).view(E8M0), sb.to(dev).view(E8M0)
    ref, mags = _product(a, sa, b, sb)
    c = torch.empty(M, N, device=dev)
    qlib.fp8_block_mm_e8m0(a, b, sa, sb, c)
    _assert_close(c, ref, mags, K, torch.float32)


def test_product_nan_blocks_reach_their_rows_only(qlib, dev):
    x = _data(200, 512, torch.bfloat16, dev, 1, 1.0)
    w = _data(300, 512, torch.bfloat16, dev, 2, 1.0)
    x[7, 130] = float("inf")
    w[250, 400] = float("nan")
    a, sa = qlib.quantize_block(x)
    b, sb = qlib.quantize_block(w)
    c = torch.empty(200, 300, device=dev)
    qlib.fp8_block_mm_e8m0(a, b, sa, sb, c)
    bad = torch.zeros(200, 300, dtype=torch.bool, device=dev)
    bad[7], bad[:, 250] = True, True
    assert torch.equal(torch.isnan(c), bad)
    # a NaN scale over finite codes
    sb2 = sb.view(torch.uint8).clone()
    sb2[1, 3] = 255
    qlib.fp8_block_mm_e8m0(a, b, sa, sb2.view(E8M0), c)
    bad[:, 3] = True
    assert torch.equal(torch.isnan(c), bad)


@pytest.mark.parametrize("M,N,K", [(16, 128, 70000), (256, 256, 40001), (600, 700, 16500), (1000, 1100, 6145)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_long_sums_keep_32_bits(qlib, dev, M, N, K, accumulate):
    """A fp32 result's error does not grow with K. The tensor cores' additions truncate; over one chain of 8192 signed terms
    that was measured as 8.6e-7 of the result's norm, in proportion to the length, so the 6144 that a chain may have lose
    6.5e-7, and parts that are added with a rounding each lose no more than that together. 1e-6 leaves half as much again;
    one chain over the longest K here would be 1.3e-5 off."""
    a, sa, b, sb = _operands(qlib, dev, M, N, K, False, False, 21, 0.5)
    ref, mags = _product(a, sa, b, sb)
    c = torch.randn(M, N, device=dev) * float(ref.abs().mean()) if accumulate else torch.empty(M, N, device=dev)
    want = ref + c.double() if accumulate else ref
    qlib.fp8_block_mm_e8m0(a, b, sa, sb, c, accumulate=accumulate)
    assert float((c.double() - want).norm() / want.norm()) <= 1e-6
    again = c.clone()
    if not accumulate:
        qlib.fp8_block_mm_e8m0(a, b, sa, sb, again)
        assert torch.equal(again, c)


@pytest.mark.parametrize("M,N,K", [(5, 300, 1000), (333, 259, 700), (1030, 1021, 384)])
def test_product_scales_at_any_address(qlib, dev, M, N, K):
    """Scales whose rows start on no word boundary, at every offset."""
    a, sa, b, sb = _operands(qlib, dev, M, N, K, False, False, 9)
    c, want = torch.empty(M, N, device=dev), torch.empty(M, N, device=dev)
    qlib.fp8_block_mm_e8m0(a, b, sa, sb, want)
    for off in (1, 2, 3):
        moved = []
        for s in (sa, sb):
            buf = torch.full((s.numel() + 8,), 255, dtype=torch.uint8, device=dev)
            m = buf[off:off + s.numel()].view(s.shape)
            m.copy_(s.view(torch.uint8))
            moved.append(m.view(E8M0))
        qlib.fp8_block_mm_e8m0(a, b, *moved, c)
        assert torch.equal(c, want)


def test_product_empty(qlib, dev):
    e = lambda r, c: qlib.quantize_block(torch.ones(r, c, device=dev))  # noqa: E731
    for M, N, K in ((0, 128, 128), (128, 0, 128), (5, 7, 0)):
        (a, sa), (b, sb) = e(M, K), e(N, K)
        c = torch.full((M, N), 3.0, device=dev)
        qlib.fp8_block_mm_e8m0(a, b, sa, sb, c, accumulate=True)
        assert bool((c == 3).all())
        qlib.fp8_block_mm_e8m0(a, b, sa, sb, c)
        assert bool((c == 0).all())


# ------------------------------------------------------------------------------------------------ far, odd and refused calls
def test_offsets_past_32_bits(qlib, dev):
    """More than 2^32 elements: the last rows and columns of every result, on values made for them."""
    rows, cols = 66100, 65536
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=dev)
    tail = _data(300, 700, torch.bfloat16, dev, 1)
    x[-300:, -700:] = tail
    q, s, qt, st = qlib.quantize_block(x, form="both")
    first, lead = rows - 300, cols - 700
    start_c, start_r = lead // 128 * 128, first // 128 * 128  # whole blocks, the zeros in front included
    q_ref, s_ref = quantize(x[first:, start_c:])
    assert torch.equal(bytes_of(q[first:, start_c:]), q_ref)
    assert torch.equal(bytes_of(s)[start_c // 128:, first:], s_ref)
    qt_ref, st_ref = quantize(x[start_r:, lead:].t())
    assert torch.equal(bytes_of(qt[lead:, start_r:]), qt_ref)
    assert torch.equal(bytes_of(st)[start_r // 128:, lead:], st_ref)
    assert int(q.view(torch.uint8)[:first].count_nonzero()) == 0
    del x, qt, st
    back = torch.empty(rows, cols, dtype=torch.bfloat16, device=dev)
    qlib.dequantize_block(q, s, out=back)
    assert torch.equal(back[first:, start_c:].cpu(), values(q_ref, s_ref).to(torch.bfloat16))
    del back
    ct, cts = qlib.requantize_block(q, s)
    full = values(q[start_r:, start_c:], s[start_c // 128:, start_r:].contiguous())[:, lead - start_c:]
    ct_ref, cts_ref = quantize(full.t())
    assert torch.equal(bytes_of(ct[lead:, start_r:]), ct_ref)
    assert torch.equal(bytes_of(cts)[start_r // 128:, lead:], cts_ref)
    del ct, cts
    # a product whose A has more than 2^32 codes, and one whose C has more than 2^32 elements
    w = _data(24, cols, torch.bfloat16, dev, 2)
    b, sb = qlib.quantize_block(w)
    c = torch.empty(rows, 24, device=dev)
    qlib.fp8_block_mm_e8m0(q, b, s, sb, c)
    av = values(q[first:, start_c:], s[start_c // 128:, first:].contiguous())
    bv = values(b[:, start_c:], sb[start_c // 128:].contiguous())
    _assert_close(c[first:], (av @ bv.t()).to(dev), (av.abs() @ bv.abs().t()).to(dev), cols, torch.float32)
    assert int(c[:first].count_nonzero()) == 0
    del q, s, c
    (a, sa), (b, sb) = (qlib.quantize_block(_data(n, 64, torch.bfloat16, dev, n, 1.0)) for n in (66000, 65600))
    c = torch.empty(66000, 65600, dtype=torch.bfloat16, device=dev)
    qlib.fp8_block_mm_e8m0(a, b, sa, sb, c)
    av, bv = values(a[-300:], sa[:, -300:].contiguous()), values(b, sb)
    _assert_close(c[-300:], (av @ bv.t()).to(dev), (av.abs() @ bv.abs().t()).to(dev), 64, torch.bfloat16)


@pytest.mark.parametrize("tile_m,tile_n,slices", [(16, 128, 1), (32, 128, 8), (64, 128, 4), (256, 256, 1), (256, 128, 1), (256, 128, 2)])
def test_a_wait_that_runs_out_is_reported(qlib, dev, monkeypatch, tile_m, tile_n, slices):
    """The host leaves out the loads of one K block (a hook of the library): the issuer's wait for it ends after about a
    second, every role and every CTA of the cluster leaves, the status says where, and the next call is right."""
    M, N, K = (16, 128, 2048) if tile_m != 256 else (256, tile_n, 2048)
    a, sa, b, sb = _operands(qlib, dev, M, N, K, False, True, 5)
    ref, mags = _product(a, sa, b, sb)
    c = torch.empty(M, N, device=dev)
    monkeypatch.setenv("QGEMM_E8M0_TILE_M", str(tile_m))
    monkeypatch.setenv("QGEMM_E8M0_TILE_N", str(tile_n))
    monkeypatch.setenv("QGEMM_E8M0_SLICES", str(slices))
    qlib.lib().qgemm_reload_env()
    try:
        assert qlib.device_status()[0] == qlib.OK
        qlib.lib().qgemm_test_arm_skip_load(1)
        qlib.fp8_block_mm_e8m0(a, b, sa, sb, c)
        rc, st = qlib.device_status()
        assert rc == qlib.ERR_DEVICE_TIMEOUT
        # the MMA issuer, waiting for K block 1, or the producer, which within the same microseconds and for as long starts
        # to wait for that block's slot to come free
        assert st[0] == 1 and ((st[2] == 2 and st[3] == 1) or (st[2] == 1 and st[3] > 1)), st
        assert qlib.device_status()[0] == qlib.OK
        qlib.fp8_block_mm_e8m0(a, b, sa, sb, c)
        assert qlib.device_status()[0] == qlib.OK
    finally:
        monkeypatch.undo()
        qlib.lib().qgemm_reload_env()
    _assert_close(c, ref, mags, K, torch.float32)


def test_captured_on_a_side_stream_with_forms_not_used_before(qlib, dev):
    """A graph of quantiser and products of several sizes replays on new values, twice with other work between."""
    sizes = [(3, 1000, 384), (40, 264, 2176), (200, 520, 1152), (700, 800, 300), (1500, 1300, 256)]
    xs = [_data(m, k, torch.bfloat16, dev, m, 1.0) for m, _, k in sizes]
    ws = [_data(n, k, torch.float32, dev, n, 1.0) for _, n, k in sizes]

    def run():
        outs = []
        for x, w in zip(xs, ws):
            a, sa = qlib.quantize_block(x)
            b, sb = qlib.quantize_block(w, square=True)
            c = torch.empty(x.shape[0], w.shape[0], device=dev)
            qlib.fp8_block_mm_e8m0(a, b, sa, sb, c)
            t, st = qlib.requantize_block(a, sa)
            outs += [c, qlib.dequantize_block(a, sa), t.view(torch.uint8), st.view(torch.uint8)]
        return outs

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        held = run()
    for seed in (1, 2):
        for t in xs + ws:
            t.copy_(_data(*t.shape, t.dtype, dev, seed + t.shape[0], 1.0))
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        for h, w in zip(held, want):
            assert torch.equal(h, w)


def test_single_rows_columns_and_odd_strides(qlib, dev):
    wide = _data(70, 400, torch.bfloat16, dev, 3, 1.0)
    for x in (wide[:, 17:18], wide[5:6], wide[::3], wide[::2, 8:264], wide[3:4, 9:10]):
        _check_forms(qlib, x, False)
        _check_forms(qlib, x, True)
    for bad in (wide.t(), wide[:, ::2], wide[:, :1].t(), wide[:1].expand(70, 400), wide.view(70, 20, 20)):
        with pytest.raises(qlib.QgemmError) as e:
            qlib.quantize_block(bad)
        assert e.value.status == qlib.ERR_INVALID_ARG


def test_python_refusals(qlib, dev):
    x = _data(40, 256, torch.bfloat16, dev, 1)
    q, s, qt, st = qlib.quantize_block(x, form="both")
    c = torch.zeros(40, 40, device=dev)
    inv, uns, ali = qlib.ERR_INVALID_ARG, qlib.ERR_UNSUPPORTED, qlib.ERR_ALIGNMENT
    odd = torch.zeros(40, 272, dtype=torch.uint8, device=dev).view(E4M3)
    calls = [
        (inv, lambda: qlib.quantize_block(x, form="rows")),
        (uns, lambda: qlib.quantize_block(x.double())),
        (inv, lambda: qlib.quantize_block(x, out=(q, s, qt, st))),
        (inv, lambda: qlib.quantize_block(x, out=(qt, st))),
        (inv, lambda: qlib.quantize_block(x, out=(q, s.float()))),
        (inv, lambda: qlib.quantize_block(x, square=True, out=(q, s))),
        (inv, lambda: qlib.requantize_block(q.view(torch.uint8), s)),
        (inv, lambda: qlib.requantize_block(q, s[:1])),
        (uns, lambda: qlib.requantize_block(*qlib.quantize_block(x, square=True))),
        (inv, lambda: qlib.dequantize_block(q, s, torch.bfloat16, out=c)),
        (uns, lambda: qlib.dequantize_block(q, s, torch.int8)),
        (inv, lambda: qlib.fp8_block_mm_e8m0(q, qt, s, st, c)),
        (inv, lambda: qlib.fp8_block_mm_e8m0(q, q, s, s, c[:39])),
        (inv, lambda: qlib.fp8_block_mm_e8m0(q, q, s, s.view(torch.uint8), c)),
        (inv, lambda: qlib.fp8_block_mm_e8m0(q, q, s, s[:, ::2], c)),
        (inv, lambda: qlib.fp8_block_mm_e8m0(q, q, s, s.cpu(), c)),
        (inv, lambda: qlib.fp8_block_mm_e8m0(q, q, s, s, c[:1].expand(40, 40))),
        (uns, lambda: qlib.fp8_block_mm_e8m0(q, q, s, s, c.bfloat16(), accumulate=True)),
        (uns, lambda: qlib.fp8_block_mm_e8m0(q, q, s, s, c.to(torch.int32))),
        (ali, lambda: qlib.fp8_block_mm_e8m0(odd[:, 8:264], q, s, s, c)),
        (ali, lambda: qlib.fp8_block_mm_e8m0(odd.view(torch.uint8).flatten()[:40 * 264].view(E4M3).view(40, 264)[:, :256], q, s, s, c)),
    ]
    for status, call in calls:
        with pytest.raises(qlib.QgemmError) as e:
            call()
        assert e.value.status == status
    assert bool((c == 0).all())
