"""C cut out of a wider matrix whose rows start on 16 bytes, with columns that end inside a 16-byte unit: every kernel writes its
M x N block and nothing else. Values are small whole numbers, so every product here is exact in every type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

# tile_n, split_k, group_m, max_ctas, cta_pair, relayout_b
FORMS = {"own choice": None, "64": (64, 1, 0, 0, -1, 0), "128": (128, 1, 0, 0, -1, 0), "128 one CTA": (128, 1, 0, 1, -1, 0),
         "256": (256, 1, 0, 0, -1, 0), "pairs": (256, 1, 0, 0, 1, 0), "pairs 128": (128, 1, 0, 0, 1, 0),
         "pairs one": (256, 1, 0, 2, 1, 0), "wide pairs": (256, 1, 0, 0, 2, 0), "split": (128, 4, 0, 0, -1, 0),
         "split pairs": (128, 2, 0, 0, 1, 0)}
TYPES = [(torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
         (torch.int8, torch.int32), (torch.int8, torch.bfloat16), (torch.float8_e4m3fn, torch.bfloat16)]


def _operand(rows, cols, dtype, dev, seed):
    """Rows that start on 16 bytes; -1, 0 and 1, few enough that sums stay below 256."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-1, 2, (rows, cols), generator=g) * (torch.rand(rows, cols, generator=g) < 0.2)
    step = 16 // torch.empty(0, dtype=dtype).element_size()
    buf = torch.zeros(rows, -(-cols // step) * step, dtype=torch.float32)
    buf[:, :cols] = x
    return buf.to(dtype).to(dev)[:, :cols], x.double().to(dev)


def _cut(M, N, dtype, dev):
    wide = torch.full((M + 8, -(-N // 16) * 16 + 48), 3, dtype=dtype, device=dev)
    c = wide[4:M + 4, 16:N + 16]
    assert c.data_ptr() % 16 == 0 and c.stride(0) * c.element_size() % 16 == 0
    return wide, c


def _check(wide, c, ref):
    assert torch.equal(c.double(), ref)
    c.fill_(3)
    assert bool((wide == 3).all())


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("types", TYPES, ids=lambda t: f"{str(t[0])[6:]}-{str(t[1])[6:]}")
@pytest.mark.parametrize("M,N,K", [(300, 301, 256), (33, 519, 1040), (520, 1023, 512), (257, 300, 384)])
def test_gemm(qlib, dev, form, types, M, N, K):
    a, av = _operand(M, K, types[0], dev, 1)
    b, bv = _operand(N, K, types[0], dev, 2)
    ref = av @ bv.t()
    wide, c = _cut(M, N, types[1], dev)
    tuning = None if FORMS[form] is None else qlib.Tuning(*FORMS[form])
    if types[0] in (torch.int8, torch.float8_e4m3fn) and types[1] != torch.int32:
        one = torch.ones(1, device=dev)
        qlib.mix_gemm(a, b, one, one, c, b_kmajor=True, tuning=tuning)
    else:
        qlib.gemm(a, b, c, b_kmajor=True, tuning=tuning)
    rc, st = qlib.device_status()
    assert rc == 0, st
    _check(wide, c, ref)


@pytest.mark.parametrize("env", [{"QGEMM_KCLUSTER": "0"}, {"QGEMM_DIRECT_STORE": "1"}, {"QGEMM_EVEN_RUNS": "1"}, {"QGEMM_ONE_TILE": "0"}])
@pytest.mark.parametrize("M,N,K", [(300, 301, 4096), (2560, 2045, 1024), (1030, 4093, 2048)])
def test_gemm_by_other_ways(qlib, dev, monkeypatch, env, M, N, K):
    """Split-K with a second launch, stores from the registers, runs across tiles, and the last wave in slices."""
    a, av = _operand(M, K, torch.bfloat16, dev, 3)
    b, bv = _operand(N, K, torch.bfloat16, dev, 4)
    ref = av @ bv.t()
    for name, value in env.items():
        monkeypatch.setenv(name, value)
    qlib.lib().qgemm_reload_env()
    try:
        for tuning in (None, qlib.Tuning(256, 1, 0, 0, 1, 0), qlib.Tuning(128, 4, 0, 0, -1, 0)):
            wide, c = _cut(M, N, torch.float32, dev)
            qlib.gemm(a, b, c, b_kmajor=True, tuning=tuning)
            _check(wide, c, ref)
        rc, st = qlib.device_status()
    finally:
        monkeypatch.undo()
        qlib.lib().qgemm_reload_env()
    assert rc == 0, st


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(300, 301, 256), (33, 519, 1040), (257, 300, 384)])
def test_block_scaled(qlib, dev, out, M, N, K):
    a, av = _operand(M, K, torch.float8_e4m3fn, dev, 5)
    b, bv = _operand(N, K, torch.float8_e4m3fn, dev, 6)
    wide, c = _cut(M, N, out, dev)
    kb = -(-K // 128)
    qlib.fp8_block_mm(a, b, torch.ones(kb, M, device=dev), torch.ones(kb, -(-N // 128), device=dev), c, reference_layout=False)
    _check(wide, c, av @ bv.t())


@pytest.mark.parametrize("n_dsts", [1, 2, 3, 8])
@pytest.mark.parametrize("types", [(torch.bfloat16, torch.bfloat16), (torch.int8, torch.int32)])
@pytest.mark.parametrize("M,N,K", [(300, 301, 256), (96, 519, 1024)])
def test_several_destinations(qlib, dev, n_dsts, types, M, N, K):
    a, av = _operand(M, K, types[0], dev, 7)
    b, bv = _operand(N, K, types[0], dev, 8)
    cuts = [_cut(M, N, types[1], dev) for _ in range(n_dsts)]
    qlib.gemm_multi_dst(a, b, None, None, [c.data_ptr() for _, c in cuts], cuts[0][1].stride(0), types[1], N, b_kmajor=True)
    rc, st = qlib.device_status()
    assert rc == 0, st
    for wide, c in cuts:
        _check(wide, c, av @ bv.t())


def test_static_split(qlib, dev):
    a, av = _operand(300, 1040, torch.bfloat16, dev, 9)
    b, bv = _operand(301, 1040, torch.bfloat16, dev, 10)
    wide, c = _cut(300, 301, torch.bfloat16, dev)
    qlib.mix_gemm_splitk_static(a, b, None, None, c, 3)
    _check(wide, c, av @ bv.t())
