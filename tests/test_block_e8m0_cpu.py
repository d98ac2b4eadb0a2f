"""Refusals of the power-of-two block-scaled operators, without a GPU: the C entries check their arguments before they touch
the device, the Python forms before they call them. No compute is launched."""
import pytest
import torch

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def test_quantize_block_arguments(qlib):
    f = qlib.lib().qgemm_quantize_block
    good = (qlib.BF16, 256, 64, 8, 64, 1, 256, 64, 256, 256, 16, 256, None)

    def call(**kw):
        names = ("in_dtype", "x", "ld_in", "rows", "cols", "block_rows", "q", "ld_q", "scale", "qt", "ld_qt", "scale_t", "stream")
        return f(*(kw.get(n, v) for n, v in zip(names, good)))

    assert call(in_dtype=qlib.FP8_E4M3) == qlib.ERR_UNSUPPORTED
    assert call(in_dtype=qlib.INT8) == qlib.ERR_UNSUPPORTED
    for bad in ({"block_rows": 2}, {"block_rows": 0}, {"x": None}, {"q": None}, {"scale": None}, {"qt": None}, {"scale_t": None},
                {"q": None, "scale": None, "qt": None, "scale_t": None}, {"ld_in": 63}, {"ld_q": 63}, {"ld_qt": 7},
                {"rows": 1 << 24, "ld_qt": 1 << 24}, {"cols": 1 << 24, "ld_in": 1 << 24, "ld_q": 1 << 24}):
        assert call(**bad) == qlib.ERR_INVALID_ARG, bad
    assert call(x=257) == qlib.ERR_ALIGNMENT
    assert call(rows=0) == qlib.OK and call(cols=0) == qlib.OK


def test_checkpoint_arguments(qlib):
    f = qlib.lib().qgemm_requantize_block
    assert f(256, 64, 256, 8, 64, 256, 16, 256, None) in (qlib.OK, qlib.ERR_CUDA, qlib.ERR_UNSUPPORTED) \
        if not torch.cuda.is_available() else True
    for bad in ((None, 64, 256, 8, 64, 256, 16, 256), (256, 64, None, 8, 64, 256, 16, 256), (256, 63, 256, 8, 64, 256, 16, 256),
                (256, 64, 256, 8, 64, None, 16, 256), (256, 64, 256, 8, 64, 256, 7, 256), (256, 64, 256, 8, 64, 256, 16, None)):
        assert f(*bad, None) == qlib.ERR_INVALID_ARG, bad
    assert f(None, 0, None, 0, 64, None, 0, None, None) == qlib.OK
    f = qlib.lib().qgemm_dequantize_block
    assert f(qlib.INT8, 256, 64, 256, 1, 8, 64, 256, 64, None) == qlib.ERR_UNSUPPORTED
    for bad in ((None, 64, 256, 1, 8, 64, 256, 64), (256, 64, None, 1, 8, 64, 256, 64), (256, 64, 256, 3, 8, 64, 256, 64),
                (256, 63, 256, 1, 8, 64, 256, 64), (256, 64, 256, 1, 8, 64, None, 64), (256, 64, 256, 1, 8, 64, 256, 63)):
        assert f(qlib.BF16, *bad, None) == qlib.ERR_INVALID_ARG, bad
    assert f(qlib.FP32, 256, 64, 256, 1, 8, 64, 258, 64, None) == qlib.ERR_ALIGNMENT
    assert f(qlib.FP32, None, 0, None, 1, 0, 0, None, 0, None) == qlib.OK


def test_product_arguments(qlib):
    f = qlib.lib().qgemm_fp8_block_e8m0_gemm
    names = ("out", "a", "lda", "sa", "a_rows", "b", "ldb", "sb", "b_rows", "acc", "c", "ldc", "M", "N", "K", "stream")
    good = (qlib.BF16, 256, 128, 256, 1, 256, 128, 256, 128, 0, 256, 64, 32, 64, 128, None)

    def call(**kw):
        return f(*(kw.get(n, v) for n, v in zip(names, good)))

    for out in (qlib.INT8, qlib.INT32, qlib.FP8_E4M3, 77):
        assert call(out=out) == qlib.ERR_UNSUPPORTED
    assert call(acc=1) == qlib.ERR_UNSUPPORTED  # into bf16
    for bad in ({"a": None}, {"b": None}, {"sa": None}, {"sb": None}, {"c": None}, {"a_rows": 64}, {"b_rows": 0}, {"lda": 112},
                {"ldb": 112}, {"ldc": 63}, {"M": 1 << 31}, {"N": 1 << 31, "ldc": 1 << 31}, {"K": 1 << 31, "lda": 1 << 31, "ldb": 1 << 31}):
        assert call(**bad) == qlib.ERR_INVALID_ARG, bad
    for bad in ({"a": 264}, {"b": 264}, {"lda": 136}, {"ldb": 136}, {"c": 257}, {"out": qlib.FP32, "c": 258}):
        assert call(**bad) == qlib.ERR_ALIGNMENT, bad
    assert call(M=0) == qlib.OK and call(N=0) == qlib.OK
    assert call(out=qlib.FP32, K=0, acc=1) == qlib.OK


def test_python_forms_refuse_cpu_tensors(qlib):
    from qgemm_b200.linear import fp8_linear, pack_weight
    x = torch.ones(4, 128)
    q, s = x.to(E4M3), torch.ones(1, 4).to(E8M0)
    for call in (lambda: qlib.quantize_block(x), lambda: qlib.requantize_block(q, s), lambda: qlib.dequantize_block(q, s),
                 lambda: qlib.fp8_block_mm_e8m0(q, q, s, s, torch.zeros(4, 4)), lambda: fp8_linear(x, x), lambda: pack_weight(x),
                 lambda: fp8_linear(x.requires_grad_(True), x)):
        with pytest.raises(qlib.QgemmError) as e:
            call()
        assert e.value.status == qlib.ERR_INVALID_ARG
