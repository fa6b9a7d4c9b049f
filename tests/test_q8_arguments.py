"""What the 8-bit and sampling entry points refuse, before any launch: no device is needed."""
import ctypes as C

import pytest

from axiom_amd import capi
from tests import q8_harness as q8

X = 1 << 20  # an address that nothing reads


def refused(code, call, *args):
    with pytest.raises(capi.AxhipError) as e:
        capi.check(call(*args))
    assert e.value.code == code, str(e.value)
    return str(e.value)


def test_struct_layouts_match_the_compiled_library():
    for which, cls in ((5, capi.RowsQ8Params), (6, capi.GemmQ8Params), (7, capi.SampleParams)):
        assert capi.lib().axhip_sizeof(which) == C.sizeof(cls)


@pytest.mark.parametrize("change,word", [(dict(dtype=3), "dtype"), (dict(dtype=9), "dtype"), (dict(rows=-1), "extent"), (dict(cols=-1), "extent"), (dict(cols=1 << 41), "extent"),
                                         (dict(ld_x=7), "overlap"), (dict(ld_q=7), "overlap")])
def test_rows(change, word):
    lib = capi.lib()
    p = q8.rows_params("f32", 4, 8, 8, 8)
    for name, value in change.items():
        setattr(p, name, value)
    assert word in refused(capi.ERR_INVALID_ARG, lib.axhip_quantize_q8, X, X, X, C.byref(p), None)
    assert word in refused(capi.ERR_INVALID_ARG, lib.axhip_rms_norm_q8, X, None, X, None, X, X, C.byref(p), None)


def test_rows_buffers():
    lib = capi.lib()
    refused(capi.ERR_INVALID_ARG, lib.axhip_quantize_q8, X, X, X, None, None)
    refused(capi.ERR_INVALID_ARG, lib.axhip_rms_norm_q8, X, None, X, None, X, X, None, None)
    p = q8.rows_params("bf16", 4, 8, 8, 8)
    for args in ((None, X, X), (X, None, X), (X, X, None), (X + 1, X, X), (X, X, X + 2)):
        refused(capi.ERR_INVALID_ARG, lib.axhip_quantize_q8, *args, C.byref(p), None)
    assert "residual" in refused(capi.ERR_INVALID_ARG, lib.axhip_rms_norm_q8, X, None, X, X, X, X, C.byref(p), None)
    p.ld_residual = 7
    assert "overlap" in refused(capi.ERR_INVALID_ARG, lib.axhip_rms_norm_q8, X, X, X, None, X, X, C.byref(p), None)
    p.ld_residual, p.ld_sum = 8, 7
    assert "overlap" in refused(capi.ERR_INVALID_ARG, lib.axhip_rms_norm_q8, X, X, X, 2 * X, X, X, C.byref(p), None)
    p.ld_sum, p.ld_x = 9, 10
    assert "place" in refused(capi.ERR_INVALID_ARG, lib.axhip_rms_norm_q8, X, 2 * X, X, X, X, X, C.byref(p), None)
    assert "place" in refused(capi.ERR_INVALID_ARG, lib.axhip_rms_norm_q8, X, 2 * X, X, 2 * X, X, X, C.byref(p), None)
    p = q8.rows_params("bf16", 4, 8, 8, 8)
    for eps in (-1e-5, float("nan"), float("inf")):
        p.eps = eps
        assert "eps" in refused(capi.ERR_INVALID_ARG, lib.axhip_rms_norm_q8, X, None, X, None, X, X, C.byref(p), None)


def gemm_params(**change):
    p = capi.GemmQ8Params()
    p.dtype, p.m, p.n, p.k, p.lda, p.ldb, p.ldc, p.scale_a, p.scale_b = capi.DTYPE_BF16, 4, 8, 32, 32, 32, 8, X, X
    for name, value in change.items():
        setattr(p, name, value)
    return p


@pytest.mark.parametrize("change", [dict(dtype=3), dict(dtype=-1), dict(m=-1), dict(n=-1), dict(k=-1), dict(m=1 << 30), dict(n=1 << 31), dict(lda=31), dict(ldb=31), dict(ldc=7), dict(scale_a=None),
                                    dict(scale_b=None), dict(epilogue_op=capi.OP["exp"]), dict(bias=X + 1), dict(residual=X + 1), dict(scale_a=X + 1)])
def test_products(change):
    refused(capi.ERR_INVALID_ARG, capi.lib().axhip_gemm_q8, X, X, X, C.byref(gemm_params(**change)), None)


def test_products_more():
    lib = capi.lib()
    refused(capi.ERR_INVALID_ARG, lib.axhip_gemm_q8, X, X, X, None, None)
    for args in ((None, X, X), (X, None, X), (X, X, None), (X, X, X + 1)):
        refused(capi.ERR_INVALID_ARG, lib.axhip_gemm_q8, *args, C.byref(gemm_params()), None)
    assert "131071" in refused(capi.ERR_UNSUPPORTED, lib.axhip_gemm_q8, X, X, X, C.byref(gemm_params(k=131072, lda=131072, ldb=131072)), None)
    refused(capi.ERR_UNSUPPORTED, lib.axhip_gemm_q8, X, X, X, C.byref(gemm_params(lda=1 << 41)), None)
    capi.check(lib.axhip_gemm_q8(None, None, None, C.byref(gemm_params(m=0)), None))  # nothing to do
    assert lib.axhip_gemm_q8_last_kernel() == b"empty"


def sample_params(**change):
    p = capi.SampleParams()
    p.dtype, p.rows, p.vocab, p.ld, p.u = capi.DTYPE_F32, 4, 100, 100, X
    for name, value in change.items():
        setattr(p, name, value)
    return p


@pytest.mark.parametrize("change", [dict(dtype=3), dict(rows=-1), dict(rows=1 << 22), dict(vocab=0), dict(vocab=-5), dict(ld=99), dict(ld=1 << 41), dict(u=None), dict(u=X + 1), dict(temperature=X + 2),
                                    dict(top_k=X + 1), dict(top_p=X + 1), dict(min_p=X + 1)])
def test_sampling(change):
    lib = capi.lib()
    refused(capi.ERR_INVALID_ARG, lib.axhip_sample, X, X, X, C.byref(sample_params(**change)), None)
    refused(capi.ERR_INVALID_ARG, lib.axhip_sample_ws, X, X, X, C.byref(sample_params(**change)), None, 0, None)


def test_sampling_more():
    lib = capi.lib()
    refused(capi.ERR_INVALID_ARG, lib.axhip_sample, X, X, X, None, None)
    for args in ((None, X, X), (X, None, X), (X + 2, X, X), (X, X + 4, X), (X, X, X + 2)):
        refused(capi.ERR_INVALID_ARG, lib.axhip_sample, *args, C.byref(sample_params()), None)
    refused(capi.ERR_UNSUPPORTED, lib.axhip_sample, X, X, X, C.byref(sample_params(vocab=(1 << 20) + 1, ld=1 << 21)), None)
    assert lib.axhip_sample_workspace_bytes(None) == 0
    capi.check(lib.axhip_sample(None, None, None, C.byref(sample_params(rows=0)), None))
