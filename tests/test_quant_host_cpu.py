"""Eight-bit blocks without a GPU: what the C ABI and the Python ops refuse before any CUDA call, the C++ calls' hand-back, packing."""
import ctypes

import numpy as np
import pytest
import torch

import qwen38_flash_ops_b200 as package
from qwen38_flash_ops_b200 import QfgError, RmsNormQuant, RowQuant, _calls, _lib
from qwen38_flash_ops_b200 import packing as P
from qwen38_flash_ops_b200 import packing_torch as PT

PTR = 1 << 20  # an address that nothing reads
BF16, F16, F32, I8, E4M3, U8 = _lib.QFG_BFLOAT16, _lib.QFG_FLOAT16, _lib.QFG_FLOAT, _lib.QFG_INT8, _lib.QFG_FLOAT8E4M3FN, _lib.QFG_UINT8


def _norm(**change):
    a = dict(dtype=BF16, x=PTR, ldx=64, residual=PTR, ldr=64, weight=PTR, weight_dtype=BF16, offset=0.0, eps=1e-6, rows=2, n=64, q_dtype=I8, q=PTR,
             scale=PTR, h=PTR, stream=None)
    a.update(change)
    lib = _lib.load()
    return lib.qfg_rmsnorm_quant(*a.values()), lib.qfg_last_error().decode()


def _rows(**change):
    a = dict(dtype=BF16, x=PTR, ldx=64, u=PTR, ldu=64, rows=2, n=64, q_dtype=E4M3, q=PTR, scale=PTR, stream=None)
    a.update(change)
    lib = _lib.load()
    return lib.qfg_row_quant(*a.values()), lib.qfg_last_error().decode()


@pytest.mark.parametrize("change,message", [
    (dict(dtype=I8), "weight must have"), (dict(dtype=U8, weight_dtype=F32), "BF16/FP16/FP32"), (dict(weight_dtype=F16), "weight must have"),
    (dict(q_dtype=BF16), "INT8 or FP8"), (dict(q_dtype=U8), "INT8 or FP8"), (dict(n=0), "bad shape"), (dict(n=1 << 31, ldx=1 << 31, ldr=1 << 31), "bad shape"),
    (dict(rows=-1), "bad shape"), (dict(ldx=63), "bad shape"), (dict(ldr=63), "bad shape"), (dict(x=None), "null"), (dict(weight=None), "null"),
    (dict(q=None), "null"), (dict(scale=None), "null"), (dict(h=None), "null"), (dict(x=PTR + 1), "misaligned"), (dict(residual=PTR + 1), "misaligned"),
    (dict(scale=PTR + 2), "misaligned"), (dict(weight=PTR + 2, weight_dtype=F32), "misaligned"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
])
def test_norms_that_are_refused(change, message):
    code, text = _norm(**change)
    assert code == _lib.QFG_INVALID_ARGUMENT and message in text and text.startswith("RmsNormQuant")


@pytest.mark.parametrize("change,message", [
    (dict(dtype=I8), "BF16/FP16/FP32"), (dict(q_dtype=F16), "INT8 or FP8"), (dict(ldu=0), "bad shape"), (dict(ldx=0), "bad shape"), (dict(x=None), "null"),
    (dict(u=PTR + 1), "misaligned"), (dict(dtype=F32, x=PTR + 2), "misaligned"),
])
def test_rows_that_are_refused(change, message):
    code, text = _rows(**change)
    assert code == _lib.QFG_INVALID_ARGUMENT and message in text and text.startswith("RowQuant")


def test_no_rows_are_no_call():
    assert _norm(rows=0, x=None, q=None)[0] == _lib.QFG_OK and _rows(rows=0, x=None, q=None)[0] == _lib.QFG_OK


def test_blocks_that_are_refused():
    lib = _lib.load()
    assert lib.qfg_quant_mlp_workspace_bytes(None, 1, 64, 64) == 0
    code = lib.qfg_quant_mlp(BF16, PTR, 64, PTR, 64, PTR, BF16, 0.0, 1e-6, 1, 64, 64, I8, None, PTR, 128, 0, None, PTR, 64, 0, PTR, PTR, PTR, None)
    assert code == _lib.QFG_INVALID_ARGUMENT and lib.qfg_last_error().decode() == "QuantMlp: null node"


def test_nodes_that_are_refused():
    lib, h = _lib.load(), ctypes.c_void_p()
    assert lib.qfg_quant_gemm_create(None, 0, I8, ctypes.byref(h)) == _lib.QFG_INVALID_ARGUMENT and not h.value
    assert lib.qfg_quant_gemm_create(None, 4, BF16, ctypes.byref(h)) == _lib.QFG_INVALID_ARGUMENT and "w_scale" in lib.qfg_last_error().decode()
    assert lib.qfg_quant_gemm_create(None, 0, BF16, None) == _lib.QFG_INVALID_ARGUMENT
    assert lib.qfg_quant_gemm_compute(None, I8, PTR, 64, PTR, 1, 64, PTR, 64, 0, 64, PTR, 64, None) == _lib.QFG_INVALID_ARGUMENT
    assert lib.qfg_quant_gemm_set_option(None, b"plan", b"") == _lib.QFG_INVALID_ARGUMENT
    lib.qfg_quant_gemm_destroy(None)
    if not torch.cuda.is_available():
        assert lib.qfg_quant_gemm_create(None, 0, BF16, ctypes.byref(h)) == _lib.QFG_FAIL and not h.value  # no device: said, not passed over


@pytest.mark.parametrize("t", [torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(2, 8, device="meta"), None, 3])
def test_other_tensors_are_handed_back_and_refused(t):
    assert _calls.row_quant(False, t, None) is None and _calls.rmsnorm_quant(1e-6, 0.0, False, t, t, None) is None
    assert _calls.quant_gemm(1, BF16, t, t, t) is None and _calls.quant_mlp(1e-6, 0.0, t, 1, t, 1, t, t, t) is None and _calls.quant_mlp() is None
    with pytest.raises(QfgError, match="CUDA"):
        RowQuant()(t)
    with pytest.raises(QfgError, match="CUDA"):
        RmsNormQuant()(t, t)


def test_odd_arguments_leave_no_error_behind():
    x = torch.zeros(2, 8, dtype=torch.bfloat16)
    for args in [(), (1, x, None), (True, x), ("", x, None)]:
        assert _calls.row_quant(*args) is None
    assert _calls.rmsnorm_quant(1, 0, True, x, x, None) is None and _calls.quant_gemm("1", "2", x, x, x) is None


def test_bind_rows_checks_its_addresses():
    with pytest.raises(TypeError):
        _calls.bind_rows(1, 2)
    with pytest.raises(ValueError):
        _calls.bind_rows(1, 0, 1)


def test_bind_mlp_checks_its_addresses():
    with pytest.raises(TypeError):
        _calls.bind_mlp(1)
    with pytest.raises(ValueError):
        _calls.bind_mlp(1, 0)


def test_lazy_names():
    assert package.QuantMlp.__name__ == "QuantMlp" and package.QuantGemm.__name__ == "QuantGemm"


def test_int8_packing():
    rng = np.random.default_rng(1)
    w = rng.standard_normal((64, 40)).astype(np.float32) * 0.02
    w[:, 7] = 0.0
    q, s = P.quantize_int8_per_column(w)
    assert q.dtype == np.int8 and s.dtype == np.float32 and q.shape == w.shape and s.shape == (40,)
    assert np.abs(q).max() == 127 and (np.abs(q.astype(np.float64) * s - w) <= 0.5 * s * (1 + 1e-6)).all() and (q[:, 7] == 0).all()
    qt, st = PT.quantize_int8_per_column_torch(torch.from_numpy(w))
    assert np.array_equal(qt.numpy(), q) and np.array_equal(st.numpy(), s)
