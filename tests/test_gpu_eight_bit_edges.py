"""RmsNormQuant and RowQuant where FP32 ends and where values lie half way.

Every case goes through each form of the kernels: rows held in registers, rows read twice (longer than 18432 values), rows through the
ring (many rows on 16 bytes); in pieces of 16 bytes, and element by element (odd lengths)."""
import numpy as np
import pytest
import torch
from test_gpu_row_quant import _SWISH, _check_rows, _norm

from qwen38_flash_ops_b200 import RmsNormQuant, RowQuant, _lib

pytestmark = pytest.mark.gpu
_TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
_EIGHT = [torch.int8, torch.float8_e4m3fn]
_TINY = 2.0 ** -100
_REL = 48 * 2.0 ** -24  # of a norm's values: as in test_gpu_row_quant.py
FORMS = [(6, 512), (6, 31), (2, 40000), (2, 40001), (400, 512), (400, 5120), (700, 129)]


def _rows(gen, rows, n):
    return torch.randn(rows, n, generator=gen, device="cuda") * torch.exp(torch.randn(n, generator=gen, device="cuda") * 0.5)


def _half_step(v, dtype):
    if dtype == torch.int8:
        return torch.full_like(v, 0.5)
    return torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 4)


# ---- small eps, small values, small weights


@pytest.mark.parametrize("q_dtype", _EIGHT)
@pytest.mark.parametrize("rows,n", FORMS)
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("eps", [0.0, 1e-14, 1e-13, 1e-12])
@pytest.mark.parametrize("weights", ["ordinary", "zero", "1e-25", "1e-30", "1e-36"])
def test_norms_of_little(cuda, q_dtype, rows, n, add, eps, weights):
    """Rows of zeros, of 1e-6 and of 1e-15 among ordinary ones, by ordinary, absent and tiny weights.

    Against the formula in 64 bits.  FP32 holds h_i w_i to 2^-150 where it is below 2^-126; the norm's factor takes that along, and the quotient by
    the scale."""
    gen = torch.Generator(device="cuda").manual_seed(n + 11)
    size = torch.tensor([1.0, 0.0, 1e-6, 1e-15], device="cuda")[torch.arange(rows, device="cuda") % 4][:, None]
    x = _rows(gen, rows, n) * size
    r = _rows(gen, rows, n) * size if add else None
    weight = (1 + 0.3 * torch.randn(n, generator=gen, device="cuda")) * (1.0 if weights == "ordinary" else 0.0 if weights == "zero" else float(weights))
    got = RmsNormQuant(eps=eps, dtype=q_dtype)(x, weight, r)
    q, scale = got[0].double(), got[1].double()
    h = (x if r is None else x + r).double()
    eps32, top = float(np.float32(eps)), _TOP[q_dtype]
    square = (h * h).mean(-1) + eps32
    none = square == 0  # zeros without eps have no norm
    assert none.any().item() == (eps == 0.0)
    root = torch.where(none, 1.0, square.rsqrt())
    y = h * weight.double() * root[:, None]
    s = y.abs().amax(-1).clamp(min=_TINY) / top
    lost = 2.0 ** -150 * root
    assert torch.equal(torch.isnan(scale), none) and (q[none] == 0).all()
    ok = ~none
    assert torch.isfinite(q).all()
    assert ((scale - s).abs() <= _REL * s + lost / top)[ok].all()
    v = y / s[:, None]
    off = (q - v).abs() - _half_step(v, q_dtype) * (1 + 1e-9) - 2 * _REL * v.abs() - 2 * (lost / s)[:, None]
    assert (off <= 0)[ok].all(), off[ok].max().item()
    if weights == "zero":
        assert (q == 0).all()


@pytest.mark.parametrize("q_dtype", _EIGHT)
@pytest.mark.parametrize("rows,n", FORMS)
def test_norms_past_fp32(cuda, q_dtype, rows, n):
    """A largest value that the norm's factor takes past FP32: the row is marked, and holds zeros."""
    x = torch.zeros(rows, n, device="cuda")
    x[:, n // 2] = 1.0  # one value, sqrt(n) behind the norm
    x[1] = 1.0
    weight = torch.full((n,), 3e38, device="cuda")
    q, scale = RmsNormQuant(eps=0.0, dtype=q_dtype)(x, weight)
    past = torch.ones(rows, dtype=torch.bool, device="cuda")
    past[1] = False
    assert torch.equal(torch.isnan(scale), past) and (q.float()[past] == 0).all()
    assert abs(scale[1].item() * _TOP[q_dtype] / 3e38 - 1) < _REL and (q[1].float() == _TOP[q_dtype]).all()


# ---- half-way values


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,n", FORMS)
def test_gated_ties_go_to_even(cuda, dtype, rows, n):
    """swish(96) is 96 in FP32, so the products are exact, the scale is 96 and the quotients are u: 127, and halves on either side."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    whole = torch.randint(-63, 63, (rows, n), generator=gen, device="cuda").float()
    u = whole + 0.5
    u[:, 0] = 127.0
    x = torch.full((rows, n), 96.0, device="cuda")
    q, scale = RowQuant(dtype=torch.int8)(x.to(dtype), u.to(dtype))
    assert (scale == 96.0).all()
    assert torch.equal(q.float(), torch.round(u))  # torch rounds halves to even


# ---- scales


@pytest.mark.parametrize("q_dtype", _EIGHT)
@pytest.mark.parametrize("rows,n", FORMS)
def test_scales_are_quotients(cuda, q_dtype, rows, n):
    """scale = largest / top, rounded once."""
    gen = torch.Generator(device="cuda").manual_seed(n + 5)
    x = _rows(gen, rows, n) * torch.rand(rows, 1, generator=gen, device="cuda")
    _, scale = RowQuant(dtype=q_dtype)(x)
    want = x.abs().amax(-1).cpu().numpy() / np.float32(_TOP[q_dtype])
    assert np.array_equal(scale.cpu().numpy(), want)


@pytest.mark.parametrize("q_dtype", _EIGHT)
@pytest.mark.parametrize("exponent", [-99, 0, 126])
def test_scales_of_every_significand(cuda, q_dtype, exponent):
    """The same over all 2^23 of them, one a row."""
    x = (torch.arange(1 << 23, device="cuda", dtype=torch.int32) | ((exponent + 127) << 23)).view(torch.float32)
    _, scale = RowQuant(dtype=q_dtype)(x[:, None])
    assert np.array_equal(scale.cpu().numpy(), x.cpu().numpy() / np.float32(_TOP[q_dtype]))


# ---- waits that run out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["rows", "gated", "norm", "added"])
@pytest.mark.parametrize("rows,n", [(400, 512), (1000, 640), (400, 5120), (3000, 2560), (300, 17408)])
def test_rows_that_never_come(cuda, dtype, kind, rows, n):
    """Every row of such a call is marked, the residual stream stays as it was, and the next call is whole."""
    if 2 * n * dtype.itemsize * (2 if kind in ("gated", "added") else 1) > 210 * 1024:
        pytest.skip("two rows do not fit the ring: they go straight into registers")
    gen = torch.Generator(device="cuda").manual_seed(n)
    x, second = _rows(gen, rows, n).to(dtype), _rows(gen, rows, n).to(dtype)
    weight, lib = torch.ones(n, device="cuda").to(dtype), _lib.load()

    def call(h):
        q, scale = torch.full((rows, n), 7, dtype=torch.int8, device="cuda"), torch.ones(rows, device="cuda")
        if kind in ("rows", "gated"):
            return RowQuant()(x, second if kind == "gated" else None, out=(q, scale))
        return RmsNormQuant()(x, weight, h if kind == "added" else None, out=(q, scale, h) if kind == "added" else (q, scale))

    want = call(second.clone())
    assert torch.isfinite(want[1]).all()
    stream = second.clone()
    assert lib.qfg_row_quant_set_option(b"give_up", b"1") == _lib.QFG_OK
    try:
        got = call(stream)
        torch.cuda.synchronize()
    finally:
        assert lib.qfg_row_quant_set_option(b"give_up", b"0") == _lib.QFG_OK
    assert torch.isnan(got[1]).all() and (got[0] == 0).all() and torch.equal(stream, second)
    again = call(stream)
    assert all(torch.equal(a, b) for a, b in zip(again, want))


def test_only_rows_of_the_ring_wait(cuda):
    x, lib = torch.ones(4, 512, device="cuda"), _lib.load()
    assert lib.qfg_row_quant_set_option(b"give_up", b"1") == _lib.QFG_OK
    try:
        q, scale = RowQuant()(x)
    finally:
        assert lib.qfg_row_quant_set_option(b"give_up", b"0") == _lib.QFG_OK
    assert (q == 127).all() and torch.isfinite(scale).all()


# ---- lengths at which another kernel takes over


@pytest.mark.parametrize("q_dtype", _EIGHT)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows", [2, 310])
@pytest.mark.parametrize("n", [504, 512, 8192, 8200, 12288, 12289, 13440, 13448, 16384, 16385, 16392, 18432, 18440, 19200, 19968, 19976, 26888])
def test_lengths_around_the_kernels_limits(cuda, q_dtype, dtype, rows, n):
    gen = torch.Generator(device="cuda").manual_seed(rows + n)
    x, second, weight = _rows(gen, rows, n).to(dtype), (3 * _rows(gen, rows, n)).to(dtype), (1 + 0.3 * torch.randn(n, generator=gen, device="cuda")).to(dtype)
    norm, act = RmsNormQuant(eps=1e-5, dtype=q_dtype), RowQuant(dtype=q_dtype)
    q, scale = norm(x, weight)
    _check_rows(q, scale, _norm(x, weight, None, 1e-5, 0.0)[0], _REL, "norm")
    q, scale, h = norm(x, weight, second)
    y, want = _norm(x, weight, second, 1e-5, 0.0)
    _check_rows(q, scale, y, _REL, "norm with residual")
    assert torch.equal(h, want)
    q, scale = act(x)
    _check_rows(q, scale, x.double(), 8 * 2.0 ** -24, "rows")
    q, scale = act(x, second)
    _check_rows(q, scale, x.double() * torch.sigmoid(x.double()) * second.double(), _SWISH + 8 * 2.0 ** -24, "gated")
