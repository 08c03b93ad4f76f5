"""QuantGemm against its definition in 64 bits.

Tolerances.  INT8 sums are exact; the result takes the sum to FP32 (2^-24), two FP32 products (2^-24 each) and the rounding to the
output's type (half an ulp: 2^-8 BF16, of eight bits, 2^-11 FP16, nothing more FP32).  E4M3 products are exact in FP32, and K of them are added there with an
error of at most an ulp, 2^-23, of the sum of magnitudes each, in whatever order."""
import numpy as np
import pytest
import torch

from qwen38_flash_ops_b200 import QfgError, QuantGemm, _lib

pytestmark = pytest.mark.gpu
_HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 0.0}
_EIGHT = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def _values(gen, dtype, *shape):
    if dtype == "int8":
        return torch.randint(-128, 128, shape, generator=gen, device="cuda", dtype=torch.int16).to(torch.int8)
    return (torch.randn(*shape, generator=gen, device="cuda") * 3).to(torch.float8_e4m3fn)


def _inputs(dtype, m, k, n, order, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + m * 31 + k * 7 + n)
    x, w = _values(gen, dtype, m, k), _values(gen, dtype, n, k)
    xs = torch.rand(m, generator=gen, device="cuda") * 1e-2 + 1e-3
    ws = torch.rand(n, generator=gen, device="cuda") * 1e-2 + 1e-3
    return x, xs, (w.t() if order == "k" else w.t().contiguous()), ws


def _check(y, x, xs, w, ws, label=""):
    xd, wd = x.double(), w.double()
    scale = xs.double()[:, None] * (ws.double() if ws is not None else 1.0)
    want = (xd @ wd) * scale
    tol = want.abs() * (_HALF_ULP[y.dtype] * 1.001 + 4 * 2.0 ** -24) + (2.0 ** -25 if y.dtype == torch.float16 else 0.0)
    if x.dtype != torch.int8:
        tol += x.shape[1] * 2.0 ** -23 * (xd.abs() @ wd.abs()) * scale
    off = (y.double() - want).abs() - tol
    assert torch.isfinite(y).all() and (off <= 0).all(), f"{label}: {int((off > 0).sum())} of {off.numel()} outside, by {off.max().item():.3g}"


SIZES = [(1, 1, 1), (1, 16, 16), (3, 31, 5), (1, 128, 128), (8, 640, 256), (16, 129, 127), (17, 256, 384), (33, 1000, 40), (64, 2048, 512), (65, 77, 259),
         (130, 515, 130), (200, 1024, 1024), (257, 384, 640), (300, 272, 528), (513, 131, 257)]


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
@pytest.mark.parametrize("order", ["n", "k"])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_sizes(cuda, dtype, order, m, k, n):
    x, xs, w, ws = _inputs(dtype, m, k, n, order)
    _check(QuantGemm(w_scale=ws.cpu().numpy())(x, xs, w), x, xs, w, ws)


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
@pytest.mark.parametrize("order", ["n", "k"])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("plan", ["16,1,0,2", "48,1,0,1", "256,1,0,1", "16,4,0,2", "32,2,0,1", "128,3,0,2", "256,8,0,1", "64,1,1,1", "256,1,1,1", "224,1,1,1"])
@pytest.mark.parametrize("m,k,n", [(70, 1100, 400), (37, 1104, 403), (515, 1152, 592)])
def test_every_launch_shape(cuda, dtype, order, out_dtype, plan, m, k, n):
    """Persistent walks, K split over clusters, pairs; rows on 16 bytes and off them; full and ragged tiles."""
    x, xs, w, ws = _inputs(dtype, m, k, n, order)
    op = QuantGemm(w_scale=ws.cpu().numpy(), out_dtype=out_dtype)
    op.set_option("plan", plan)
    on16 = k % 16 == 0 and (order == "k" or n % 16 == 0)
    if plan.split(",")[2] == "1" and not on16:
        with pytest.raises(QfgError, match="bad launch shape"):
            op(x, xs, w)
        return
    _check(op(x, xs, w), x, xs, w, ws, plan)


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
@pytest.mark.parametrize("plan", ["64,1,0,1", "64,1,0,2", "96,1,1,1"])
def test_more_tiles_than_the_gpu_holds(cuda, dtype, plan):
    x, xs, w, ws = _inputs(dtype, 700, 256, 148 * 128 + 48, "n")
    op = QuantGemm(w_scale=ws.cpu().numpy())
    op.set_option("plan", plan)
    _check(op(x, xs, w), x, xs, w, ws)


@pytest.mark.parametrize("order", ["n", "k"])
@pytest.mark.parametrize("offset", [1, 2, 4, 8, 16])
def test_rows_that_begin_anywhere(cuda, order, offset):
    """Views into larger buffers: bases and row distances off 16 bytes for x, for the weight, for both.  What lies beside the rows is
    not read as part of them: it is NaN."""
    m, k, n = 21, 272, 144
    for bx, bw, ldx, ldw in [(offset, 0, 272, 288), (0, offset, 288, 288), (offset, offset, 288, 304), (0, 0, 272 + offset, 304), (0, 0, 272, 304 + offset)]:
        x0, xs, w0, ws = _inputs("e4m3", m, k, n, order, seed=offset)
        rows = n if order == "k" else k
        xbuf = torch.full((m * ldx + 64,), 0x7F, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        wbuf = torch.full((rows * ldw + 64,), 0x7F, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        x = torch.as_strided(xbuf, (m, k), (ldx, 1), bx)
        w = torch.as_strided(wbuf, (k, n), (1, ldw) if order == "k" else (ldw, 1), bw)
        x.copy_(x0)
        w.copy_(w0)
        _check(QuantGemm(w_scale=ws.cpu().numpy())(x, xs, w), x0, xs, w0, ws, f"{bx} {bw} {ldx} {ldw}")


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,ldo,base", [(5, 100, 103, 1), (5, 128, 160, 0), (300, 264, 272, 8), (300, 257, 300, 3)])
def test_outputs_given(cuda, out_dtype, m, n, ldo, base):
    x, xs, w, ws = _inputs("int8", m, 320, n, "k")
    buf = torch.full((m * ldo + 16,), 7.0, dtype=out_dtype, device="cuda")
    out = torch.as_strided(buf, (m, n), (ldo, 1), base)
    op = QuantGemm(w_scale=ws.cpu().numpy(), out_dtype=out_dtype)
    assert op(x, xs, w, out=out) is out
    _check(out, x, xs, w, ws)
    mask = torch.ones_like(buf, dtype=torch.bool)
    torch.as_strided(mask, (m, n), (ldo, 1), base).fill_(False)
    assert (buf[mask] == 7.0).all()


def test_shapes_and_the_smallest(cuda):
    x, xs, w, ws = _inputs("int8", 6, 64, 48, "n")
    op = QuantGemm(w_scale=ws.cpu().numpy())
    flat = op(x, xs, w)
    assert torch.equal(op(x.view(2, 3, 64), xs.view(2, 3), w), flat.view(2, 3, 48))
    assert torch.equal(op(x[0], xs[0], w), flat[0])
    assert op(x[:0], xs[:0], w).shape == (0, 48)
    _check(QuantGemm()(x, xs, w), x, xs, w, None)


@pytest.mark.parametrize("split", [1, 8])
def test_the_longest_integer_sums(cuda, split):
    """131071 products of -128 by -128, 2147467264, and of both signs."""
    k, n = 131071, 40
    x = torch.full((2, k), -128, dtype=torch.int8, device="cuda")
    x[1] = 127
    w = torch.full((k, n), -128, dtype=torch.int8, device="cuda")
    op = QuantGemm(out_dtype=torch.float32)
    op.set_option("plan", f"16,{split},0,1")
    y = op(x, torch.ones(2, device="cuda"), w)
    assert (y[0] == np.float32(131071 * 16384)).all() and (y[1] == np.float32(-131071 * 127 * 128)).all()


def test_sums_do_not_depend_on_the_launch_shape(cuda):
    x, xs, w, ws = _inputs("int8", 40, 2000, 512, "k")
    op = QuantGemm(w_scale=ws.cpu().numpy())
    first = op(x, xs, w)
    for plan in ("48,5,0,2", "64,1,1,1", "16,1,0,1"):
        op.set_option("plan", plan)
        assert torch.equal(op(x, xs, w), first)


@pytest.mark.parametrize("plan", ["", "16,4,0,2", "64,1,1,1"])
def test_e4m3_nan_stays_in_its_row_and_column(cuda, plan):
    x, xs, w, ws = _inputs("e4m3", 9, 640, 272, "n")
    w = w.contiguous()
    x.view(torch.uint8)[4, 100] = 0x7F
    w.view(torch.uint8)[333, 200] = 0xFF
    op = QuantGemm(w_scale=ws.cpu().numpy())
    op.set_option("plan", plan)
    bad = torch.isnan(op(x, xs, w))
    want = torch.zeros_like(bad)
    want[4], want[:, 200] = True, True
    assert torch.equal(bad, want)


def test_scales_pass_through(cuda):
    """A row with scale NaN (as RmsNormQuant marks one) is NaN, one with scale 0 is 0."""
    x, xs, w, ws = _inputs("int8", 4, 96, 64, "n")
    xs[1], xs[2] = float("nan"), 0.0
    y = QuantGemm(w_scale=ws.cpu().numpy())(x, xs, w)
    assert torch.isnan(y[1]).all() and (y[2] == 0).all() and torch.isfinite(y[[0, 3]]).all()


def test_side_stream_and_graph(cuda):
    x, xs, w, ws = _inputs("int8", 12, 512, 384, "k")
    op = QuantGemm(w_scale=ws.cpu().numpy())
    want = op(x, xs, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = op(x, xs, w)
    side.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = op(x, xs, w)
    x.copy_(torch.flip(x, [0]))
    xs.copy_(torch.flip(xs, [0]))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, torch.flip(want, [0]))


@pytest.mark.parametrize("plan", ["16,1,0,2", "16,4,0,2", "64,1,1,1"])
@pytest.mark.parametrize("k", [1024, 1021])
def test_waits_that_run_out(cuda, plan, k):
    """No operand comes: the call ends, its outputs are NaN, and the next call is whole."""
    if k % 16 and plan.endswith("1,1"):
        pytest.skip("pairs take rows on 16 bytes")
    x, xs, w, ws = _inputs("int8", 20, k, 300, "k")
    op = QuantGemm(w_scale=ws.cpu().numpy())
    op.set_option("plan", plan)
    op.set_option("give_up", 1)
    assert torch.isnan(op(x, xs, w)).all()
    op.set_option("give_up", 0)
    _check(op(x, xs, w), x, xs, w, ws)


def test_refusals(cuda):
    x, xs, w, ws = _inputs("int8", 4, 64, 48, "n")
    op = QuantGemm(w_scale=ws.cpu().numpy())
    e4m3 = torch.zeros(4, 64, device="cuda").to(torch.float8_e4m3fn)
    for args, match in [((x.float(), xs, w), "int8"), ((e4m3, xs, w), "type of x"), ((x, xs[:3], w), "one value per row"), ((x, xs.double(), w), "float32"),
                        ((x.cpu(), xs, w), "CUDA"), ((x, xs, w.cpu()), "CUDA"), ((x, xs, w[:63]), "64 rows"), ((x, xs, w[None]), "matrix"),
                        ((x, xs, torch.as_strided(w, (64, 24), (48, 2))), "contiguous"), ((x, xs, torch.as_strided(w, (64, 48), (16, 1))), "overlap"),
                        ((x.t(), xs, w), "rows"), ((x, xs, w[:, :40]), "one value per column"), ((x[:, :0], xs, w[:0]), "no elements")]:
        with pytest.raises(QfgError, match=match) as e:
            op(*args)
        assert e.value.code == _lib.QFG_INVALID_ARGUMENT
    for out in (torch.empty(4, 48, device="cuda"), torch.empty(4, 47, dtype=torch.bfloat16, device="cuda"), torch.empty(4, 48, dtype=torch.bfloat16)):
        with pytest.raises(QfgError, match="out must be"):
            op(x, xs, w, out=out)
    with pytest.raises(QfgError, match="131071"):
        QuantGemm()(torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), xs[:1], torch.zeros(131072, 16, dtype=torch.int8, device="cuda"))
    with pytest.raises(QfgError, match="out_dtype"):
        QuantGemm(out_dtype=torch.int8)
    with pytest.raises(QfgError, match="unknown option"):
        op.set_option("plans", "")
    for plan in ("15,1,0,1", "272,1,0,1", "16,9,0,1", "16,1,1,1", "64,2,1,1", "16,1,0,3"):
        op.set_option("plan", plan)
        with pytest.raises(QfgError, match="bad launch shape"):
            op(x, xs, w)
    op.set_option("plan", "")
    _check(op(x, xs, w), x, xs, w, ws)
