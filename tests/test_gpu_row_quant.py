"""RmsNormQuant, RowQuant and the MLP made of them, against their definitions in 64 bits.

Tolerances.  The sum of squares is added in at most 64 + 10 steps a path, so its relative error is below 80 * 2^-24 and the
norm's factor's below half of that; the rest of a value takes fewer than eight more FP32 operations, and exp and its quotient 2^-20.
A scale may be off by that much, and a quotient y / scale, at most 127 or 448, by twice as much before it is rounded to eight bits."""
import os
import subprocess
import sys

import pytest
import torch

from qwen38_flash_ops_b200 import QfgError, QuantGemm, QuantMlp, RmsNormQuant, RowQuant, _lib, ops

pytestmark = pytest.mark.gpu
_NORM, _SWISH = 48 * 2.0 ** -24, 2.0 ** -20
_TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
_TYPES = [torch.bfloat16, torch.float16, torch.float32]
_EIGHT = [torch.int8, torch.float8_e4m3fn]


def _half_step(v, dtype):
    """Half the distance of neighbouring eight-bit values around v."""
    if dtype == torch.int8:
        return torch.full_like(v, 0.5)
    return torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 4)


def _check_rows(q, scale, y, rel, label=""):
    top = _TOP[q.dtype]
    s = torch.clamp(y.abs().amax(dim=-1), min=2.0 ** -100) / top
    assert q.shape == y.shape and scale.shape == y.shape[:-1] and scale.dtype == torch.float32
    assert ((scale.double() - s).abs() <= rel * s).all(), f"{label}: scale off by {((scale.double() - s).abs() / s).max().item():.3g}"
    v = y / s[..., None]
    got = q.double()
    assert (got.abs() <= top).all() and ((got - v).abs() <= _half_step(v, q.dtype) * (1 + 1e-9) + 2 * rel * v.abs()).all(), label


def _norm(x, weight, residual, eps, offset):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    d = h.double()
    return d / torch.sqrt((d * d).mean(-1, keepdim=True) + eps) * (offset + weight.double()), h


def _rows(gen, rows, n, dtype, size=1.0):
    return (torch.randn(rows, n, generator=gen, device="cuda") * torch.exp(torch.randn(n, generator=gen, device="cuda") * 0.5) * size).to(dtype)


SIZES = [(1, 1), (1, 8), (3, 7), (2, 64), (1, 5120), (5, 257), (300, 128), (301, 48), (700, 129), (400, 2560), (310, 5125), (2, 17408), (3, 20481), (310, 8200),
         (2, 40000), (298, 33000)]


@pytest.mark.parametrize("q_dtype", _EIGHT)
@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("rows,n", SIZES)
def test_norm(cuda, q_dtype, dtype, add, rows, n):
    gen = torch.Generator(device="cuda").manual_seed(rows * 31 + n)
    x, r = _rows(gen, rows, n, dtype), _rows(gen, rows, n, dtype, 4.0) if add else None
    for w in {dtype, torch.float32}:
        weight = (1 + 0.3 * torch.randn(n, generator=gen, device="cuda")).to(w)
        got = RmsNormQuant(eps=1e-5, dtype=q_dtype)(x, weight, r)
        y, h = _norm(x, weight, r, 1e-5, 0.0)
        _check_rows(got[0], got[1], y, _NORM, f"{rows} x {n}")
        assert len(got) == (3 if add else 2)
        if add:
            assert torch.equal(got[2], h)


@pytest.mark.parametrize("q_dtype", _EIGHT)
@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,n", SIZES)
def test_rows(cuda, q_dtype, dtype, gated, rows, n):
    gen = torch.Generator(device="cuda").manual_seed(rows * 17 + n)
    x, u = _rows(gen, rows, n, dtype, 3.0), _rows(gen, rows, n, dtype)
    q, scale = RowQuant(dtype=q_dtype)(x, u if gated else None)
    y = x.double() * torch.sigmoid(x.double()) * u.double() if gated else x.double()
    _check_rows(q, scale, y, _SWISH + 8 * 2.0 ** -24 if gated else 8 * 2.0 ** -24, f"{rows} x {n}")


@pytest.mark.parametrize("dtype", _TYPES)
def test_swish_over_its_range(cuda, dtype):
    """A value a row, so that each is its row's largest and its scale says what it was."""
    g = torch.cat([torch.linspace(-87, 87, 4001, device="cuda"), torch.logspace(-6, 2, 200, device="cuda"), torch.tensor([0.0, 120.0, 1000.0], device="cuda")]).to(dtype)
    g = g[:, None].contiguous()
    u = torch.full_like(g, 1.0)
    _, scale = RowQuant(dtype=torch.int8)(g, u)
    want = torch.clamp((g.double() * torch.sigmoid(g.double())).abs()[:, 0], min=2.0 ** -100) / 127
    assert ((scale.double() - want).abs() <= (_SWISH + 8 * 2.0 ** -24) * want).all()


@pytest.mark.parametrize("q_dtype", _EIGHT)
def test_weight_offset_and_eps(cuda, q_dtype):
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = _rows(gen, 6, 640, torch.bfloat16, 1e-3)
    weight = (0.3 * torch.randn(640, generator=gen, device="cuda")).bfloat16()
    for eps in (0.0, 1e-6, 0.5):
        q, scale = RmsNormQuant(eps=eps, weight_offset=1.0, dtype=q_dtype)(x, weight)
        _check_rows(q, scale, _norm(x, weight, None, eps, 1.0)[0], _NORM)


def test_ties_go_to_even(cuda):
    """Quotients that lie half way: 127 and multiples of a half, with a scale of exactly one."""
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 125.5, 126.5]], device="cuda")
    q, scale = RowQuant(dtype=torch.int8)(x)
    assert scale.item() == 1.0 and q.tolist() == [[127, 0, 2, 2, 0, -2, 126, 126]]
    x = torch.tensor([[448.0, 17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10, 432.0]], device="cuda")
    q, scale = RowQuant(dtype=torch.float8_e4m3fn)(x)
    assert scale.item() == 1.0 and q.float().tolist() == [[448.0, 16.0, 20.0, 0.0, 2.0 ** -8, 448.0]]


@pytest.mark.parametrize("q_dtype", _EIGHT)
@pytest.mark.parametrize("n", [8, 31, 5120, 40000])
def test_rows_that_are_not_ordinary(cuda, q_dtype, n):
    inf, nan = float("inf"), float("nan")
    weight = torch.ones(n, device="cuda")
    for special in (inf, -inf, nan):
        x = torch.ones(4, n, device="cuda")
        x[1, n // 2] = special
        x[2] = 0.0
        for q, scale in (RmsNormQuant(dtype=q_dtype)(x, weight), RowQuant(dtype=q_dtype)(x), RowQuant(dtype=q_dtype)(x.clone().fill_(1.0), x)):
            assert torch.isnan(scale).tolist() == [False, True, False, False]
            assert (q[1].float() == 0).all() and (q[2].float() == 0).all() and (q[0].float() == _TOP[q_dtype]).all()
            assert scale[2].item() == pytest.approx(2.0 ** -100 / _TOP[q_dtype], rel=1e-6)
    # a sum of squares past FP32 is not passed off as a row of zeros; rows of tiny values have the least scale
    x = torch.full((2, n), 1e25, device="cuda")
    x[1] = 1e-35
    q, scale = RmsNormQuant(dtype=q_dtype)(x, weight)
    assert torch.isnan(scale[0]) and (q[0].float() == 0).all() and torch.isfinite(scale[1])
    q, scale = RowQuant(dtype=q_dtype)(x)
    assert scale[0].item() == pytest.approx(1e25 / _TOP[q_dtype], rel=1e-6) and (q[0].float() == _TOP[q_dtype]).all()
    assert scale[1].item() == pytest.approx(2.0 ** -100 / _TOP[q_dtype], rel=1e-6)
    _check_rows(q[1:], scale[1:], x[1:].double(), 8 * 2.0 ** -24)  # 0 in INT8, 0.0059 in E4M3


@pytest.mark.parametrize("n", [8, 31, 5120])
def test_zeros_without_eps_have_no_norm(cuda, n):
    """0 / 0 is not passed off as a row of zeros."""
    x = torch.ones(2, n, device="cuda")
    x[1] = 0.0
    q, scale = RmsNormQuant(eps=0.0)(x, torch.ones(n, device="cuda"))
    assert torch.isnan(scale).tolist() == [False, True] and (q[0] == 127).all() and (q[1] == 0).all()


@pytest.mark.parametrize("rows,n", [(3, 512), (400, 512), (400, 5120)])
def test_a_first_call_may_be_captured(cuda, rows, n):
    """In a process that has made no call yet."""
    code = f"""
import torch
from qwen38_flash_ops_b200 import QuantGemm, RmsNormQuant, RowQuant
x, w, g = torch.randn({rows}, {n}, device="cuda").bfloat16(), torch.ones({n}, device="cuda").bfloat16(), torch.ones({n}, 64, dtype=torch.int8, device="cuda")
norm, act, gemm, graph = RmsNormQuant(), RowQuant(), QuantGemm(), torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    q, s, h = norm(x, w, x)
    q2, s2 = act(h, x)
    y = gemm(q2, s2, g)
graph.replay()
torch.cuda.synchronize()
a, b, c = norm(x, w, x)
d, e = act(c, x)
assert torch.equal(a, q) and torch.equal(b, s) and torch.equal(c, h) and torch.equal(d, q2) and torch.equal(gemm(d, e, g), y)
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True, timeout=240)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("dtype", _TYPES)
@pytest.mark.parametrize("rows,n,ld,base", [(5, 96, 128, 0), (5, 96, 97, 1), (310, 64, 80, 3), (3, 5120, 10240, 5120), (1, 33, 33, 2)])
def test_rows_that_begin_anywhere(cuda, dtype, rows, n, ld, base):
    gen = torch.Generator(device="cuda").manual_seed(n)

    def view(values):
        buf = torch.full((rows * ld + base + 8,), float("nan"), dtype=dtype, device="cuda")
        t = torch.as_strided(buf, (rows, n), (ld, 1), base)
        t.copy_(values)
        return t

    x0, r0 = _rows(gen, rows, n, dtype), _rows(gen, rows, n, dtype)
    x, r, weight = view(x0), view(r0), torch.as_strided(torch.ones(n + 1, dtype=dtype, device="cuda"), (n,), (1,), 1)
    norm, act = RmsNormQuant(), RowQuant()
    for a, b in ((norm(x, weight, r), norm(x0, weight.clone(), r0)), (act(x, r), act(x0, r0))):
        _check_rows(a[0], a[1], _norm(x0, weight, r0, 1e-6, 0.0)[0] if len(a) == 3 else x0.double() * torch.sigmoid(x0.double()) * r0.double(),
                    _NORM if len(a) == 3 else _SWISH + 8 * 2.0 ** -24)
        if len(a) == 3:
            assert torch.equal(a[2], b[2])


@pytest.mark.parametrize("rows,n", [(4, 512), (400, 640), (3, 700), (2, 40000)])
def test_in_place(cuda, rows, n):
    """The residual stream may be updated where it lies."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    x, r, weight = _rows(gen, rows, n, torch.bfloat16), _rows(gen, rows, n, torch.bfloat16), torch.ones(n, device="cuda").bfloat16()
    op = RmsNormQuant()
    want = op(x, weight, r)
    for into in ("residual", "x"):
        a, b = x.clone(), r.clone()
        h = b if into == "residual" else a
        q, scale = torch.empty_like(want[0]), torch.empty_like(want[1])
        got = op(a, weight, b, out=(q, scale, h))
        assert got[2] is h and all(torch.equal(g, w) for g, w in zip(got, want))


def test_shapes(cuda):
    gen = torch.Generator(device="cuda").manual_seed(6)
    x, weight = _rows(gen, 6, 64, torch.bfloat16), torch.ones(64, device="cuda")
    for op in (lambda t: RmsNormQuant()(t, weight), RowQuant()):
        q, scale = op(x)
        a, b = op(x.view(2, 3, 64))
        assert torch.equal(a.view(6, 64), q) and torch.equal(b.view(6), scale)
        a, b = op(x[2])
        assert a.shape == (64,) and b.shape == () and torch.equal(a, q[2]) and b == scale[2]
        a, b = op(x[:0])
        assert a.shape == (0, 64) and b.shape == (0,)


def test_side_stream_and_graph(cuda):
    gen = torch.Generator(device="cuda").manual_seed(7)
    x, r, weight = _rows(gen, 9, 512, torch.bfloat16), _rows(gen, 9, 512, torch.bfloat16), torch.ones(512, device="cuda").bfloat16()
    ops = lambda: [*RmsNormQuant()(x, weight, r), *RowQuant()(x, r)]
    want = ops()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops()
    x.copy_(torch.flip(x, [0]))
    r.copy_(torch.flip(r, [0]))
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, torch.flip(b.float(), [0]).to(b.dtype)) for a, b in zip(out, want))


def test_refusals(cuda):
    x, weight = torch.ones(4, 64, device="cuda").bfloat16(), torch.ones(64, device="cuda").bfloat16()
    norm, act = RmsNormQuant(), RowQuant()
    for call, match in [(lambda: norm(x.to(torch.int32), weight), "bfloat16"), (lambda: norm(x.cpu(), weight), "CUDA"), (lambda: norm(x, weight.half()), "weight must be"),
                        (lambda: norm(x, weight[:63]), "64 elements"), (lambda: norm(x, weight.cpu()), "CUDA"), (lambda: norm(x, weight, x[:3]), "shape of x"),
                        (lambda: norm(x, weight, x.float()), "residual must be"), (lambda: norm(x.t(), weight[:4]), "contiguous"),
                        (lambda: norm(x[:1].expand(4, 64), weight), "overlap"), (lambda: act(x, x[:, :32]), "shape of x"), (lambda: act(x, x.float()), "u must be"),
                        (lambda: act(x[:, :0]), "no elements"), (lambda: act(torch.tensor(1.0, device="cuda")), "no elements"),
                        (lambda: act(x, out=(torch.empty(4, 64, device="cuda"), torch.empty(4, device="cuda"))), "q must be"),
                        (lambda: norm(x, weight, x, out=(torch.empty(4, 64, dtype=torch.int8, device="cuda"), torch.empty(4, device="cuda"))), "out must be"),
                        (lambda: RowQuant(dtype=torch.uint8), "dtype"), (lambda: RmsNormQuant(dtype=torch.float16), "dtype"), (lambda: RmsNormQuant(eps=-1.0), "eps"),
                        (lambda: RmsNormQuant(eps=float("nan")), "eps")]:
        with pytest.raises(QfgError, match=match) as e:
            call()
        assert e.value.code == _lib.QFG_INVALID_ARGUMENT


@pytest.mark.parametrize("dtype", _EIGHT)
@pytest.mark.parametrize("order", ["n", "k"])
@pytest.mark.parametrize("rows,hidden,width", [(1, 256, 512), (7, 640, 264), (300, 512, 384), (5, 129, 77)])
def test_mlp(cuda, monkeypatch, dtype, order, rows, hidden, width):
    """The block against its definition, of which each eight-bit rounding moves a value by up to half a step: the products' relative
    errors add up to a few times 2^-8 (INT8) or 2^-4 (E4M3) of a row's typical value, as the sums of independent ones."""
    gen = torch.Generator(device="cuda").manual_seed(rows + hidden)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")

    def quantised(k, n):
        w = rand(n, k) * 0.05
        s = w.abs().amax(1) / _TOP[dtype]
        q = w / s[:, None]
        q = (q.round() if dtype == torch.int8 else q).to(dtype)
        return (q.t() if order == "k" else q.t().contiguous()), s

    (q1, s1), (q2, s2) = quantised(hidden, 2 * width), quantised(width, hidden)
    g = (1 + 0.2 * rand(hidden)).bfloat16()
    x, r = rand(rows, hidden).bfloat16(), rand(rows, hidden).bfloat16()
    mlp = QuantMlp(g, q1, s1.cpu().numpy(), q2, s2.cpu().numpy())
    y, h = mlp(x, r)
    normed, hw = _norm(x, g, r, 1e-6, 0.0)
    assert torch.equal(h, hw) and y.shape == x.shape and y.dtype == torch.bfloat16
    both = normed @ (q1.double() * s1.double())
    a, b = both[:, :width], both[:, width:]
    want = (a * torch.sigmoid(a) * b) @ (q2.double() * s2.double())
    bound = 0.03 if dtype == torch.int8 else 0.12
    assert ((y.double() - want).norm() / want.norm()).item() < bound
    with monkeypatch.context() as m:  # the same four calls from Python
        m.setattr(ops._calls, "quant_mlp", lambda *args: None)
        assert all(torch.equal(a, b) for a, b in zip(mlp(x, r), (y, h)))
    padded = torch.zeros(rows, hidden + 24, device="cuda").bfloat16()[:, :hidden].copy_(x)
    assert torch.equal(mlp(padded, r)[0], y) and torch.equal(mlp(x[:1], r[:1])[1], h[:1])
    if rows > 1:
        assert torch.equal(mlp(x.view(rows, 1, hidden), r.view(rows, 1, hidden))[0].view(rows, hidden), y)


def test_mlp_refusals(cuda):
    w1, w2, s = torch.zeros(64, 96, dtype=torch.int8, device="cuda"), torch.zeros(48, 64, dtype=torch.int8, device="cuda"), torch.ones(96)
    g, x = torch.ones(64, device="cuda").bfloat16(), torch.ones(3, 64, device="cuda").bfloat16()
    mlp = QuantMlp(g, w1, s.numpy(), w2, s[:64].numpy())
    for bad in ((x[:, :32], x[:, :32]), (x, x[:2]), (x.cpu(), x), (x, x.float()), (x.half(), x.half())):
        with pytest.raises(QfgError):
            mlp(*bad)
    assert mlp(x[:0], x[:0])[0].shape == (0, 64)
    for shapes in ((w1[:, :95], w2), (w1, w2[:, :63]), (w1, w2.float())):
        with pytest.raises(ValueError, match="QuantMlp"):
            QuantMlp(g, shapes[0], None, shapes[1], None)


@pytest.mark.parametrize("rows,hidden,width", [(1, 256, 512), (8, 2048, 4096), (40, 1024, 2048), (200, 512, 1536), (6, 520, 1001)])
def test_mlp_waits_for_what_ran_before(cuda, monkeypatch, rows, hidden, width):
    """Weights, inputs and residual written right before each call, its results read right behind it."""
    gen = torch.Generator(device="cuda").manual_seed(31)
    ints = lambda *s: torch.randint(-127, 128, s, generator=gen, device="cuda").to(torch.int8)
    w1s, w2s = [ints(hidden, 2 * width) for _ in range(3)], [ints(width, hidden) for _ in range(3)]
    xs = [torch.randn(rows, hidden, generator=gen, device="cuda").bfloat16() for _ in range(3)]
    g = torch.ones(hidden, device="cuda").bfloat16()
    w1, w2, x, r = w1s[0].clone(), w2s[0].clone(), xs[0].clone(), xs[0].clone()
    mlp = QuantMlp(g, w1, torch.full((2 * width,), 1e-3).numpy(), w2, torch.full((hidden,), 1e-3).numpy())

    def passes():
        got = []
        for i in range(24):
            w1.copy_(w1s[i % 3]), w2.copy_(w2s[i % 3]), x.copy_(xs[i % 3]), r.copy_(xs[(i + 1) % 3])
            y, h = mlp(x, r)
            again, _ = mlp(y, h)  # and one call behind another
            got += [y + 0, h + 0, again + 0]
        return got

    one = passes()
    monkeypatch.setattr(ops._calls, "quant_mlp", lambda *args: None)
    assert all(torch.equal(a, b) for a, b in zip(one, passes()))


def test_mlp_on_two_streams(cuda, monkeypatch):
    gen = torch.Generator(device="cuda").manual_seed(32)
    ints = lambda *s: torch.randint(-127, 128, s, generator=gen, device="cuda").to(torch.int8)
    s = torch.full((2048,), 1e-3).numpy()
    mlps = [QuantMlp(torch.ones(512, device="cuda").bfloat16(), ints(512, 2048), s, ints(1024, 512), s[:512]) for _ in range(2)]
    xs = [torch.randn(16, 512, generator=gen, device="cuda").bfloat16() for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(40):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(mlps[i](xs[i], xs[i])[0])
    torch.cuda.synchronize()
    monkeypatch.setattr(ops._calls, "quant_mlp", lambda *args: None)
    for i in range(2):
        want = mlps[i](xs[i], xs[i])[0]
        assert all(torch.equal(y, want) for y in got[i])


@pytest.mark.parametrize("change,message", [
    (dict(workspace=None), "null argument"), (dict(workspace="odd"), "256 bytes"), (dict(residual=None), "null argument"), (dict(y=None), "null argument"),
    (dict(rows=-1), "bad shape"), (dict(width=0), "bad shape"), (dict(hidden=0), "bad shape"), (dict(width=1 << 30), "bad shape"), (dict(ldx=63), "bad shape"),
    (dict(ldw1=255), "bad shape"), (dict(ldw2=63), "bad shape"), (dict(q_dtype=_lib.QFG_UINT8), "INT8 or FP8"), (dict(order1=2), "bad order"),
    (dict(weight=None), "null argument"), (dict(w1=None), "null argument"), (dict(w2=None), "null argument"), (dict(h=None), "null argument"),
])
def test_blocks_that_are_refused(cuda, change, message):
    lib = _lib.load()
    up, down = QuantGemm(), QuantGemm()
    rows, hidden, width = 3, 64, 128
    keep = [torch.zeros(rows, hidden, device="cuda").bfloat16() for _ in range(5)]
    w1, w2 = torch.zeros(hidden, 2 * width, dtype=torch.int8, device="cuda"), torch.zeros(width, hidden, dtype=torch.int8, device="cuda")
    bytes_ = lib.qfg_quant_mlp_workspace_bytes(up._p, rows, hidden, width)
    assert bytes_ >= rows * (hidden + width + 4 * width)
    workspace = torch.zeros(bytes_ + 16, dtype=torch.uint8, device="cuda")
    a = dict(dtype=_lib.QFG_BFLOAT16, x=keep[0].data_ptr(), ldx=hidden, residual=keep[1].data_ptr(), ldr=hidden, weight=keep[2].data_ptr(),
             weight_dtype=_lib.QFG_BFLOAT16, offset=0.0, eps=1e-6, rows=rows, hidden=hidden, width=width, q_dtype=_lib.QFG_INT8, up=up._p, w1=w1.data_ptr(),
             ldw1=2 * width, order1=0, down=down._p, w2=w2.data_ptr(), ldw2=hidden, order2=0, workspace=workspace.data_ptr(), y=keep[3].data_ptr(),
             h=keep[4].data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    assert lib.qfg_quant_mlp(*a.values()) == _lib.QFG_OK
    a.update(change)
    if a["workspace"] == "odd":
        a["workspace"] = workspace.data_ptr() + 16
    assert lib.qfg_quant_mlp(*a.values()) == _lib.QFG_INVALID_ARGUMENT and message in lib.qfg_last_error().decode()
    torch.cuda.synchronize()
