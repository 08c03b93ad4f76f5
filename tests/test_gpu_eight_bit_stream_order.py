"""Eight-bit calls see what the kernels before them in the stream wrote, although their blocks may be placed before those have ended: behind copies into the
same buffers, and behind a kernel that lets its dependents in at its start and writes what they read at its end."""
import pytest
import torch
from test_gpu_stream_order import _Early, _rand

from qwen38_flash_ops_b200 import QuantGemm, QuantMlp, RmsNormQuant, RowQuant, SharedExpertDown
from qwen38_flash_ops_b200 import workloads as W

pytestmark = pytest.mark.gpu
ROWS = 400  # of the buffer, [ROWS, 2560] BF16: many enough for the ring of the row kernels; the predecessor writes rows 32 to 39


def _bits(t):
    return t.contiguous().view(torch.uint8)


def _ints(seed, *shape):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-127, 128, shape, generator=gen, device="cuda").to(torch.int8)


def _row_call(kind, reads, form):
    """buffer -> outputs.  form: rows in registers, through the ring, element by element."""
    part = {"few": lambda b: b[32:40], "ring": lambda b: b, "odd": lambda b: b[32:40, 1:]}[form]
    n = 2560 - (form == "odd")
    rows = ROWS if form == "ring" else 8
    other, weight = _rand(31, rows, n), _rand(32, n)
    if kind == "act":
        op = RowQuant()
        return {"x": lambda b: op(part(b), other), "u": lambda b: op(other, part(b))}[reads]
    op = RmsNormQuant(dtype=torch.float8_e4m3fn)
    return {"x": lambda b: op(part(b), weight, other), "residual": lambda b: op(other, weight, part(b)), "weight": lambda b: op(other, b[39, 2560 - n:]),
            "alone": lambda b: op(part(b), weight)}[reads]


def _gemm_call(reads, plan, odd):
    """Bytes of rows 32 to 39 as x [8 or 64, K], as the weight [K, 256], or as the rows' scales."""
    op = QuantGemm(out_dtype=torch.float32)
    op.set_option("plan", plan)
    raw = lambda b: b[32:40].view(torch.int8).reshape(-1)
    if reads == "x":
        w = _ints(33, 640 - odd, 384)
        return lambda b: [op(raw(b).reshape(64, 640)[:, odd:], torch.ones(64, device="cuda"), w)]
    if reads == "weight":
        x = _ints(34, 40, 160)
        return lambda b: [op(x, torch.ones(40, device="cuda"), raw(b).reshape(160, 256)[:, odd:])]
    x, w = _ints(35, 40, 640 - odd), _ints(36, 640 - odd, 384)
    return lambda b: [op(x, b[32].view(torch.float32)[:40], w)]


def _mlp_call(reads):
    rows, hidden, width = 8, 2560, 1024
    mlp = QuantMlp(_rand(37, hidden), _ints(38, hidden, 2 * width), torch.full((2 * width,), 1e-4).numpy(), _ints(39, width, hidden), torch.full((hidden,), 1e-3).numpy())
    other = _rand(40, rows, hidden)
    if reads == "weight":  # the down projection of a narrower block: [160, 256] int8
        small = lambda b: b[32:40].view(torch.int8).reshape(160, 256)
        g, w1, s1, s2, x = _rand(41, 256), _ints(42, 256, 320), torch.full((320,), 1e-3).numpy(), torch.full((256,), 1e-3).numpy(), _rand(43, rows, 256)
        block = QuantMlp(g, w1, s1, torch.zeros(160, 256, dtype=torch.int8, device="cuda"), s2)

        def call(b):
            block.down = small(b)
            return block(x, x)

        return call
    return {"x": lambda b: mlp(b[32:40], other), "residual": lambda b: mlp(other, b[32:40])}[reads]


CALLS = ([("act", r, f) for r in ("x", "u") for f in ("few", "ring", "odd")] + [("norm", r, f) for r in ("x", "residual", "weight", "alone") for f in ("few", "ring", "odd")] +
         [("gemm", r, p, o) for r in ("x", "weight", "scale") for p in ("16,1,0,2", "16,4,0,2", "64,1,0,1", "64,1,1,1") for o in (0, 1) if not (o and p == "64,1,1,1")] +
         [("mlp", r) for r in ("x", "residual", "weight")])


def _call(case):
    return _gemm_call(*case[1:]) if case[0] == "gemm" else _mlp_call(case[1]) if case[0] == "mlp" else _row_call(*case)


@pytest.mark.parametrize("case", CALLS, ids=lambda c: "-".join(map(str, c)))
def test_behind_a_predecessor_that_released_its_dependents(cuda, case):
    early, call, buffer = _Early(), _call(case), _rand(920, ROWS, 2560)
    alone = []
    for i in range(2):
        early(i, buffer[32:40])
        torch.cuda.synchronize()
        alone.append([o.clone() for o in call(buffer)])
        torch.cuda.synchronize()
    assert any(not torch.equal(_bits(a), _bits(b)) for a, b in zip(*alone))  # the two inputs tell
    got = []
    for i in range(12):
        early(i, buffer[32:40])
        got.append(call(buffer))
        if i % 3 == 2:
            torch.cuda.synchronize()
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(_bits(p), _bits(q)) for p, q in zip(alone[i % 2], g)), i


@pytest.mark.parametrize("case", CALLS, ids=lambda c: "-".join(map(str, c)))
def test_inputs_written_just_before(cuda, case):
    call, sources = _call(case), [_rand(950 + i, ROWS, 2560) for i in range(6)]
    alone = []
    for s in sources:
        alone.append([o.clone() for o in call(s)])
        torch.cuda.synchronize()
    buffer, delay, got = torch.empty_like(sources[0]), torch.empty(1 << 24, device="cuda"), []
    for s in sources:
        delay.fill_(1.0)  # the copy behind it is in the stream before it is done
        buffer.copy_(s)
        got.append(call(buffer))
    torch.cuda.synchronize()
    for a, g in zip(alone, got):
        assert all(torch.equal(_bits(p), _bits(q)) for p, q in zip(a, g))


@pytest.mark.parametrize("rows,hidden,width", [(1, 512, 1024), (8, 2560, 1024), (64, 1024, 2048), (400, 512, 768), (5, 515, 333)])
def test_calls_in_a_row(cuda, rows, hidden, width):
    """Norm, product, activation, product, each reading what the one before it writes, with nothing waited for."""
    norm, act, up, down = RmsNormQuant(), RowQuant(), QuantGemm(), QuantGemm()
    g, w1, w2 = _rand(1, hidden), _ints(2, hidden, 2 * width), _ints(3, width, hidden)
    streams = [_rand(10 + i, rows, hidden) for i in range(6)]

    def block(x, wait):
        q, s, h = norm(x, g, x)
        wait()
        both = up(q, s, w1)
        wait()
        q, s = act(both[:, :width], both[:, width:])
        wait()
        y = down(q, s, w2)
        wait()
        return [y, h]

    alone = [[o.clone() for o in block(x, torch.cuda.synchronize)] for x in streams]
    got = [block(x, lambda: None) for x in streams * 3]
    torch.cuda.synchronize()
    for a, b in zip(alone * 3, got):
        assert all(torch.equal(_bits(p), _bits(q)) for p, q in zip(a, b))


@pytest.mark.parametrize("mode", [0, 1, 2])
def test_products_that_a_shared_expert_lets_in(cuda, mode):
    """A many-row kernel that takes tensor memory and releases its dependents early, products that take theirs before they wait for it, and more of them on a
    second stream."""
    K, N, rows = 1024, 1024, 600
    shared, gemm = SharedExpertDown(trigger=1), QuantGemm(out_dtype=torch.float32)
    w, gs, u = W.make_weight(mode, K, N, 7)[0], [_rand(60 + i, rows, K) for i in range(2)], _rand(63, rows, K)
    gx, gw, routed = _rand(64, rows, 256), _rand(65, 256, 1) * 0.02, _rand(66, rows, N)
    w8, ones, other = _ints(67, 2 * N, 1024), torch.ones(rows, device="cuda"), _ints(68, rows, 2 * N)
    step = lambda i: gemm(shared(gs[i % 2], u, w, gx, gw, routed).view(torch.int8), ones, w8)
    alone = []
    for i in range(2):
        alone.append(step(i).clone())
        torch.cuda.synchronize()
    beside = gemm(other, ones, w8).clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got, more = [], []
    for i in range(24):
        got.append(step(i))
        with torch.cuda.stream(side):
            more.append(gemm(other, ones, w8))
    torch.cuda.synchronize()
    assert all(torch.equal(_bits(g), _bits(alone[i % 2])) for i, g in enumerate(got)) and all(torch.equal(m, beside) for m in more)
