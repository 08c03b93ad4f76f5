"""QkNormRope, CacheWrite and CacheRead against their formulas in 64 bits."""
import pytest
import torch

from _attention import FORMS, half_step, held, new_cache, quantised, same_bits, same_codes
from qwen38_flash_ops_b200 import CacheRead, CacheWrite, QfgError, QkNormRope

pytestmark = pytest.mark.gpu


def exact(x, weight, offset, eps, positions, freq, axes, interleaved, rotary_scale):
    """Norm and rotation in 64 bits on the host.  x [tokens, heads, dim], positions [axes, tokens]."""
    y = x.double().cpu()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * (offset + weight.double().cpu())
    n = len(freq)
    if n == 0:
        return y
    angle = positions.cpu().double()[axes].t() * torch.tensor(freq, dtype=torch.float64)
    cos, sin = (angle.cos() * rotary_scale)[:, None], (angle.sin() * rotary_scale)[:, None]
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    out = y.clone()
    out[..., a], out[..., b] = y[..., a] * cos - y[..., b] * sin, y[..., b] * cos + y[..., a] * sin
    return out


def close(got, want, dtype):
    # one rounding to `dtype`; FP32 before it: a norm of 256 squares, four products, the sine of an angle to 2^-23: 2^-19 of the row's largest value is more than all
    tol = half_step(dtype) * want.abs() + 2.0 ** -19 * want.abs().amax(-1, keepdim=True) + 1e-30
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half of the smallest subnormal
    assert torch.isfinite(got).all()
    assert ((got.double().cpu() - want).abs() <= tol).all()


CASES = [(128, None, False, 1), (128, 64, True, 1), (64, 32, False, 3), (64, 64, True, 2), (256, 64, False, 1), (256, 256, True, 3), (128, 0, False, 1)]


@pytest.mark.parametrize("tokens,q_heads,kv_heads", [(1, 1, 1), (5, 8, 2), (240, 40, 4), (296, 64, 8), (300, 3, 3), (700, 12, 4)])
@pytest.mark.parametrize("dim,rotary,interleaved,n_axes", CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_norm_and_rotation(cuda, dtype, dim, rotary, interleaved, n_axes, tokens, q_heads, kv_heads):
    gen = torch.Generator().manual_seed(tokens + dim)
    r = dim if rotary is None else rotary
    channel = torch.exp(torch.randn(dim, generator=gen))
    q, k = ((torch.randn(tokens, h, dim, generator=gen) * channel).to(dtype).cuda() for h in (q_heads, kv_heads))
    qw, kw = ((1 + 0.3 * torch.randn(dim, generator=gen)).to(dtype).cuda() for _ in range(2))
    positions = torch.randint(-5000, 1 << 20, (n_axes, tokens), generator=gen).cuda()
    sections = [r // 2 - (n_axes - 1) * (r // 2 // n_axes)] + [r // 2 // n_axes] * (n_axes - 1) if r else None
    op = QkNormRope(dim, rotary_dim=rotary, base=500000.0, sections=sections if n_axes > 1 else None, interleaved=interleaved, eps=1e-5, weight_offset=0.25, rotary_scale=1.125)
    got_q, got_k = op(q, k, positions[0] if n_axes == 1 else positions, qw, kw)
    freq = [500000.0 ** (-i / (r // 2)) for i in range(r // 2)]
    axes = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)] if n_axes > 1 else [0] * (r // 2), dtype=torch.long)
    for got, x, w in ((got_q, q, qw), (got_k, k, kw)):
        close(got, exact(x, w, 0.25, 1e-5, positions, freq, axes, interleaved, 1.125), dtype)


def test_without_weights_with_fp32_weights_and_given_frequencies(cuda):
    gen = torch.Generator().manual_seed(2)
    q, k = torch.randn(33, 4, 128, generator=gen).bfloat16().cuda(), torch.randn(33, 2, 128, generator=gen).bfloat16().cuda()
    w = (1 + 0.3 * torch.randn(128, generator=gen)).cuda()
    positions = torch.arange(33, dtype=torch.int32).cuda()
    freq = [0.5 ** (i / 3) * 7 for i in range(64)]  # up to seven radians a position
    op = QkNormRope(128, inv_freq=freq, axes=[0] * 64)
    axes = torch.zeros(64, dtype=torch.long)
    got_q, got_k = op(q, k, positions, None, w)
    close(got_q, exact(q, None, 0, 1e-6, positions[None], freq, axes, False, 1.0), torch.bfloat16)
    close(got_k, exact(k, w, 0, 1e-6, positions[None], freq, axes, False, 1.0), torch.bfloat16)


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("tokens", [7, 400])
def test_strided_rows_of_one_projection(cuda, tokens, shift):
    """Parts of the columns of one matrix, whose rows lie off 16 bytes (shift 1)."""
    gen = torch.Generator().manual_seed(3)
    both = torch.randn(tokens, 10 * 64 + 5 * shift, generator=gen).bfloat16().cuda()
    q, k, v = (both[:, shift + 64 * a:shift + 64 * b].unflatten(1, (-1, 64)) for a, b in ((0, 6), (6, 8), (8, 10)))
    assert q.data_ptr() == both.data_ptr() + 2 * shift
    w, positions, slots = torch.ones(64).bfloat16().cuda(), torch.arange(tokens).cuda(), torch.randperm(13 * 32, generator=gen)[:tokens].cuda()
    a, b = new_cache("nvfp4", 13, 2, 64), new_cache("nvfp4", 13, 2, 64)
    op = QkNormRope(64)
    got_q, got_k = op(q, k, positions, w, w, v, a, slots, keys=True)
    want_q, want_k = op(q.contiguous(), k.contiguous(), positions, w, w, v.contiguous(), b, slots, keys=True)
    assert torch.equal(got_q, want_q) and torch.equal(got_k, want_k)
    assert all(same_bits(getattr(a, n), getattr(b, n)) for n in ("k", "k_scale", "v", "v_scale"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,q_heads,kv_heads,dim", [(297, 1, 1, 64), (593, 3, 1, 64), (700, 24, 8, 128), (1185, 8, 2, 128), (1337, 24, 4, 256), (2369, 5, 5, 128), (4097, 16, 2, 64), (9600, 2, 1, 256)])
def test_rows_do_not_depend_on_the_call_they_are_in(cuda, tokens, q_heads, kv_heads, dim, dtype):
    """Tokens go one to eight to a block, by their number: the same bits as in calls of a hundred, each of whose rows is a warp's."""
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    q, k, v = (torch.randn(tokens, h, dim, generator=gen, device="cuda").to(dtype) for h in (q_heads, kv_heads, kv_heads))
    w, positions, slots, op = torch.rand(dim, generator=gen, device="cuda"), torch.arange(tokens, device="cuda") * 37, torch.arange(tokens, device="cuda"), QkNormRope(dim)
    caches = [new_cache("e4m3", -(-tokens // 32), kv_heads, dim) for _ in range(3)]
    got = op(q, k, positions, w, w, v=v, cache=caches[0], slots=slots, keys=True)
    CacheWrite()(got[1], v, caches[2], slots)
    for i in range(0, tokens, 100):
        part = op(q[i:i + 100], k[i:i + 100], positions[i:i + 100], w, w, v=v[i:i + 100], cache=caches[1], slots=slots[i:i + 100], keys=True)
        assert all(torch.equal(a[i:i + 100], b) for a, b in zip(got, part))
    assert all(same_bits(getattr(caches[0], name), getattr(caches[1], name)) for name in ("k", "v", "k_scale", "v_scale"))
    assert all(same_bits(getattr(caches[0], name), getattr(caches[2], name)) for name in (("k", "v", "k_scale", "v_scale") if dtype == torch.float32 else ("v", "v_scale")))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim,rotary,interleaved", [(128, 128, False), (64, 32, False), (64, 64, True), (256, 128, False), (256, 96, False)])
@pytest.mark.parametrize("tokens", [3, 270, 330])
def test_the_cache_holds_the_rotated_keys(cuda, form, dim, rotary, interleaved, tokens):
    gen = torch.Generator().manual_seed(4)
    channel = torch.exp(torch.randn(dim, generator=gen))
    q, k, v = ((torch.randn(tokens, h, dim, generator=gen) * channel).bfloat16().cuda() for h in (4, 2, 2))
    w, positions = (1 + 0.3 * torch.randn(dim, generator=gen)).bfloat16().cuda(), torch.randint(0, 100000, (1, tokens), generator=gen).cuda()
    cache = new_cache(form, 12, 2, dim)
    slots = torch.randperm(12 * 32, generator=gen)[:tokens]
    op = QkNormRope(dim, rotary_dim=rotary, interleaved=interleaved)
    alone = op(q, k, positions[0], w, w)
    assert torch.equal(op(q, k, positions[0], w, w, v, cache, slots.cuda()), alone[0])
    freq = [10000.0 ** (-i / (rotary // 2)) for i in range(rotary // 2)]
    want = exact(k, w, 0, 1e-6, positions, freq, torch.zeros(rotary // 2, dtype=torch.long), interleaved, 1.0)
    at = (slots // 32, slice(None), slots % 32)
    got = held(cache.k, cache.k_scale, cache.k_unit)[at]
    scale = cache.k_scale.cpu().double()[at]
    room = 2.0 ** -19 * want.abs().amax(-1, keepdim=True)  # FP32 ahead of the rounding
    if form == "e4m3":
        assert ((scale - want.abs().amax(-1) / 448).abs() <= 2.0 ** -19 * scale).all()
        step = torch.maximum(half_step(torch.float8_e4m3fn) * want.abs(), 2.0 ** -10 * scale[..., None])
    else:
        most = want.unflatten(-1, (-1, 16)).abs().amax(-1) / (6 * cache.k_unit)
        assert ((scale - most).abs() <= torch.maximum(half_step(torch.float8_e4m3fn) * most, torch.tensor(2.0 ** -9)) * (1 + 2.0 ** -10)).all()
        unit = scale.repeat_interleave(16, -1) * cache.k_unit
        a = want.abs() / unit
        step = torch.where(a < 2, 0.25, torch.where(a < 4, 0.5, 1.0)) * unit
    assert ((got - want).abs() <= step + room).all()
    codes, scales = quantised(v.cpu().double(), form, cache.v_unit)  # values are as they came: bit for bit
    assert same_codes(cache.v[at[0].cuda(), :, at[2].cuda()] if form == "nvfp4" else cache.v.view(torch.uint8)[at[0].cuda(), :, at[2].cuda()], codes.view(torch.uint8), form)
    raw = cache.v_scale.view(torch.uint8) if form == "nvfp4" else cache.v_scale
    assert same_bits(raw[at[0].cuda(), :, at[2].cuda()], scales.view(torch.uint8) if form == "nvfp4" else scales)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_written_rows_bit_for_bit(cuda, form, dtype, dim):
    """Every rounding of a write is one of the value itself: half-way values, zeros, tiny and huge blocks."""
    gen = torch.Generator().manual_seed(5)
    k, v = ((torch.randn(90, 3, dim, generator=gen) * torch.exp2(torch.randint(-14, 9, (90, 3, 1), generator=gen).float())).to(dtype) for _ in range(2))
    k[0], v[1, 1] = 0, 0
    k[2, 0, :16] = torch.tensor([6, 5, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, -6]).to(dtype)
    k[3, 0, :] = torch.finfo(dtype).tiny if dtype != torch.float16 else 2.0 ** -24
    v[4, 0, 0] = 30000.0
    cache = new_cache(form, 4, 3, dim, k_unit=1.0, v_unit=0.125)
    slots = torch.randperm(4 * 32, generator=gen)[:90]
    CacheWrite()(k.cuda(), v.cuda(), cache, slots.cuda())
    for rows, codes, scale, unit in ((k, cache.k, cache.k_scale, 1.0), (v, cache.v, cache.v_scale, 0.125)):
        want, scales = quantised(rows.double(), form, unit)
        assert same_codes(codes.view(torch.uint8).cpu()[slots // 32, :, slots % 32], want.view(torch.uint8), form)
        raw = scale.view(torch.uint8).cpu() if form == "nvfp4" else scale.cpu()
        assert same_bits(raw[slots // 32, :, slots % 32], scales.view(torch.uint8) if form == "nvfp4" else scales)
    out = [torch.full((200, 3, dim), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
    table = torch.tensor([[2, 0, 3], [1, -1, 9]], dtype=torch.int32).cuda()  # pages that are none of the cache's
    offsets = torch.tensor([3, 90, 190], dtype=torch.int32).cuda()  # and a sequence past its three pages
    CacheRead(dtype=dtype)(cache, table, offsets, 200, out=out)
    for got, codes, scale, unit in ((out[0], cache.k, cache.k_scale, 1.0), (out[1], cache.v, cache.v_scale, 0.125)):
        pages = held(codes, scale, unit).transpose(1, 2)
        first = torch.cat([pages[2], pages[0], pages[3]])[:87]
        want = torch.cat([first, pages[1], torch.zeros(68, 3, dim, dtype=torch.float64)])
        got = got.cpu()
        assert (got[:3] == 7).all() and (got[190:] == 7).all()
        assert torch.equal(got[3:190], want.float().to(dtype))  # FP32 holds code times scale times a power of two exactly


@pytest.mark.parametrize("form", FORMS)
def test_slots_outside_and_rows_that_are_no_numbers(cuda, form):
    cache = new_cache(form, 2, 1, 64)
    k = torch.randn(6, 1, 64).bfloat16().cuda()
    v = k.clone()
    k[1, 0, 20], v[2, 0, 63] = float("inf"), float("nan")
    slots = torch.tensor([-1, 5, 6, 64, 1 << 40, -(1 << 40)]).cuda()
    CacheWrite()(k, v, cache, slots)
    written = torch.zeros(64, dtype=torch.bool)
    written[5:7] = True
    kv = [held(c, s, u).transpose(1, 2).flatten(0, 1)[:, 0] for c, s, u in ((cache.k, cache.k_scale, 0.25), (cache.v, cache.v_scale, 0.0625))]
    for rows in kv:
        assert (rows[~written] == 0).all()
    block = slice(16, 32) if form == "nvfp4" else slice(0, 64)
    assert torch.isnan(kv[0][5, block]).all() and torch.isnan(kv[1][6, slice(48, 64) if form == "nvfp4" else block]).all()
    keep = torch.ones(64, dtype=torch.bool)
    keep[block] = False
    assert torch.isfinite(kv[0][5, keep]).all() and torch.isfinite(kv[0][6]).all() and torch.isfinite(kv[1][5]).all()


def test_calls_that_are_refused(cuda):
    x = torch.zeros(4, 2, 128, device="cuda").bfloat16()
    at, cache, slots = torch.arange(4, device="cuda"), new_cache("e4m3", 1, 2, 128), torch.arange(4, device="cuda")
    op, three = QkNormRope(128), QkNormRope(128, sections=[32, 16, 16])
    w = torch.ones(128, device="cuda").bfloat16()
    for call, message in ((lambda: op(x, x[:3], at), "as many tokens"), (lambda: op(x, x, at[:3]), r"positions must be \[4\]"), (lambda: op(x, x), "no positions"),
                          (lambda: op(x, x, at.float()), "positions must be"), (lambda: three(x, x, at), r"positions must be \[3, 4\]"), (lambda: op(x, x.float(), at), "k must be bfloat16"),
                          (lambda: op(x[..., :64], x, at), "channels|128"), (lambda: op(x, x, at, w[:64]), "128 elements"), (lambda: op(x, x, at, w, w.float()), "one type"),
                          (lambda: op(x, x, at, w, w, x), "go with a cache"), (lambda: op(x, x, at, w, w, x, cache), "slots must be"),
                          (lambda: op(x, x, at, w, w, x[:, :1], cache, slots), "must fit k"), (lambda: op(x, x, at, w, w, x, cache, slots[:3]), "must fit k"),
                          (lambda: op(x.transpose(1, 2), x, at), "128"), (lambda: op(x[:, ::2], x, at), None), (lambda: op(x, x, at, w, w, x, "cache", slots), "KvCache"),
                          (lambda: CacheWrite()(x, x, cache, slots.int()), "slots must be"), (lambda: CacheWrite()(x[:, :1], x[:, :1], cache, slots), "must fit one another"),
                          (lambda: CacheRead()(cache, at[None].int(), at[:3].int(), 4), "offsets"), (lambda: CacheRead()(cache, at[None], at[:2].int(), 4), "the table must be")):
        if message is None:
            call()  # one head of two: allowed
            continue
        with pytest.raises(QfgError, match=message):
            call()


def test_captured_and_replayed(cuda):
    """A graph of a write and a read, replayed on other inputs."""
    op, back = QkNormRope(128), CacheRead()
    gen = torch.Generator().manual_seed(6)
    new = lambda h: torch.randn(9, h, 128, generator=gen).bfloat16().cuda()
    q, k, v, w, at, slots = new(4), new(2), new(2), torch.ones(128).bfloat16().cuda(), torch.arange(9).cuda(), torch.arange(9).cuda()
    cache, table, offsets = new_cache("nvfp4", 1, 2, 128), torch.zeros(1, 1, dtype=torch.int32).cuda(), torch.tensor([0, 9], dtype=torch.int32).cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = op(q, k, at, w, w, v, cache, slots)
        rows = back(cache, table, offsets, 9)
    for i in range(2):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=gen))
        at.add_(1000 * i)
        graph.replay()
        other = new_cache("nvfp4", 1, 2, 128)
        assert torch.equal(got, op(q, k, at, w, w, v, other, slots))
        assert all(torch.equal(a, b) for a, b in zip(rows, back(other, table, offsets, 9)))
