"""CacheAttention against softmax(q k^T) v in 64 bits over what the cache stands for."""
import math

import pytest
import torch

from _attention import FORMS, attention, fill, half_step, held, new_cache
from qwen38_flash_ops_b200 import CacheAttention, QfgError

pytestmark = pytest.mark.gpu


def a_case(form, dim, heads, group, tokens, lengths, dtype, page=32, seed=1, spare=2):
    gen = torch.Generator().manual_seed(seed)
    most = max(1, -(-max(lengths) // page))
    cache = new_cache(form, len(lengths) * most + spare, heads, dim, page)
    fill(cache, gen)
    table = torch.randperm(cache.pages, generator=gen)[:len(lengths) * most].view(-1, most).int()
    q = torch.randn(len(lengths), tokens, heads * group, dim, generator=gen).to(dtype)
    return cache, table.cuda(), q.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()


def check(got, lse, cache, table, q, lengths, scale):
    seqs, tokens, heads, dim = q.shape
    group = heads // cache.kv_heads
    k, v = held(cache.k, cache.k_scale, cache.k_unit), held(cache.v, cache.v_scale, cache.v_unit)
    for i, n in enumerate(lengths.tolist()):
        pages = table[i].cpu().long()
        for h in range(cache.kv_heads):
            ki, vi = (t[pages, h].flatten(0, 1)[:n] for t in (k, v))
            rows = q[i, :, h * group:(h + 1) * group].cpu().double().flatten(0, 1)
            seen = (n - tokens + 1 + torch.arange(tokens)).clamp(min=0).repeat_interleave(group)
            y, size, log = attention(rows, ki, vi, seen, scale)
            # weights are FP16 (2^-11 of each, below 2^-14 of the largest 2^-25 of it), scores FP32: sums of 256 products, off by 2^-18 of what they add up
            slack = (rows.abs() @ ki.abs().t()).amax() * scale * 2.0 ** -18 if n else 0.0
            tol = half_step(q.dtype) * y.abs() + (2.0 ** -11 + slack) * 1.01 * size + n * 2.0 ** -25 * (vi.abs().amax() if n else 0.0) + 2.0 ** -25
            a = got[i, :, h * group:(h + 1) * group].cpu().double().flatten(0, 1)
            assert torch.isfinite(a).all() and ((a - y).abs() <= tol).all(), (i, h, ((a - y).abs() / tol).max())
            assert (a[seen == 0] == 0).all()
            if lse is not None:
                b = lse[i, :, h * group:(h + 1) * group].cpu().double().flatten()
                some = seen > 0
                assert ((b - log).abs()[some] <= slack + 2.0 ** -18 * (1 + log.abs()[some])).all() and (b[~some] == -math.inf).all()


LENGTHS = [[1], [31, 32, 33], [0, 5, 0, 64], [200, 1, 777], [1500, 64, 0, 129, 96, 95, 1]]


@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
@pytest.mark.parametrize("heads,group,tokens", [(1, 1, 1), (2, 8, 1), (3, 5, 2), (1, 12, 3), (2, 16, 1)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_against_64_bits(cuda, form, dim, heads, group, tokens, lengths):
    dtype = torch.float16 if dim == 128 and group == 5 else torch.bfloat16
    cache, table, q, n = a_case(form, dim, heads, group, tokens, lengths, dtype)
    got, lse = CacheAttention()(q, cache, table, n, lse=True)
    check(got, lse, cache, table, q, n, 1 / math.sqrt(dim))
    assert torch.equal(got, CacheAttention()(q, cache, table, n))  # and again, the same bits


@pytest.mark.parametrize("form,dim,heads,group,tokens,lengths,page", [
    ("nvfp4", 128, 8, 8, 1, [9000, 4097], 64),    # pieces of many blocks
    ("e4m3", 128, 2, 4, 8, [20000], 96),          # four blocks of rows, pages that do not divide a length
    ("nvfp4", 64, 1, 3, 1, [100] * 300, 32),      # more sequences than a block has threads
    ("e4m3", 64, 4, 1, 1, [0] * 299 + [33], 32),  # nearly all empty
    ("nvfp4", 256, 1, 1, 40, [50, 39, 3000], 160),
])
def test_shapes_of_a_server(cuda, form, dim, heads, group, tokens, lengths, page):
    cache, table, q, n = a_case(form, dim, heads, group, tokens, lengths, torch.bfloat16, page)
    check(CacheAttention(scale=0.3 / math.sqrt(dim))(q, cache, table, n), None, cache, table, q, n, 0.3 / math.sqrt(dim))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim,group,tokens,lengths", [(64, 8, 1, [30011]), (128, 4, 2, [14000, 100]), (128, 16, 1, [12001]), (256, 2, 1, [13000, 0, 25000])])
def test_few_heads_of_long_sequences(cuda, form, dim, group, tokens, lengths):
    """Shares of several tiles where there could be one for each warp."""
    cache, table, q, n = a_case(form, dim, 1, group, tokens, lengths, torch.bfloat16, page=64)
    got, lse = CacheAttention()(q, cache, table, n, lse=True)
    check(got, lse, cache, table, q, n, 1 / math.sqrt(dim))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_nothing_behind_a_length_takes_part(cuda, form, dim):
    lengths = [45, 1, 0, 130]
    cache, table, q, n = a_case(form, dim, 2, 4, 2, lengths, torch.bfloat16, page=64)
    want, log = CacheAttention()(q, cache, table, n, lse=True)
    live = torch.zeros(cache.pages, cache.page, dtype=torch.bool)
    for i, m in enumerate(lengths):
        for t in range(m):
            live[table[i, t // 64].item(), t % 64] = True
    dead = ~live.cuda()
    for t, nan in ((cache.k, 0x7F), (cache.v, 0x7F), (cache.k_scale, 0x7F), (cache.v_scale, 0x7F)):  # E4M3's NaN
        if t.dtype == torch.float32:
            t.transpose(1, 2)[dead] = float("nan")
        else:
            t.view(torch.uint8).transpose(1, 2)[dead] = nan
    wide = torch.cat([table, torch.full((4, 3), 1 << 30, dtype=torch.int32).cuda()], dim=1)  # entries that no length reaches may be anything
    got, also = CacheAttention()(q, cache, wide, n, lse=True)
    assert torch.equal(got, want) and torch.equal(also, log)


def test_pages_outside_the_cache_and_lengths_past_the_table(cuda):
    cache, table, q, _ = a_case("nvfp4", 128, 1, 2, 1, [96, 96], torch.bfloat16)
    n = torch.tensor([96, 500], dtype=torch.int32).cuda()
    table[0, 1], table[1, 0] = -3, cache.pages
    got = CacheAttention()(q, cache, table, n)
    for i, pages in ((0, [0, 2]), (1, [1, 2])):  # the tokens that are there
        ids = table[i:i + 1, pages].contiguous()
        want = CacheAttention()(q[i:i + 1], cache, ids, torch.tensor([64], dtype=torch.int32).cuda())
        assert (got[i] - want[0]).abs().max() <= 2.0 ** -7 * want.abs().max()
    assert (CacheAttention()(q, cache, table, -n) == 0).all()
    assert (CacheAttention()(q, cache, table[:, :0], n) == 0).all()


@pytest.mark.parametrize("form", FORMS)
def test_extreme_scores_and_scales(cuda, form):
    """Scores far apart, q far from 1, values whose scales span many powers of two, and a q that is no number: its row alone."""
    cache, table, q, n = a_case(form, 128, 1, 4, 2, [700, 64], torch.bfloat16, spare=0)
    q[0, 0, 0] *= 2.0 ** 60
    q[0, 0, 1] *= 2.0 ** -70
    q[1, 1, 2] *= 300
    if form == "e4m3":
        cache.v_scale.mul_(torch.exp2(torch.randint(-30, 5, cache.v_scale.shape, generator=torch.Generator().manual_seed(1)).float()).cuda())
    got = CacheAttention()(q, cache, table, n)
    k, v = held(cache.k, cache.k_scale, cache.k_unit), held(cache.v, cache.v_scale, cache.v_unit)
    rows = q[0, 0].cpu().double()
    y, _, _ = attention(rows[:2], k[table[0].cpu().long(), 0].flatten(0, 1)[:699], v[table[0].cpu().long(), 0].flatten(0, 1)[:699], torch.tensor([699, 699]), 128 ** -0.5)
    a = got[0, 0, :2].cpu().double()
    # One key alone, within a rounding of the weight; and the mean of all values, whose weights are one.  In eight bits a weight is FP16 times the value's scale, measured
    # from the largest score + log2(scale): of a score past 2^24 (here 2^66) FP32 keeps nothing of that logarithm, the point is the score and the weight the scale itself,
    # which FP16 holds to 2^-25: relative to it 2^-25 / scale.
    winner = (rows[0] @ k[table[0].cpu().long(), 0].flatten(0, 1)[:699].t()).argmax()
    small = 2.0 ** -25 / cache.v_scale[table[0].long(), 0].flatten()[winner].item() if form == "e4m3" else 0.0
    assert ((a[0] - y[0]).abs() <= (2.0 ** -7 + small) * y[0].abs() + 1e-30).all()
    assert ((a[1] - y[1]).abs() <= half_step(q.dtype) * y[1].abs() + 2.0 ** -10 * v.abs().amax()).all()
    q[0, 1, 3, 5] = float("nan")
    bad = CacheAttention()(q, cache, table, n)
    assert torch.isnan(bad[0, 1, 3]).all()
    bad[0, 1, 3], got[0, 1, 3] = 0, 0
    # the rows of a head take up their maxima together, so that the others may be rounded at other points
    assert ((bad.double() - got.double()).abs() <= 2 * half_step(q.dtype) * got.abs().double() + 2.0 ** -10 * v.abs().amax().item()).all()


def test_strided_queries_and_one_token_in_three_dimensions(cuda):
    cache, table, q, n = a_case("nvfp4", 128, 2, 4, 2, [70, 40], torch.float16)
    want = CacheAttention()(q, cache, table, n)
    wide = torch.zeros(2, 3, 5 * 8 * 128, device="cuda").half()
    view = wide[:, 1:, 1024:2048].unflatten(2, (8, 128))
    view.copy_(q)
    out = torch.empty_like(want)
    assert torch.equal(CacheAttention()(view, cache, table, n), want)
    assert CacheAttention()(view, cache, table, n, out=out) is out and torch.equal(out, want)
    pitched = torch.zeros(2, 7, dtype=torch.int32, device="cuda")
    pitched[:, :table.shape[1]] = table
    assert torch.equal(CacheAttention()(q, cache, pitched[:, :table.shape[1]], n), want)
    one = q[:, 1].contiguous()
    assert torch.equal(CacheAttention()(one, cache, table, n), CacheAttention()(one[:, None].contiguous(), cache, table, n)[:, 0])


def test_parts_are_joined_by_their_logarithms(cuda):
    """Two halves of a sequence, one call each, joined on the outside: what lse is for."""
    cache, table, q, n = a_case("nvfp4", 128, 2, 8, 1, [640, 640], torch.float16, page=64)
    whole = CacheAttention()(q, cache, table, n).double()
    half = torch.full_like(n, 320)
    a, la = CacheAttention()(q, cache, table[:, :5].contiguous(), half, lse=True)
    b, lb = CacheAttention()(q, cache, table[:, 5:].contiguous(), half, lse=True)
    w = torch.sigmoid((la - lb).double())[..., None]
    assert ((a.double() * w + b.double() * (1 - w) - whole).abs() <= 2.0 ** -9 * (a.abs() + b.abs()).double() + 2.0 ** -10).all()


def test_captured_replayed_and_at_once(cuda):
    """A graph, replayed when lengths, table and q have changed; and calls on two streams, each with a workspace of its own."""
    cache, table, q, n = a_case("nvfp4", 128, 4, 8, 1, [3000, 50, 1200], torch.bfloat16)
    op = CacheAttention()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = op(q, cache, table, n)
    with torch.cuda.graph(other, pool=graph.pool()):
        also = op(q, cache, table, n)
    for lengths in ([3000, 50, 1200], [1, 2900, 0], [0, 0, 0], [77, 78, 79]):
        n.copy_(torch.tensor(lengths))
        q.normal_()
        table.copy_(table.flip(1))
        graph.replay()
        want = op(q, cache, table, n)
        assert torch.equal(got, want)
        other.replay()
        assert torch.equal(also, want)
    n.copy_(torch.tensor([3000, 50, 1200]))
    want = op(q, cache, table, n)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(op(q, cache, table, n))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_calls_that_are_refused(cuda):
    cache, table, q, n = a_case("nvfp4", 128, 2, 4, 1, [70, 40], torch.bfloat16)
    op = CacheAttention()
    for call, message in ((lambda: op(q.float(), cache, table, n), "BF16 or FP16"), (lambda: op(q[..., :64], cache, table, n), "128"), (lambda: op(q[:, :, :3], cache, table, n), "multiple"),
                          (lambda: op(q, cache, table.long(), n), "table must be"), (lambda: op(q, cache, table, n.long()), "lengths must be"), (lambda: op(q, cache, table[:1], n), "each of 2"),
                          (lambda: op(q, cache, table, n[:1]), "each of 2"), (lambda: op(q.cpu(), cache, table, n), "current CUDA device"), (lambda: op(q, None, table, n), "KvCache"),
                          (lambda: op(q, cache, table, n, out=q.float()), "out must be"), (lambda: op(q[:, :, ::2], cache, table, n), "beside one another")):
        with pytest.raises(QfgError, match=message):
            call()
