"""PromptAttention against softmax(q k^T) v in 64 bits."""
import math

import pytest
import torch

from _attention import attention, half_step
from qwen38_flash_ops_b200 import PromptAttention, QfgError, _lib

pytestmark = pytest.mark.gpu


def offsets(lengths, first=0):
    return torch.tensor([first, *(first + torch.tensor(lengths).cumsum(0)).tolist()], dtype=torch.int32).cuda()


def a_case(queries, keys, heads, kv_heads, dim, dtype, seed=1, spare=0):
    gen = torch.Generator().manual_seed(seed)
    q = torch.randn(sum(queries) + spare, heads, dim, generator=gen).to(dtype).cuda()
    k, v = (torch.randn(sum(keys) + spare, kv_heads, dim, generator=gen).to(dtype).cuda() for _ in range(2))
    return q, k, v


def check(got, lse, q, k, v, queries, keys, causal, scale):
    dtype, group = q.dtype, q.shape[1] // k.shape[1]
    a = b = 0
    for n, m in zip(queries, keys):
        for h in range(k.shape[1]):
            ki, vi = k[b:b + m, h].cpu().double(), v[b:b + m, h].cpu().double()
            rows = q[a:a + n, h * group:(h + 1) * group].cpu().double().transpose(0, 1).flatten(0, 1)
            seen = ((torch.arange(n) + 1 + m - n).clamp(min=0) if causal else torch.full((n,), m)).repeat(group)
            y, size, log = attention(rows, ki, vi, seen, scale)
            # weights are rounded to the inputs' type (BF16: made to 7.5e-5; FP16: below 2^-14 of the largest 2^-25 of it); scores are FP32 sums of 128 products, cut off
            # at every 16 by the tensor core: off by 2^-17 of what they add up
            slack = (rows.abs() @ ki.abs().t()).amax() * scale * 2.0 ** -17 if n and m else 0.0
            tol = half_step(dtype) * y.abs() + (half_step(dtype) + 1e-4 + slack) * size + m * 2.0 ** -25 * (vi.abs().amax() if m else 0.0) + 2.0 ** -25
            got_rows = got[a:a + n, h * group:(h + 1) * group].cpu().double().transpose(0, 1).flatten(0, 1)
            assert torch.isfinite(got_rows).all() and ((got_rows - y).abs() <= tol).all(), (a, h, ((got_rows - y).abs() / tol).max())
            assert (got_rows[seen == 0] == 0).all()
            if lse is not None:
                c = lse[a:a + n, h * group:(h + 1) * group].cpu().double().t().flatten()
                some = seen > 0
                assert ((c - log).abs()[some] <= slack + 1e-4 + 2.0 ** -18 * log.abs()[some]).all() and (c[~some] == -math.inf).all()
        a, b = a + n, b + m


LENGTHS = [([1], [1]), ([1], [300]), ([128], [128]), ([129], [129]), ([255, 256, 257], [255, 256, 257]), ([0, 3, 0, 700, 1], [0, 3, 5, 700, 130]), ([300, 5], [100, 0]), ([64] * 40, [65] * 40)]


@pytest.mark.parametrize("queries,keys", LENGTHS, ids=lambda v: str(v[:6]))
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (6, 2), (8, 1)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
def test_against_64_bits(cuda, causal, dtype, dim, heads, kv_heads, queries, keys):
    q, k, v = a_case(queries, keys, heads, kv_heads, dim, dtype)
    got, lse = PromptAttention(causal=causal)(q, k, v, offsets(queries), offsets(keys), lse=True)
    check(got, lse, q, k, v, queries, keys, causal, 1 / math.sqrt(dim))
    assert torch.equal(got, PromptAttention(causal=causal)(q, k, v, offsets(queries), offsets(keys)))


@pytest.mark.parametrize("dim", [64, 128])
def test_a_long_prompt(cuda, dim):
    q, k, v = a_case([3001], [3001], 2, 1, dim, torch.bfloat16)
    q *= 4  # scores that make the maximum be taken up again and again
    check(PromptAttention(scale=0.2)(q, k, v, offsets([3001])), None, q, k, v, [3001], [3001], True, 0.2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_of_others_take_no_part(cuda, dtype, causal):
    """NaN in the keys, values and queries of no sequence and of the next one; rows ahead and behind are left as they were."""
    queries, keys, first = [70, 200, 129], [70, 300, 131], 13
    q, k, v = a_case(queries, keys, 4, 2, 128, dtype, spare=40)
    qo, ko = offsets(queries, first), offsets(keys, first)
    op = PromptAttention(causal=causal)
    want = op(q, k, v, qo, ko)
    for t, ends in ((q, qo), (k, ko), (v, ko)):
        t[:first], t[ends[-1]:] = float("nan"), float("nan")
        t[ends[1]:ends[2]] = float("inf")
    out = torch.full_like(q, 5)
    assert op(q, k, v, qo, ko, out=out) is out
    for i in (0, 2):
        assert torch.equal(out[qo[i]:qo[i + 1]], want[qo[i]:qo[i + 1]])
    assert (out[:first] == 5).all() and (out[qo[-1]:] == 5).all() and torch.isnan(out[qo[1]:qo[2]].float()).all()


def test_one_bad_query_is_alone(cuda):
    q, k, v = a_case([300], [300], 2, 1, 64, torch.bfloat16)
    want = PromptAttention()(q, k, v, offsets([300]))
    q[77, 1, 3] = float("nan")
    got = PromptAttention()(q, k, v, offsets([300]))
    assert torch.isnan(got[77, 1].float()).all()
    got[77, 1], want[77, 1] = 0, 0
    assert ((got.double() - want.double()).abs() <= 2 * half_step(q.dtype) * (want.abs() + v.abs().amax()).double()).all()


def test_extreme_scores(cuda):
    """Scores far from one another and from zero, all of them far below zero, and equal ones."""
    q, k, v = a_case([256], [256], 1, 1, 128, torch.float16)
    k[:, 0, 0], q[:, 0, 0] = 60.0, -300.0  # every score is below -1000
    q[200:, 0] = 0
    q[:50] *= 100
    q[:50, 0, 0] = 0
    check(PromptAttention(scale=0.25)(q, k, v, offsets([256])), None, q, k, v, [256], [256], True, 0.25)


def test_parts_of_a_projection_and_chunks(cuda):
    """Views of one matrix's columns; and a prompt in two chunks, the second of which attends to the first's keys as well, as the whole of it."""
    gen = torch.Generator().manual_seed(3)
    both = torch.randn(400, 12 * 64, generator=gen).half().cuda()
    q, k, v = (both[:, 64 * a:64 * b].unflatten(1, (-1, 64)) for a, b in ((0, 8), (8, 10), (10, 12)))
    op = PromptAttention()
    whole = op(q, k, v, offsets([400]))
    assert torch.equal(whole, op(q.contiguous(), k.contiguous(), v.contiguous(), offsets([400])))
    for cut in (128, 131):
        assert torch.equal(op(q[:cut], k[:cut], v[:cut], offsets([cut])), whole[:cut])
        rest = op(q[cut:], k, v, offsets([400 - cut]), offsets([400]))
        assert ((rest.double() - whole[cut:].double()).abs() <= 2 * half_step(torch.float16) * (whole[cut:].abs() + v.abs().amax()).double()).all()


def test_captured_and_on_two_streams(cuda):
    q, k, v = a_case([300, 200], [300, 200], 8, 2, 128, torch.bfloat16)
    at, op, graph = offsets([300, 200]), PromptAttention(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = op(q, k, v, at)
    for lengths in ([300, 200], [1, 499], [500, 0], [0, 77]):
        at.copy_(offsets(lengths))
        q.normal_()
        graph.replay()
        assert torch.equal(got[:sum(lengths)], op(q, k, v, at)[:sum(lengths)])
    at.copy_(offsets([300, 200]))
    want, streams, outs = op(q, k, v, at), [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for i in range(10):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(op(q, k, v, at))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_offsets_that_are_none(cuda):
    """Offsets that fall, or leave the tensors, reach nothing outside of them."""
    q, k, v = a_case([200], [200], 2, 1, 64, torch.bfloat16)
    for qo, ko in (([0, 100, 50, 200], [0, 100, 50, 200]), ([-5, 90, 1000, 2000], [-5, 90, 1000, 2000]), ([0, 200, 200, 200], [150, 400, 3, -9])):
        PromptAttention()(q, k, v, torch.tensor(qo, dtype=torch.int32).cuda(), torch.tensor(ko, dtype=torch.int32).cuda())
    torch.cuda.synchronize()


@pytest.mark.parametrize("seqs", [2, 31, 32, 33, 70, 500])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_more_blocks_than_the_gpu_holds(cuda, causal, dim, seqs):
    """Blocks take on the work of others, the longest first (of more than 32 sequences in the order of their rows): every row is written once, whatever its turn."""
    gen = torch.Generator().manual_seed(seqs)
    most = 9000 // seqs
    queries = [int(n) for n in torch.randint(0, most, (seqs,), generator=gen)]
    keys = [max(0, n + int(d)) for n, d in zip(queries, torch.randint(-40, 400, (seqs,), generator=gen))]
    q, k, v = a_case(queries, keys, 24, 8, dim, torch.bfloat16, seed=seqs)
    out = torch.full_like(q, float("nan"))
    op = PromptAttention(causal=causal)
    op(q, k, v, offsets(queries), offsets(keys), out=out)
    assert torch.isfinite(out).all() and torch.equal(out, op(q, k, v, offsets(queries), offsets(keys)))
    # each sequence by itself, where no block waits for a place
    a = b = 0
    for n, m in zip(queries, keys):
        for h in range(0, 24, 12):
            alone = op(q[a:a + n, h:h + 12], k[b:b + m, h // 3:h // 3 + 4], v[b:b + m, h // 3:h // 3 + 4], offsets([n]), offsets([m]))
            assert torch.equal(out[a:a + n, h:h + 12], alone)
        a, b = a + n, b + m
    few = max(range(seqs), key=lambda i: queries[i] if queries[i] < 300 else 0)
    a, b, n, m = sum(queries[:few]), sum(keys[:few]), queries[few], keys[few]
    check(out[a:a + n], None, q[a:a + n], k[b:b + m], v[b:b + m], [n], [m], causal, 1 / math.sqrt(dim))


@pytest.mark.parametrize("dim", [64, 128])
def test_many_blocks_captured_and_at_once(cuda, dim):
    """Each call takes on blocks of its own alone, in a graph and beside another call as well."""
    lengths = [300, 200, 1, 700, 64] * 4
    cases = [a_case(lengths, lengths, 24, 8, dim, torch.bfloat16, seed=i) for i in range(2)]
    at, op, graph = offsets(lengths), PromptAttention(), torch.cuda.CUDAGraph()
    want = [op(*c, at) for c in cases]
    with torch.cuda.graph(graph):
        captured = op(*cases[0], at)
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for i in range(12):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(op(*cases[i % 2], at))
        if i % 4 == 3:
            graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i % 2]) for i, o in enumerate(outs)) and torch.equal(captured, want[0])


def test_waits_that_run_out_of_many_blocks(cuda):
    lib = _lib.load()
    q, k, v = a_case([200] * 30, [200] * 30, 24, 8, 64, torch.bfloat16)
    at, op = offsets([200] * 30), PromptAttention()
    want = op(q, k, v, at)
    assert lib.qfg_prompt_attention_set_option(b"give_up", b"1") == 0
    try:
        got, lse = op(q, k, v, at, lse=True)
        torch.cuda.synchronize()
    finally:
        assert lib.qfg_prompt_attention_set_option(b"give_up", b"0") == 0
    assert torch.isnan(got.float()).all() and torch.isnan(lse).all()
    assert torch.equal(op(q, k, v, at), want)


def test_waits_that_run_out(cuda):
    """No operand comes: the block's waits end, its rows are NaN, and the next call is whole."""
    lib = _lib.load()
    for dim in (64, 128):
        q, k, v = a_case([200], [200], 2, 1, dim, torch.bfloat16)
        at, op = offsets([200]), PromptAttention()
        want = op(q, k, v, at)
        assert lib.qfg_prompt_attention_set_option(b"give_up", b"1") == 0
        try:
            got, lse = op(q, k, v, at, lse=True)
            torch.cuda.synchronize()
        finally:
            assert lib.qfg_prompt_attention_set_option(b"give_up", b"0") == 0
        assert torch.isnan(got.float()).all() and torch.isnan(lse).all()
        assert torch.equal(op(q, k, v, at), want)


def test_calls_that_are_refused(cuda):
    q, k, v = a_case([200], [200], 4, 2, 64, torch.bfloat16)
    at, op = offsets([200]), PromptAttention()
    wide = torch.zeros(200, 4 * 256, device="cuda").bfloat16()
    for call, message in ((lambda: op(q.float(), k, v, at), "q must be bfloat16 / float16"), (lambda: op(q, k.half(), v, at), "k must be bfloat16"), (lambda: op(q, k, v[:, :1], at), "same tokens and heads"),
                          (lambda: op(q[:, :3], k, v, at), "multiple"), (lambda: op(q, k, v, at.long()), "q_offsets must be"), (lambda: op(q, k, v, at, at[:1]), "one offset more"),
                          (lambda: op(q, k, v, at[:0]), "one offset more"), (lambda: op(wide.view(200, 4, 256), wide.view(200, 4, 256), wide.view(200, 4, 256), at), "64 or 128"),
                          (lambda: op(wide[:, 1:257].unflatten(1, (4, 64)), k, v, at), "misaligned"), (lambda: op(q, k, v, at, out=q[:10]), "out must be"), (lambda: op(q.cpu(), k, v, at), "current CUDA")):
        with pytest.raises(QfgError, match=message):
            call()
