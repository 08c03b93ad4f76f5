"""PromptAttention of values that are no numbers, that are as large as their type has them, or whose weights are tiny."""
import math

import pytest
import torch

from _attention import attention, half_step
from qwen38_flash_ops_b200 import PromptAttention

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def offsets(*lengths):
    return torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32).cuda()


def a_case(n, heads, kv_heads, dim, dtype, seed=1):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(n, h, dim, generator=gen).to(dtype).cuda() for h in (heads, kv_heads, kv_heads)]


def alike(got, want, v):
    """The same rows, but that the rows of a warp take up their maxima together, so that weights may be rounded at other points."""
    bound = 2 * half_step(got.dtype) * (want.abs() + v[torch.isfinite(v)].abs().amax()).double()
    return torch.isfinite(got).all() and ((got.double() - want.double()).abs() <= bound).all()


@pytest.mark.parametrize("n", [1, 2, 3, 130])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_query_that_is_no_number(cuda, dtype, dim, causal, n):
    """Its row alone is NaN, however few keys it sees."""
    op = PromptAttention(causal=causal)
    for bad in (row for row in (0, 1, 2, 64, 129) if row < n):
        q, k, v = a_case(n, 2, 1, dim, dtype)
        want, log = op(q, k, v, offsets(n), lse=True)
        q[bad, 1, 3] = NAN
        got, also = op(q, k, v, offsets(n), lse=True)
        assert torch.isnan(got[bad, 1].float()).all() and torch.isnan(also[bad, 1]), (bad, got[bad, 1], also[bad, 1])
        got[bad, 1], also[bad, 1] = want[bad, 1], log[bad, 1]
        assert alike(got, want, v) and torch.allclose(also, log, atol=1e-3)


@pytest.mark.parametrize("value", [NAN, INF])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_key_that_is_no_number(cuda, dtype, dim, causal, value):
    """At every place of a tile's eight, of the first tile and of a later one: the rows that see it are NaN, the others as they were."""
    n, op = 200, PromptAttention(causal=causal)
    for key in (*range(16), *range(136, 144)):
        q, k, v = a_case(n, 2, 1, dim, dtype)
        q[:, :, 5] = 1.0  # a score of infinity, not of its negative
        want, log = op(q, k, v, offsets(n), lse=True)
        k[key, 0, 5] = value
        got, also = op(q, k, v, offsets(n), lse=True)
        first = key if causal else 0
        assert torch.isnan(got[first:].float()).all() and torch.isnan(also[first:]).all(), (key, torch.isfinite(got.float()).all(-1).nonzero().tolist()[:4])
        assert alike(got[:first], want[:first], v) and torch.isfinite(also[:first]).all()


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_masked_values_may_be_as_large_as_there_are(cuda, dtype, dim, sign):
    """The type's largest and lowest value in keys and values of a token that causal rows do not see yet: those rows are as they were, to the bit where they see one key."""
    n, op = 200, PromptAttention()
    for token in (*range(1, 17), *range(136, 144)):
        q, k, v = a_case(n, 2, 1, dim, dtype)
        want = op(q, k, v, offsets(n))
        v[token] = sign * torch.finfo(dtype).max
        got = op(q, k, v, offsets(n))
        assert torch.equal(got[0], want[0]) and alike(got[:token], want[:token], v[:token]), (token, (got[:token].float() - want[:token].float()).abs().max())


def test_rows_that_see_nothing_beside_masked_values(cuda):
    """More queries than keys: the first ones see none, and are 0 whatever the keys' finite values are."""
    for dtype in (torch.bfloat16, torch.float16):
        q, k, v = a_case(90, 2, 1, 64, dtype)
        v[:] = torch.finfo(dtype).max
        got, lse = PromptAttention()(q, k[:40], v[:40], offsets(90), offsets(40), lse=True)
        assert (got[:50] == 0).all() and (lse[:50] == -math.inf).all() and torch.isfinite(lse[50:]).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_many_weights_that_are_tiny_beside_one(cuda, dim):
    """A first key whose score is 18 above those of 120000 others: each weighs 2^-26 of it and all of them a 500th, which is all there is, as the first value is 0."""
    count, gen = 120000, torch.Generator().manual_seed(1)
    q, k, v = torch.zeros(3, 2, dim), torch.zeros(count, 1, dim), 1 + 0.25 * torch.rand(count, 1, dim, generator=gen)
    q[..., 0], k[0, 0, 0], v[0] = 4.0, 4.5, 0.0
    got, lse = PromptAttention(scale=1.0, causal=False)(q.half().cuda(), k.half().cuda(), v.half().cuda(), offsets(3), offsets(count), lse=True)
    y, size, log = attention(q[0].half().double(), k[:, 0].half().double(), v[:, 0].half().double(), torch.tensor([count, count]), 1.0)
    # A weight is off by 2^-11 of itself and, below 2^-14, by 2^-25 where the largest is 2^7 or more.  A quarter of a row's weights are added one after another in FP32, each sum
    # off by up to 2^-24 of itself; the products, sixteen keys at a time, are cut off at up to 2^-23.
    sums = count / 4 * 2.0 ** -24
    tol = (half_step(torch.float16) + sums + count / 16 * 2.0 ** -23) * y.abs() + (2.0 ** -11 + 1e-5) * size + count * 2.0 ** -32 * v.abs().amax() + 2.0 ** -25
    assert ((got.cpu().double() - y).abs() <= tol).all(), ((got.cpu().double() - y).abs() / tol).max()
    assert ((lse.cpu().double() - log).abs() <= 2.0 ** -18 * (1 + log) + sums).all()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scores_past_what_fp32_tells_apart(cuda, dtype, dim, causal):
    """Scores of 2^20 to 2^140: a row is that of its largest score, or NaN, never one that saw nothing."""
    n, op = 40, PromptAttention(scale=2.0 ** 10 * 1.1, causal=causal)
    for power in ((0, 5, 7) if dtype == torch.float16 else range(0, 64, 3)):
        q, k, v = a_case(n, 2, 1, dim, dtype, seed=power)
        q, k = q * 2.0 ** power, k * 2.0 ** power
        got, lse = op(q, k, v, offsets(n), lse=True)
        bad = torch.isnan(got.float()).any(-1)
        s = torch.einsum("ihd,jd->ihj", q.cpu().double(), k[:, 0].cpu().double()) * (2.0 ** 10 * 1.1)
        if causal:
            s.masked_fill_(torch.arange(n)[None, None] > torch.arange(n)[:, None, None], -INF)
        top = s.topk(2).values
        sure = (~bad.cpu()) & (top[..., 0] - top[..., 1] > 2.0 ** -17 * s[torch.isfinite(s)].abs().amax() + 50)  # FP32 sums tell the largest from the next, by far
        sure[0] = ~bad[0].cpu()
        want = v[:, 0].cpu().double()[s.argmax(-1)]
        assert ((got.cpu().double() - want).abs()[sure] <= 2.0 ** -7 * want.abs()[sure]).all(), power
        assert (torch.isnan(lse) == bad).all() and torch.isfinite(lse[~bad]).all()
        assert power > 0 or not bad.any()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_that_see_nothing_beside_values_that_are_no_numbers(cuda, dtype, dim, causal):
    """More queries than keys: the first ones see none, and are 0 whatever the keys and values are; not causal, only those of a sequence without keys."""
    for value in (NAN, INF):
        q, k, v = a_case(90, 2, 1, dim, dtype)
        k[:], v[:] = value, value
        at = torch.tensor([0, 10, 90], dtype=torch.int32).cuda()
        got, lse = PromptAttention(causal=causal)(q, k[:30], v[:30], at, torch.tensor([0, 0, 30], dtype=torch.int32).cuda(), lse=True)
        none = 60 if causal else 10
        assert (got[:none] == 0).all() and (lse[:none] == -math.inf).all()
        assert torch.isnan(got[none:].float()).all() and torch.isnan(lse[none:]).all()
