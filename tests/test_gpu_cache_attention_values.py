"""CacheAttention of values and queries as large as their types have them, and of weights that are tiny."""
import math

import pytest
import torch

from _attention import FORMS, attention, half_step, held, new_cache
from qwen38_flash_ops_b200 import CacheAttention, CacheWrite
from test_gpu_cache_attention import a_case, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,group,tokens", [(64, 4, 1), (128, 8, 2), (256, 2, 1)])
@pytest.mark.parametrize("power", [40, 76, 90, 106, 112])
@pytest.mark.parametrize("some", [1, 7, 64])
def test_large_values(cuda, some, power, dim, group, tokens):
    """In eight bits, scales of every one, seventh or 64th token up to 2^107: values up to 2^115."""
    cache, table, q, n = a_case("e4m3", dim, 1, group, tokens, [300, 2000, 1], torch.bfloat16)
    flat = cache.v_scale.view(-1)
    flat[::some] = (flat[::some] * 2.0 ** power).clamp(max=2.0 ** 107)
    got, lse = CacheAttention()(q, cache, table, n, lse=True)
    check(got, lse, cache, table, q, n, 1 / math.sqrt(dim))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("power", [112, 122, 125])
def test_large_queries(cuda, form, power):
    """Queries up to BF16's largest exponent, with a scale that makes ordinary scores of them."""
    cache, table, q, n = a_case(form, 128, 2, 4, 2, [300, 65], torch.bfloat16)
    q[0] *= 2.0 ** power
    assert torch.isfinite(q).all()
    got, lse = CacheAttention(scale=2.0 ** -power)(q, cache, table, n, lse=True)
    check(got, lse, cache, table, q, n, 2.0 ** -power)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_many_weights_that_are_tiny_beside_one(cuda, dim, form):
    """A first token whose score is 18 above those of 120000 others: each weighs 2^-26 of it and all of them a 500th, which is all there is, as the first value is 0.  As many
    sequences, of the same pages, that a warp has a whole one to itself."""
    count, seqs, gen = 120000, 2400, torch.Generator().manual_seed(1)
    cache = new_cache(form, -(-count // 64), 1, dim, page=64)
    k, v = torch.zeros(count, 1, dim), 1 + 0.25 * torch.rand(count, 1, dim, generator=gen)
    k[0, 0, 0], v[0] = 4.5, 0.0
    CacheWrite()(k.half().cuda(), v.half().cuda(), cache, torch.arange(count).cuda())
    table, n = torch.arange(cache.pages).int().repeat(seqs, 1).cuda(), torch.full((seqs,), count, dtype=torch.int32).cuda()
    q = torch.zeros(seqs, 2, dim)
    q[..., 0] = 4.0
    got, lse = CacheAttention(scale=1.0)(q.half().cuda(), cache, table, n, lse=True)
    ki, vi = (held(c, s, u)[:, 0].flatten(0, 1)[:count] for c, s, u in ((cache.k, cache.k_scale, cache.k_unit), (cache.v, cache.v_scale, cache.v_unit)))
    y, size, log = attention(q[0].double(), ki, vi, torch.tensor([count, count]), 1.0)
    # A weight is off by 2^-11 of itself and, below 2^-14, by 2^-25 where the largest is 2^7 or more (in eight bits the zero row's scale of 2^-40 makes it small).  An eighth of a
    # row's weights are added one after another in FP32, each sum off by up to 2^-24 of itself; the products, sixteen tokens at a time, are cut off at up to 2^-23.
    tiny, sums = count * 2.0 ** -32 * vi.abs().amax(), count / 8 * 2.0 ** -24
    tol = (half_step(torch.float16) + sums + count / 16 * 2.0 ** -23) * y.abs() + 2.0 ** -11 * size + tiny + 2.0 ** -25
    assert ((got.cpu().double() - y).abs() <= tol).all(), ((got.cpu().double() - y).abs() / tol).max()
    assert ((lse.cpu().double() - log).abs() <= 2.0 ** -18 * (1 + log) + sums).all()


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_queries_that_are_no_numbers(cuda, form, dim, value):
    """Infinities as well, whose scores may all be -infinity: rows that see a key are NaN, those that see none 0, and others as they were."""
    for lengths in ([1, 0], [2, 1], [400, 33]):
        cache, table, q, n = a_case(form, dim, 1, 3, 2, lengths, torch.bfloat16)
        for c in (3, 7):  # keys of one sign in channel 3, of the other in channel 7
            cache.k.view(torch.uint8)[..., c if form == "e4m3" else c // 2] = 0x30 if c == 3 else 0xB0
        want, log = CacheAttention()(q, cache, table, n, lse=True)
        for c in (3, 7):
            bad = q.clone()
            bad[:, :, 1, c] = value
            got, lse = CacheAttention()(bad, cache, table, n, lse=True)
            for i, m in enumerate(lengths):
                for t in range(2):
                    sees = m - 1 + t > 0
                    if sees:
                        assert torch.isnan(got[i, t, 1].float()).all() and torch.isnan(lse[i, t, 1]), (lengths, c, i, t)
                    else:
                        assert (got[i, t] == 0).all() and (lse[i, t] == -math.inf).all()
            got[:, :, 1], lse[:, :, 1] = want[:, :, 1], log[:, :, 1]
            assert torch.isfinite(got).all() and ((got.double() - want.double()).abs() <= 2.0 ** -7 * want.double().abs() + 2.0 ** -9).all()
            assert torch.equal(lse == -math.inf, log == -math.inf) and torch.allclose(lse, log, atol=1e-3)


@pytest.mark.parametrize("dim,group,tokens", [(64, 4, 3), (128, 8, 3), (256, 2, 3)])
@pytest.mark.parametrize("form", FORMS)
def test_rows_that_see_nothing_beside_values_that_are_no_numbers(cuda, form, dim, group, tokens):
    """A padded place is 0, whatever the tokens hold that only later rows see."""
    lengths = [1, 2, 0, 3]
    cache, table, q, n = a_case(form, dim, 2, group, tokens, lengths, torch.bfloat16)
    want, log = CacheAttention()(q, cache, table, n, lse=True)
    if form == "e4m3":
        cache.v_scale.fill_(math.nan)
    else:
        cache.v_scale.view(torch.uint8).fill_(0x7F)
    got, lse = CacheAttention()(q, cache, table, n, lse=True)
    for i, m in enumerate(lengths):
        none = max(0, tokens - m)
        assert (got[i, :none] == 0).all() and (lse[i, :none] == -math.inf).all() and torch.isnan(got[i, none:].float()).all()
        assert torch.allclose(lse[i, none:], log[i, none:], atol=1e-4)
