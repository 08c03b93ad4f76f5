"""QuantAttention: what it refuses it refuses before anything is written, and calls of nothing are calls."""
import pytest
import torch

from _attention import FORMS, same_bits
from qwen38_flash_ops_b200 import KvCache, QfgError, QkNormRope, QuantAttention
from qwen38_flash_ops_b200.packing_torch import quantize_int8_per_column_torch

pytestmark = pytest.mark.gpu
HIDDEN, HEADS, KV, PAGE = 256, 4, 2, 32


def a_block(dim, form="e4m3"):
    gen = torch.Generator().manual_seed(1)
    (q1, s1), (q2, s2) = (quantize_int8_per_column_torch(torch.randn(*s, generator=gen).cuda() * 0.06) for s in ((HIDDEN, (HEADS + 2 * KV) * dim), (HEADS * dim, HIDDEN)))
    cache = KvCache(8, KV, dim, PAGE, FORMS[form])
    return QuantAttention(torch.ones(HIDDEN).bfloat16().cuda(), q1, s1.cpu().numpy(), q2, s2.cpu().numpy(), HEADS, KV, QkNormRope(dim), cache)


def whole(*v):
    return torch.tensor(v, dtype=torch.int32).cuda()


def inputs(rows):
    gen = torch.Generator().manual_seed(2)
    x, r = (torch.randn(rows, HIDDEN, generator=gen).bfloat16().cuda() for _ in range(2))
    return x, r, torch.arange(rows).cuda(), torch.arange(rows).cuda()


def held(cache):
    return [t.clone() for t in (cache.k, cache.k_scale, cache.v, cache.v_scale)]


@pytest.mark.parametrize("form", FORMS)
def test_a_refused_call_writes_nothing(cuda, form):
    table = torch.arange(8).int().view(2, 4).cuda()
    for dim, given in ((256, {"offsets": whole(0, 6)}), (64, {"offsets": whole(0, 6).long()}), (64, {"offsets": whole(0, 6).cpu()}), (64, {"offsets": whole(0, 6).view(1, 2)}),
                       (64, {"offsets": whole()}), (64, {"table": table}), (64, {"lengths": whole(3, 3)}), (64, {"table": table, "lengths": whole(3)}),
                       (64, {"table": table, "lengths": whole(3, 3).long()}), (64, {"table": table.long(), "lengths": whole(3, 3)}), (64, {"table": table[0], "lengths": whole(3, 3)}),
                       (64, {"table": table[:, ::2], "lengths": whole(3, 3)}), (64, {"table": table.repeat(2, 1), "lengths": whole(3, 3, 3, 3)}),
                       (64, {"table": table[:0], "lengths": whole()}), (64, {"table": table, "lengths": whole(3, 3), "offsets": whole(0, 6)}), (64, {"offsets": whole(0, 6), "lengths": whole(3, 3)})):
        block = a_block(dim, form)
        before = held(block.cache)
        with pytest.raises((ValueError, QfgError), match="QuantAttention"):
            block(*inputs(6), **given)
        torch.cuda.synchronize()
        assert all(same_bits(a, b) for a, b in zip(before, held(block.cache))), given
    block = a_block(64, form)
    before = held(block.cache)
    with pytest.raises(QfgError, match="at most 1024 tokens"):
        block(*inputs(2050), table=table, lengths=whole(3, 3))
    torch.cuda.synchronize()
    assert all(same_bits(a, b) for a, b in zip(before, held(block.cache)))


def test_steps_over_heads_of_256(cuda):
    block = a_block(256)
    y, h = block(*inputs(6), table=torch.arange(8).int().view(2, 4).cuda(), lengths=whole(3, 3))
    assert torch.isfinite(y).all() and y.shape == h.shape == (6, HIDDEN)


@pytest.mark.parametrize("given", [{"offsets": (0, 0)}, {"offsets": (0,)}, {"table": 0, "lengths": ()}, {"table": 2, "lengths": (3, 3)}], ids=str)
def test_no_rows(cuda, given):
    block = a_block(64)
    before = held(block.cache)
    given = {k: whole(*v) if k != "table" else torch.zeros(v, 4, dtype=torch.int32).cuda() for k, v in given.items()}
    y, h = block(*inputs(0), **given)
    assert y.shape == h.shape == (0, HIDDEN) and all(same_bits(a, b) for a, b in zip(before, held(block.cache)))


def test_rotations_and_caches_that_do_not_fit(cuda):
    block = a_block(64)
    with pytest.raises(ValueError, match="QuantAttention"):
        QuantAttention(block.norm_weight, block.qkv, None, block.out, None, HEADS, KV, QkNormRope(128), block.cache)
