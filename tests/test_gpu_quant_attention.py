"""The operators of an attention block as they are used together: a prompt, then steps over its cache, against the block's formula in 64 bits."""
import pytest
import torch

from _attention import FORMS, attention, held
from qwen38_flash_ops_b200 import CacheAttention, CacheRead, KvCache, PromptAttention, QkNormRope, QuantAttention, QuantGemm, RmsNormQuant, RowQuant
from qwen38_flash_ops_b200.packing_torch import quantize_int8_per_column_torch

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, DIM, PAGE = 256, 6, 2, 64, 32


def a_block(form, gen):
    randn = lambda *s: torch.randn(*s, generator=gen)
    (q1, s1), (q2, s2) = quantize_int8_per_column_torch(randn(HIDDEN, (HEADS + 2 * KV) * DIM).cuda() * 0.06), quantize_int8_per_column_torch(randn(HEADS * DIM, HIDDEN).cuda() * 0.05)
    norm, qw, kw = ((1 + 0.2 * randn(n)).bfloat16().cuda() for n in (HIDDEN, DIM, DIM))
    cache = KvCache(20, KV, DIM, PAGE, FORMS[form], k_unit=0.01, v_unit=0.01)
    block = QuantAttention(norm, q1, s1.cpu().numpy(), q2, s2.cpu().numpy(), HEADS, KV, QkNormRope(DIM, rotary_dim=32), cache, qw, kw)
    return block, (norm, q1, s1, q2, s2, qw, kw)


@pytest.mark.parametrize("form", FORMS)
def test_a_prompt_and_steps(cuda, form):
    gen = torch.Generator().manual_seed(1)
    block, (norm, q1, s1, q2, s2, qw, kw) = a_block(form, gen)
    lengths = [75, 130]
    table = torch.randperm(20, generator=gen).view(2, 10).int().cuda()
    seq = torch.repeat_interleave(torch.arange(2), torch.tensor(lengths)).cuda()
    at = torch.cat([torch.arange(n) for n in lengths]).cuda()
    slots = lambda seq, at: table[seq, at // PAGE].long() * PAGE + at % PAGE
    x, r = (torch.randn(sum(lengths), HIDDEN, generator=gen).bfloat16().cuda() for _ in range(2))
    offsets = torch.tensor([0, 75, 205], dtype=torch.int32).cuda()
    y, h = block(x, r, at, slots(seq, at), offsets=offsets)
    assert torch.equal(h, x + r)
    # the same operators, one by one
    rows8, scale, _ = RmsNormQuant()(x, norm, r)
    both = QuantGemm(w_scale=s1.cpu().numpy())(rows8, scale, q1).view(205, -1, DIM)
    rope = QkNormRope(DIM, rotary_dim=32)
    q, k = rope(both[:, :HEADS], both[:, HEADS:-KV], at, qw, kw)
    v = both[:, -KV:]
    mid = PromptAttention()(q, k, v, offsets)
    rows8, scale = RowQuant()(mid.view(205, -1))
    assert torch.equal(y, QuantGemm(w_scale=s2.cpu().numpy())(rows8, scale, q2))
    # what the cache gives back is what went in, to its type
    kc, vc = CacheRead()(block.cache, table, offsets, 205)
    room = 0.3 if form == "nvfp4" else 0.07  # of a block's largest: half of E2M1's widest step is a sixth; half of E4M3's a sixteenth
    for a, b in ((kc, k), (vc, v)):
        assert ((a.double() - b.double()).abs() <= room * b.double().abs().amax(-1, keepdim=True)).all()
    # three steps of two tokens each: attention over what the cache holds by then
    for step in range(3):
        n = torch.tensor([m + 2 * step + 2 for m in lengths], dtype=torch.int32).cuda()
        s2q = torch.arange(2).repeat_interleave(2).cuda()
        pos = (n.long()[:, None] - 2 + torch.arange(2).cuda()).flatten()
        x, r = (torch.randn(4, HIDDEN, generator=gen).bfloat16().cuda() for _ in range(2))
        y, h = block(x, r, pos, slots(s2q, pos), table=table, lengths=n)
        rows8, scale, _ = RmsNormQuant()(x, norm, r)
        both = QuantGemm(w_scale=s1.cpu().numpy())(rows8, scale, q1).view(4, -1, DIM)
        q, _ = rope(both[:, :HEADS], both[:, HEADS:-KV], pos, qw, kw)
        mid = CacheAttention()(q.view(2, 2, HEADS, DIM), block.cache, table, n)
        rows8, scale = RowQuant()(mid.view(4, -1))
        assert torch.equal(y, QuantGemm(w_scale=s2.cpu().numpy())(rows8, scale, q2))
        ks, vs = held(block.cache.k, block.cache.k_scale, 0.01), held(block.cache.v, block.cache.v_scale, 0.01)
        for i in range(2):
            pages = table[i].cpu().long()
            for g in range(KV):
                ki, vi = (t[pages, g].flatten(0, 1)[:n[i]] for t in (ks, vs))
                rows = q.view(2, 2, HEADS, DIM)[i, :, g * 3:g * 3 + 3].cpu().double().flatten(0, 1)
                want, size, _ = attention(rows, ki, vi, (n[i].item() - 1 + torch.arange(2)).repeat_interleave(3), DIM ** -0.5)
                got = mid[i, :, g * 3:g * 3 + 3].cpu().double().flatten(0, 1)
                assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * size + 1e-5).all()


def test_a_step_in_a_graph(cuda):
    """A whole step, captured once and replayed as the sequences grow."""
    gen = torch.Generator().manual_seed(2)
    block, _ = a_block("nvfp4", gen)
    table = torch.arange(20).view(2, 10).int().cuda()
    x, r = (torch.randn(2, HIDDEN, generator=gen).bfloat16().cuda() for _ in range(2))
    pos, n, slots = torch.zeros(2, dtype=torch.long).cuda(), torch.ones(2, dtype=torch.int32).cuda(), (torch.arange(2) * 320).cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h = block(x, r, pos, slots, table=table, lengths=n)
    for i in range(40):
        x.copy_(torch.randn(x.shape, generator=gen))
        graph.replay()
        got = y.clone()
        if i % 13 == 0:
            assert torch.equal(got, block(x, r, pos, slots, table=table, lengths=n)[0])
        pos.add_(1), n.add_(1), slots.add_(1)


def test_a_block_that_does_not_fit(cuda):
    gen = torch.Generator().manual_seed(3)
    block, (norm, q1, s1, q2, s2, qw, kw) = a_block("e4m3", gen)
    with pytest.raises(ValueError, match="qkv is"):
        QuantAttention(norm, q1, s1.cpu().numpy(), q2, s2.cpu().numpy(), HEADS, KV + 1, QkNormRope(DIM), block.cache)
    with pytest.raises(ValueError, match="offsets"):
        block(torch.zeros(1, HIDDEN).bfloat16().cuda(), None, None, None)
