"""QkNormRope: forms of its arguments that the documentation allows."""
import pytest
import torch

from _attention import FORMS, held, new_cache
from qwen38_flash_ops_b200 import QfgError, QkNormRope

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [5, 300])
@pytest.mark.parametrize("sections", [(32, 32, 0), (64, 0, 0), (0, 64, 0), (16, 0, 48, 0)], ids=str)
def test_sections_without_pairs(cuda, sections, tokens):
    """An axis by which no pair goes has a row of positions all the same, the last ones too."""
    gen = torch.Generator().manual_seed(1)
    q, k = (torch.randn(tokens, h, 128, generator=gen).bfloat16().cuda() for h in (4, 2))
    positions = torch.randint(0, 1 << 20, (len(sections), tokens), generator=gen).cuda()
    op = QkNormRope(128, sections=sections)
    assert op.axes == len(sections)
    got = op(q, k, positions)
    used = [a for a, n in enumerate(sections) if n]
    same = QkNormRope(128, axes=[i for i, a in enumerate(used) for _ in range(sections[a])])
    want = same(q, k, positions[used].contiguous())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    wide = torch.zeros(len(sections), tokens + 3, dtype=torch.int64).cuda()
    wide[:, :tokens] = positions
    assert all(torch.equal(a, b) for a, b in zip(op(q, k, wide[:, :tokens]), want))
    for bad in (positions[0], positions[:len(sections) - 1], positions[:, 1:], None):
        with pytest.raises(QfgError, match="positions"):
            op(q, k, bad)


@pytest.mark.parametrize("tokens", [3, 400])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_whose_squares_fp32_does_not_hold(cuda, dtype, dim, tokens):
    """They are NaN, in the outputs and in a cache, and alone; as large as their squares allow rows are as they should be."""
    gen = torch.Generator().manual_seed(3)
    w = (1 + 0.3 * torch.randn(dim, generator=gen)).cuda()
    op, slots, at = QkNormRope(dim, eps=0.0), torch.arange(tokens).cuda(), torch.arange(tokens).cuda()
    x = (torch.rand(tokens, 4, dim, generator=gen) - 0.5).to(dtype)
    x[2] *= 2.0 ** 58  # sums of squares up to 2^124
    x[1, 1, 5], x[1, 2], x[1, 3, 0] = 2.0 ** 64, 2.0 ** 63 * (1 + x[1, 2]), torch.finfo(dtype).max
    bad = torch.zeros(tokens, 4, dtype=torch.bool)
    bad[1, 1:] = True
    for form in FORMS:
        cache = new_cache(form, -(-tokens // 32), 4, dim)
        q, k = op(x.cuda(), x.cuda(), at, w, w, x.cuda(), cache, slots, True)
        held_k = held(cache.k, cache.k_scale, cache.k_unit).transpose(1, 2).flatten(0, 1)[:tokens]
        for got in (q.cpu(), k.cpu(), held_k):
            assert torch.isnan(got[bad]).all() and torch.isfinite(got[~bad]).all()
    y = x.double()
    want = y / (y * y).mean(-1, keepdim=True).sqrt() * w.cpu().double()
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -19 * want.abs().amax(-1, keepdim=True)
    got = QkNormRope(dim, rotary_dim=0, eps=0.0)(x.cuda(), x.cuda(), None, w, w)[0].cpu().double()
    assert ((got - want).abs() <= tol)[~bad].all()
