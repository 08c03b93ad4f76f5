"""CacheRead of offsets that no program should have: rows that they put past a table's width are zeros, wherever that is."""
import pytest
import torch

from _attention import FORMS, fill, held, new_cache
from qwen38_flash_ops_b200 import CacheRead

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("offsets", [(-(1 << 31), 40, 60), (-(1 << 31), -(1 << 31), 60), (1 - (1 << 31), 0, (1 << 31) - 1), (-64, 0, 60), (-(1 << 30), 30, 30), (-1, 5, (1 << 31) - 1)], ids=str)
@pytest.mark.parametrize("form", FORMS)
def test_offsets_far_below_zero(cuda, form, offsets):
    rows, page = 60, 32
    cache = new_cache(form, 5, 2, 64, page)
    fill(cache, torch.Generator().manual_seed(1))
    table = torch.tensor([[3, 1], [0, 4]], dtype=torch.int32).cuda()
    out = [torch.full((rows, 2, 64), 7.0, device="cuda") for _ in range(2)]
    CacheRead(torch.float32)(cache, table, torch.tensor(offsets, dtype=torch.int32).cuda(), rows, out=out)
    for got, codes, scale, unit in ((out[0], cache.k, cache.k_scale, cache.k_unit), (out[1], cache.v, cache.v_scale, cache.v_unit)):
        pages = held(codes, scale, unit).transpose(1, 2)
        for row in range(rows):
            seqs = [i for i in range(2) if offsets[i] <= row < offsets[i + 1]]
            if not seqs:
                want = torch.full((2, 64), 7.0)
            else:
                at = row - offsets[seqs[0]]
                want = pages[table[seqs[0], at // page].item(), at % page].float() if at < 2 * page else torch.zeros(2, 64)
            assert torch.equal(got[row].cpu(), want), row
