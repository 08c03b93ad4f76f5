"""QkNormRope: forms of its arguments that the documentation allows."""
import pytest
import torch

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
