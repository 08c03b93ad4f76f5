"""PromptAttention of offsets that fall, leave the tensors or leave rows out: nothing is written but rows of its sequences, and sequences whose offsets hold are as ever."""
import pytest
import torch

from qwen38_flash_ops_b200 import PromptAttention

pytestmark = pytest.mark.gpu
ROWS, GUARD, MARK = 200, 300, 7.0


def whole(*v):
    return torch.tensor(v, dtype=torch.int32).cuda()


@pytest.mark.parametrize("qo,ko", [((0, 100, 50, 200), (0, 100, 50, 200)), ((-5, 90, 1000, 2000), (-5, 90, 1000, 2000)), ((0, 200, 200, 200), (150, 400, 3, -9)),
                                   ((60, 80, 80, 130), (60, 80, 80, 130)), ((200, 100, 0, -100), (0, 50, 100, 150)), ((1 << 30, 0, 64, 1 << 30), (0, 0, 64, 64)),
                                   ((-(1 << 31), -1, 64, (1 << 31) - 1), (0, 0, 64, (1 << 31) - 1)), ((10, 10, 10, 10), (0, 200, 200, 200))], ids=str)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", [64, 128])
def test_rows_of_no_sequence_are_left(cuda, dim, causal, qo, ko):
    gen = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(ROWS, h, dim, generator=gen).bfloat16().cuda() for h in (2, 1, 1))
    wide = torch.full((ROWS + 2 * GUARD, 2, dim), MARK, device="cuda").bfloat16()
    out, op = wide[GUARD:-GUARD], PromptAttention(causal=causal)
    op(q, k, v, whole(*qo), whole(*ko), out=out)
    torch.cuda.synchronize()
    assert (wide[:GUARD] == MARK).all() and (wide[-GUARD:] == MARK).all()
    inside = lambda n: min(max(n, 0), ROWS)
    spans = [(inside(a), inside(b)) for a, b in zip(qo, qo[1:])]
    of_some = torch.zeros(ROWS, dtype=torch.bool)
    for a, b in spans:
        of_some[a:b] = True
    assert (out[~of_some.cuda()] == MARK).all()
    for i, (a, b) in enumerate(spans):
        others = [s for j, s in enumerate(spans) if j != i and s[0] < s[1]]
        if a < b and not any(c < b and a < d for c, d in others):  # rows of this sequence alone
            c, d = inside(ko[i]), max(inside(ko[i]), inside(ko[i + 1]))
            alone = op(q[a:b], k[c:d], v[c:d], whole(0, b - a), whole(0, d - c))
            assert torch.equal(out[a:b], alone), i
