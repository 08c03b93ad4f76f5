"""Arguments of a wrong kind among tensors that are right: every call refuses them with a reason."""
import pytest
import torch

from _attention import new_cache
from qwen38_flash_ops_b200 import CacheAttention, CacheRead, CacheWrite, KvCache, QfgError, QkNormRope

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", [0, 5, 4096, 1 << 62, -1, True, 1.5, "cache", object()], ids=lambda c: "object" if type(c) is object else str(c))
def test_what_is_no_cache(cuda, cache):
    x = torch.zeros(4, 2, 64, device="cuda").bfloat16()
    at, slots, table, n = torch.arange(4).cuda(), torch.arange(4).cuda(), torch.zeros(4, 1, dtype=torch.int32).cuda(), torch.ones(4, dtype=torch.int32).cuda()
    rope = QkNormRope(64)
    for call in (lambda: rope(x, x, at, v=x, cache=cache, slots=slots), lambda: rope(x, x, at, cache=cache), lambda: CacheWrite()(x, x, cache, slots),
                 lambda: CacheRead()(cache, table, torch.arange(5).int().cuda(), 4), lambda: CacheAttention()(x, cache, table, n), lambda: CacheAttention()(x, cache, table, n, lse=True)):
        with pytest.raises(QfgError, match="the cache must be a KvCache"):
            call()


def test_a_kind_of_kv_cache(cuda):
    """A class made of KvCache goes the same way."""
    class Named(KvCache):
        pass

    x, slots, table, n = torch.randn(3, 2, 64).bfloat16().cuda(), torch.arange(3).cuda(), torch.zeros(3, 1, dtype=torch.int32).cuda(), torch.ones(3, dtype=torch.int32).cuda() * 3
    a, b = new_cache("e4m3", 1, 2, 64), Named(1, 2, 64, 32, torch.float8_e4m3fn)
    for cache in (a, b):
        CacheWrite()(x, x, cache, slots)
    assert torch.equal(CacheAttention()(x, a, table, n), CacheAttention()(x, b, table, n))
