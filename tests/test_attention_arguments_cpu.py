"""Arguments of heads, caches and attention that are of a wrong kind, without a GPU: refused with a reason, never taken for an address."""
import copy
import ctypes
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")

from qwen38_flash_ops_b200 import CacheRead, QfgError, attention, ops  # noqa: E402


@pytest.mark.parametrize("cache", [5, 4096, 1 << 62, -1, True, 3.0, "cache", None, object()], ids=lambda c: "object" if type(c) is object else str(c))
def test_what_is_no_cache(cache):
    """In a process of its own: an address that is read ends it."""
    table, offsets = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    if type(cache) is int:
        call = f"import torch; from qwen38_flash_ops_b200 import CacheRead; CacheRead()({cache}, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 4)"
        r = subprocess.run([sys.executable, "-c", call], capture_output=True, text=True, timeout=300)
        assert r.returncode == 1 and "CacheRead: the cache must be a KvCache" in r.stderr, (r.returncode, r.stderr[-500:])
    with pytest.raises(QfgError, match="CacheRead: the cache must be a KvCache"):
        CacheRead()(cache, table, offsets, 4)


def test_other_capsules():
    if not hasattr(ops._calls, "torch_version"):
        pytest.skip("the calls in C++ are not built")
    room = ctypes.create_string_buffer(256)
    for name in (b"qfg_kv_caches", None):
        assert ops._calls.cache_read(10, attention._new_capsule(ctypes.addressof(room), name, None), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 4) is None


def test_a_cache_is_not_copied_by_its_addresses():
    """A deep copy of a KvCache would hold other tensors and the first one's addresses."""
    cache = attention.KvCache.__new__(attention.KvCache)
    cache._capsule = attention._new_capsule(1 << 20, attention._CAPSULE, None)
    with pytest.raises(TypeError):
        copy.deepcopy(cache)
