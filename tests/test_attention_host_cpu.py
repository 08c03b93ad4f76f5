"""Heads, their cache and attention without a GPU: what is refused is refused before any CUDA call, and with a reason."""
import ctypes

import pytest

from qwen38_flash_ops_b200 import _lib

P = 1 << 20  # an address nothing reads
NAN, INF = float("nan"), float("inf")


class Cache(ctypes.Structure):  # qfg_kv_cache
    _fields_ = [("k", ctypes.c_void_p), ("k_scale", ctypes.c_void_p), ("v", ctypes.c_void_p), ("v_scale", ctypes.c_void_p), ("dtype", ctypes.c_int32),
                ("pages", ctypes.c_int64), ("kv_heads", ctypes.c_int64), ("page", ctypes.c_int64), ("head_dim", ctypes.c_int64), ("k_unit", ctypes.c_float),
                ("v_unit", ctypes.c_float)]


def cache(**other):
    c = Cache(P, P, P, P, _lib.QFG_UINT8, 10, 2, 64, 128, 1.0, 1.0)
    for name, value in other.items():
        setattr(c, name, value)
    return c


BAD_CACHES = [({"k": None}, "null cache"), ({"v_scale": P + 8}, "must begin on 16 bytes"), ({"dtype": _lib.QFG_INT8}, "a cache holds"), ({"pages": 0}, "at least one page"),
              ({"kv_heads": 0}, "at least one page"), ({"kv_heads": 5000}, "at least one page"), ({"page": 16}, "multiple of 32"), ({"page": 72}, "multiple of 32"),
              ({"page": 1 << 17}, "multiple of 32"), ({"head_dim": 96}, "64, 128 or 256"), ({"pages": 1 << 62}, "too large"), ({"pages": 1 << 31}, "at most 2147483647"),
              ({"k_unit": 0.0}, "units"), ({"v_unit": NAN}, "units"), ({"v_unit": 1e30}, "units"), ({"k_unit": -1.0}, "units")]


def refused(code, message):
    lib = _lib.load()
    assert code == _lib.QFG_INVALID_ARGUMENT, code
    assert message in lib.qfg_last_error().decode(), lib.qfg_last_error().decode()


def write(c, dtype=_lib.QFG_BFLOAT16, k=P, ldk=256, v=P, ldv=256, tokens=3, slots=P):
    return _lib.load().qfg_cache_write(dtype, k, ldk, v, ldv, tokens, ctypes.byref(c) if c else None, slots, None)


def read(c, table=P, ldt=4, seqs=2, most=4, offsets=P, rows=5, dtype=_lib.QFG_BFLOAT16, k=P, v=P):
    return _lib.load().qfg_cache_read(ctypes.byref(c), table, ldt, seqs, most, offsets, rows, dtype, k, v, None)


def attend(c, dtype=_lib.QFG_BFLOAT16, q=P, ld_seq=1024, ld_token=1024, seqs=2, tokens=1, heads=8, table=P, ldt=40, most=40, lengths=P, scale=0.1, workspace=P, out=P,
           lse=None):
    return _lib.load().qfg_cache_attention(dtype, q, ld_seq, ld_token, seqs, tokens, heads, ctypes.byref(c), table, ldt, most, lengths, scale, workspace, out, lse, None)


def prompt(dtype=_lib.QFG_BFLOAT16, q=P, ldq=512, q_rows=9, heads=4, k=P, ldk=256, v=P, ldv=256, k_rows=9, kv_heads=2, dim=128, qo=P, ko=P, seqs=1, causal=1, scale=0.1,
           out=P, lse=None):
    return _lib.load().qfg_prompt_attention(dtype, q, ldq, q_rows, heads, k, ldk, v, ldv, k_rows, kv_heads, dim, qo, ko, seqs, causal, scale, out, lse, None)


@pytest.mark.parametrize("other,message", BAD_CACHES)
def test_caches_that_are_refused(other, message):
    refused(write(cache(**other)), "CacheWrite: ")
    refused(read(cache(**other)), message)
    refused(attend(cache(**other)), message)
    need = ctypes.c_size_t(7)
    refused(_lib.load().qfg_cache_attention_workspace_bytes(ctypes.byref(cache(**other)), 1, 1, 8, 4, ctypes.byref(need)), message)
    assert need.value == 0


@pytest.mark.parametrize("call,message", [
    (lambda: write(None), "null cache"), (lambda: write(cache(), dtype=_lib.QFG_INT8), "BF16/FP16/FP32"), (lambda: write(cache(), k=None), "null k"),
    (lambda: write(cache(), ldv=255), "overlap"), (lambda: write(cache(), v=P + 1), "misaligned"), (lambda: write(cache(), tokens=-1), "number of tokens"),
    (lambda: write(cache(), slots=None), "no slots"), (lambda: write(cache(), slots=P + 4), "no slots"),
    (lambda: read(cache(), dtype=_lib.QFG_UINT8), "BF16/FP16/FP32"), (lambda: read(cache(), table=None), "no table"), (lambda: read(cache(), ldt=3), "overlap"),
    (lambda: read(cache(), seqs=70000), "65536"), (lambda: read(cache(), most=1 << 26, ldt=1 << 26), "2147483647 tokens"), (lambda: read(cache(), rows=-1), "number of rows"),
    (lambda: read(cache(), offsets=None), "no offsets"), (lambda: read(cache(), v=P + 2), "16 bytes"),
    (lambda: attend(cache(), dtype=_lib.QFG_FLOAT), "BF16/FP16"), (lambda: attend(cache(), heads=7), "multiple of the cache's"), (lambda: attend(cache(), heads=0), "multiple"),
    (lambda: attend(cache(), tokens=1025), "1024 tokens"), (lambda: attend(cache(), q=P + 8), "16 bytes"), (lambda: attend(cache(), ld_seq=1028), "16 bytes"),
    (lambda: attend(cache(), ld_seq=512), "overlap"), (lambda: attend(cache(), tokens=2, ld_token=512, ld_seq=4096), "overlap"), (lambda: attend(cache(), scale=0.0), "scale"),
    (lambda: attend(cache(), scale=NAN), "scale"), (lambda: attend(cache(), scale=INF), "scale"), (lambda: attend(cache(), scale=-1.0), "scale"),
    (lambda: attend(cache(), lengths=None), "null or misaligned"), (lambda: attend(cache(), out=None), "null or misaligned"), (lambda: attend(cache(), lse=P + 2), "null or misaligned"),
    (lambda: attend(cache(), most=1 << 26, ldt=1 << 26), "2147483647 tokens"), (lambda: attend(cache(), seqs=60000, most=1 << 16, ldt=1 << 16), "too large"),
    (lambda: attend(cache(kv_heads=2000), heads=4000, ld_seq=1 << 30, ld_token=1 << 20, tokens=1024, seqs=16, most=1 << 20, ldt=1 << 20), "too large"),
    (lambda: prompt(dtype=_lib.QFG_FLOAT), "BF16/FP16"), (lambda: prompt(dim=256), "64 or 128"), (lambda: prompt(heads=3), "multiple of the key heads"),
    (lambda: prompt(kv_heads=0), "multiple of the key heads"), (lambda: prompt(seqs=-1), "65536"), (lambda: prompt(q_rows=-1), "number of rows"),
    (lambda: prompt(q=P + 8), "misaligned"), (lambda: prompt(ldq=516), "16 bytes"), (lambda: prompt(ldk=128), "overlap"), (lambda: prompt(v=None), "null v"),
    (lambda: prompt(qo=None), "no offsets"), (lambda: prompt(ko=P + 1), "no offsets"), (lambda: prompt(out=P + 8), "16 bytes"), (lambda: prompt(scale=0.0), "scale"),
])
def test_calls_that_are_refused(call, message):
    refused(call(), message)


def test_options():
    lib = _lib.load()
    refused(lib.qfg_prompt_attention_set_option(b"give_ups", b"1"), "unknown option give_ups")
    refused(lib.qfg_prompt_attention_set_option(None, b"1"), "null argument")
    assert lib.qfg_prompt_attention_set_option(b"give_up", b"0") == _lib.QFG_OK


def test_calls_of_nothing_are_no_calls():
    assert write(cache(), tokens=0, k=None, v=None, slots=None) == 0
    assert read(cache(), rows=0) == 0 and read(cache(), seqs=0, table=None) == 0
    assert attend(cache(), seqs=0, q=None, out=None) == 0 and attend(cache(), tokens=0) == 0
    assert prompt(q_rows=0, q=None) == 0 and prompt(seqs=0) == 0


@pytest.mark.parametrize("freq,axis,pairs,dim,eps,scale,message", [
    ([1.0] * 16, None, 16, 100, 0.0, 1.0, "64, 128 or 256"), ([1.0] * 17, None, 17, 128, 0.0, 1.0, "multiple of 32"), ([1.0] * 48, None, 48, 64, 0.0, 1.0, "multiple of 32"),
    (None, None, 16, 64, 0.0, 1.0, "null frequencies"), ([1.0] * 16, None, 16, 64, -1.0, 1.0, "eps"), ([1.0] * 16, None, 16, 64, 0.0, NAN, "finite"),
    ([INF] * 16, None, 16, 64, 0.0, 1.0, "frequencies must be finite"), ([1.0] * 16, [8] * 16, 16, 64, 0.0, 1.0, "axis"), ([1.0] * 16, [-1] * 16, 16, 64, 0.0, 1.0, "axis"),
])
def test_rotations_that_are_refused(freq, axis, pairs, dim, eps, scale, message):
    lib, h = _lib.load(), ctypes.c_void_p(5)
    f = (ctypes.c_double * len(freq))(*freq) if freq else None
    a = (ctypes.c_int32 * len(axis))(*axis) if axis else None
    refused(lib.qfg_qk_norm_rope_create(f, a, pairs, dim, 0, scale, eps, 0.0, ctypes.byref(h)), message)
    assert not h.value
    refused(lib.qfg_qk_norm_rope_create(f, a, pairs, dim, 0, scale, eps, 0.0, None), "null handle")
    refused(lib.qfg_qk_norm_rope_compute(None, *[0] * 2, *[0] * 20, None), "null node")


def test_python_refuses_on_the_host():
    torch = pytest.importorskip("torch")
    from qwen38_flash_ops_b200 import CacheAttention, CacheRead, KvCache, PromptAttention, QkNormRope, QfgError

    with pytest.raises(QfgError, match="contiguous CUDA tensors"):
        KvCache.of(torch.zeros(2, 1, 32, 64, dtype=torch.uint8), torch.zeros(1), torch.zeros(1), torch.zeros(1))
    for make, message in ((lambda: KvCache(1, 1, 128, dtype=torch.int8), "torch.uint8"), (lambda: KvCache(1, 1, 100), "64, 128 or 256"), (lambda: KvCache(1, 1, 64, page=40), "32"),
                          (lambda: QkNormRope(128, rotary_dim=48), "multiple of 32"), (lambda: QkNormRope(128, base=-1.0), "base"),
                          (lambda: QkNormRope(128, inv_freq=[1.0]), "frequency"), (lambda: QkNormRope(128, sections=[64], axes=[0] * 64), "sections or axes"),
                          (lambda: QkNormRope(128, sections=[10, 10]), "frequency and an axis"), (lambda: CacheRead(dtype=torch.int8), "dtype"),
                          (lambda: CacheAttention(scale=0), "scale"), (lambda: PromptAttention(scale=float("nan")), "scale")):
        with pytest.raises(QfgError, match=message):
            make()
