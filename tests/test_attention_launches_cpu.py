"""The launches of heads, caches and attention, against a CUDA runtime that runs nothing (fake_cuda.c): every kernel that is built is one that some call launches, and
blocks and workspaces are as large as the calls need."""
import json
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)

SHIM = """
#include "fake_cuda.c"
API const char* fake_registered(int i) { return i < n_fn ? g_fn[i].name : 0; }
"""
BODY = """
import ctypes, importlib.util, json, os, re, sys
sys.path.insert(0, {here!r})
spec = importlib.util.spec_from_file_location("qfg_lib", os.path.join({root!r}, "qwen38_flash_ops_b200", "_lib.py"))
L = importlib.util.module_from_spec(spec)
spec.loader.exec_module(L)
lib, fake = L.load(), ctypes.CDLL({fake!r})
fake.fake_log.restype = fake.fake_registered.restype = ctypes.c_char_p
class Cache(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "k_scale", "v", "v_scale")] + [("dtype", ctypes.c_int32)] + [(n, ctypes.c_int64) for n in ("pages", "kv_heads", "page", "head_dim")] + [
        ("k_unit", ctypes.c_float), ("v_unit", ctypes.c_float)]
P = 1 << 20  # an address nothing reads
names = ("HeadsKernel", "CacheReadKernel", "CacheAttentionKernel", "JoinKernel", "PromptAttentionKernel")
built, i = set(), 0
while fake.fake_registered(i):
    name = fake.fake_registered(i).decode()
    built |= {{name}} if any(n in name for n in names) else set()
    i += 1
launched, failed, grids = set(), [], []
def run(call, what):
    fake.fake_clear()
    if call() != 0:
        failed.append([str(what), lib.qfg_last_error().decode()])
    lines = fake.fake_log().decode().splitlines()
    launched.update(l.split()[1] for l in lines)
    grids.append([str(what), lines])
for dim in (64, 128, 256):
    for form in (L.QFG_UINT8, L.QFG_FLOAT8E4M3FN):
        c = Cache(P, P, P, P, form, 100, 2, 64, dim, 1.0, 1.0)
        for dtype in (L.QFG_BFLOAT16, L.QFG_FLOAT16, L.QFG_FLOAT):
            run(lambda: lib.qfg_cache_read(ctypes.byref(c), P, 4, 2, 4, P, 50, dtype, P, P, None), ("read", dim, form, dtype))
            for base in (P, P + 4):
                for tokens in (1, 236, 237, 296, 297, 5000):
                    run(lambda: lib.qfg_cache_write(dtype, base, 2 * dim, base, 2 * dim, tokens, ctypes.byref(c), P, None), ("write", dim, form, dtype, base, tokens))
                    h = ctypes.c_void_p()
                    assert lib.qfg_qk_norm_rope_create((ctypes.c_double * 32)(*[0.5] * 32), None, 32, dim, 0, 1.0, 1e-6, 0.0, ctypes.byref(h)) == 0
                    run(lambda: lib.qfg_qk_norm_rope_compute(h, dtype, base, 40 * dim, 40, base, 2 * dim, 2, base, 2 * dim, P, 8, tokens, 1, P, P, dtype, tokens, P, None, ctypes.byref(c), P, None),
                        ("heads", dim, form, dtype, base, tokens))
                    lib.qfg_qk_norm_rope_destroy(h)
        for seqs, tokens, heads, most in ((1, 1, 2, 1), (1, 1, 16, 16), (3, 2, 16, 5), (64, 1, 16, 200), (1, 40, 6, 2000), (500, 1, 32, 3)):
            need = ctypes.c_size_t()
            assert lib.qfg_cache_attention_workspace_bytes(ctypes.byref(c), seqs, tokens, heads, most, ctypes.byref(need)) == 0
            ld = heads * dim
            run(lambda: lib.qfg_cache_attention(L.QFG_BFLOAT16, P, tokens * ld, ld, seqs, tokens, heads, ctypes.byref(c), P, most, most, P, 0.1, P, P, None, None),
                ("attend", dim, form, seqs, tokens, heads, most, need.value))
for dim in (64, 128):
    for dtype in (L.QFG_BFLOAT16, L.QFG_FLOAT16):
        for rows, seqs in ((1, 1), (77, 1), (300, 5), (8192, 1), (3, 9)):
            run(lambda: lib.qfg_prompt_attention(dtype, P, 8 * dim, rows, 8, P, 2 * dim, P, 2 * dim, rows, 2, dim, P, P, seqs, 1, 0.1, P, None, None), ("prompt", dim, rows, seqs))
print(json.dumps([sorted(built), sorted(launched), failed, grids]))
"""


def test_every_kernel_is_reached_and_blocks_are_enough(tmp_path):
    source, so = tmp_path / "shim.c", str(tmp_path / "libfake_cuda.so")
    source.write_text(SHIM)
    inc = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")
    subprocess.check_call(["gcc", "-shared", "-fPIC", "-O1", "-I" + inc, "-I" + HERE, "-Wl,-soname,libcublas.so.12", "-o", so, str(source)])
    r = subprocess.run([sys.executable, "-c", BODY.format(root=ROOT, here=HERE, fake=so)], env={**os.environ, "LD_PRELOAD": so}, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]
    built, launched, failed, calls = json.loads(r.stdout)
    assert not failed and launched
    assert set(built) == set(launched), f"{len(set(built) - set(launched))} of {len(built)} kernels are never launched: {sorted(set(built) - set(launched))[:3]}"
    for what, lines in calls:
        what = eval(what)
        x, y = [int(v) for v in lines[0].split("grid=")[1].split()[0].split(",")]
        if what[0] in ("heads", "write"):  # every run of rows of every token has a warp that comes by
            tokens, dim = what[-1], what[1]
            rows = 512 // dim
            runs = sum(-(-h // rows) for h in ((40, 2, 2) if what[0] == "heads" else (2, 2)))
            per_block = -(-tokens // x)
            assert (y == 1 and per_block in (1, 2, 4, 8)) or (y * 8 >= runs and x == tokens), (what, x, y)
        if what[0] == "attend":
            _, dim, form, seqs, tokens, heads, most, need = what
            group = tokens * heads // 2
            nt = 2 if group > 8 and dim < 256 else 1
            units = seqs * 2 * -(-group // (8 * nt))
            assert x <= 148 * (2 if dim * nt <= 128 else 1)
            assert need == -(-8 * units // 16) * 16 + x * 8 * 2 * 8 * nt * (dim + 2) * 4
            assert len(lines) == 2 and "JoinKernel" in lines[1] and int(lines[1].split("grid=")[1].split(",")[0]) == units
        if what[0] == "prompt":
            _, dim, rows, seqs = what
            tile = 128 if dim == 64 else 256
            assert x >= 8 * max(-(-rows // tile), min(rows, seqs))
