"""The row kernels' launches, against a CUDA runtime that runs nothing (fake_cuda.c): every kernel that is built is one that some call launches."""
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
import ctypes, importlib.util, json, os
spec = importlib.util.spec_from_file_location("qfg_lib", os.path.join({root!r}, "qwen38_flash_ops_b200", "_lib.py"))
L = importlib.util.module_from_spec(spec)
spec.loader.exec_module(L)
lib, fake = L.load(), ctypes.CDLL({fake!r})
fake.fake_log.restype = fake.fake_registered.restype = ctypes.c_char_p
P = 1 << 20  # an address nothing reads
mine = lambda name: "RowQuantKernel" in name or "RowRingKernel" in name
built, i = set(), 0
while fake.fake_registered(i):
    name = fake.fake_registered(i).decode()
    built |= {{name}} if mine(name) else set()
    i += 1
edges = {{e + d for e in (4096, 8192, 12288, 13440, 16384, 18432, 19968, 26880) for d in (-8, -1, 0, 1, 8)}}
lengths = sorted(edges | {{1, 7, 8, 31, 64, 128, 255, 256, 257, 504, 512, 513, 520, 640, 2048, 2560, 5120, 6144, 10240, 30000, 40000, 45000}})
launched, failed = set(), []
for dtype in (L.QFG_BFLOAT16, L.QFG_FLOAT16, L.QFG_FLOAT):
    for rows in (1, 8, 296, 297, 4096):
        for n in lengths:
            for base in (P, P + 4):
                calls = [lambda u=u: lib.qfg_row_quant(dtype, base, n, u, n, rows, n, L.QFG_INT8, P, P, None) for u in (None, P)]
                calls += [lambda r=r: lib.qfg_rmsnorm_quant(dtype, base, n, r, n, P, dtype, 0.0, 1e-6, rows, n, L.QFG_INT8, P, P, P, None) for r in (None, P)]
                for call in calls:
                    fake.fake_clear()
                    if call() != 0:
                        failed.append([dtype, rows, n, base, lib.qfg_last_error().decode()])
                    launched |= {{l.split()[1] for l in fake.fake_log().decode().splitlines()}}
print(json.dumps([sorted(built), sorted(launched), failed]))
"""


def test_every_row_kernel_is_reached(tmp_path):
    source, so = tmp_path / "shim.c", str(tmp_path / "libfake_cuda.so")
    source.write_text(SHIM)
    inc = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")
    subprocess.check_call(["gcc", "-shared", "-fPIC", "-O1", "-I" + inc, "-I" + HERE, "-Wl,-soname,libcublas.so.12", "-o", so, str(source)])
    r = subprocess.run([sys.executable, "-c", BODY.format(root=ROOT, fake=so)], env={**os.environ, "LD_PRELOAD": so}, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]
    built, launched, failed = json.loads(r.stdout)
    assert not failed and launched and set(launched) <= set(built)
    assert set(built) == set(launched), f"{len(set(built) - set(launched))} of {len(built)} kernels are never launched: {sorted(set(built) - set(launched))[:3]}"
