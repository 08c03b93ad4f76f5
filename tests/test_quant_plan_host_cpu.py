"""QuantGemm's choice of a launch shape on the host, against a CUDA runtime that runs nothing (fake_cuda.c)."""
import json
import os
import subprocess
import sys
import textwrap

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)

PRELUDE = """
import ctypes, importlib.util, json, os, time
spec = importlib.util.spec_from_file_location("qfg_lib", os.path.join({root!r}, "qwen38_flash_ops_b200", "_lib.py"))
L = importlib.util.module_from_spec(spec)
spec.loader.exec_module(L)
lib, fake = L.load(), ctypes.CDLL({fake!r})
fake.fake_log.restype = ctypes.c_char_p
P = 1 << 20  # an address nothing reads
h = ctypes.c_void_p()
assert lib.qfg_quant_gemm_create(None, 0, L.QFG_BFLOAT16, ctypes.byref(h)) == 0

def call(m, k, n, order, odd=0):
    return lib.qfg_quant_gemm_compute(h, L.QFG_INT8, P + odd, k, P, m, k, P, k if order else n, order, n, P, n, None)
"""


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("fake") / "libfake_cuda.so")
    inc = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")
    subprocess.check_call(["gcc", "-shared", "-fPIC", "-O1", "-I" + inc, "-Wl,-soname,libcublas.so.12", "-o", so, os.path.join(HERE, "fake_cuda.c")])

    def run(body):
        code = PRELUDE.format(root=ROOT, fake=so) + textwrap.dedent(body)
        r = subprocess.run([sys.executable, "-c", code], env={**os.environ, "LD_PRELOAD": so}, capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stderr[-2000:]
        return json.loads(r.stdout)

    return run


def test_the_search_does_not_grow_with_the_rows(fake):
    """A call of a million rows takes the host no longer than one of 4096 does: both try a handful of tile heights."""
    few, many = fake("""
        def host(m):
            times = []
            for _ in range(200):
                t = time.perf_counter()
                assert call(m, 5120, 5120, 0) == 0
                times.append(time.perf_counter() - t)
                fake.fake_clear()
            return sorted(times)[20]
        host(64)
        print(json.dumps([host(4096), host(1 << 20)]))
        """)
    assert many < 3 * few, (few, many)
