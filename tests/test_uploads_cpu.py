"""What a node uploads when it is made is on the device before the node is handed out, against a CUDA runtime that runs nothing (fake_cuda.c): a copy from pageable memory may
return while its last part is still on its way, and streams that do not wait for the default stream would read what is there ahead of it."""
import json
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)

SHIM = """
#define cudaMemcpy unused_copy
#define cudaStreamSynchronize unused_wait
#include "fake_cuda.c"
#undef cudaMemcpy
#undef cudaStreamSynchronize
API cudaError_t cudaMemcpy(void* d, const void* s, size_t n, enum cudaMemcpyKind k) { (void)d; (void)s; (void)n; (void)k; note("copy"); return cudaSuccess; }
API cudaError_t cudaStreamSynchronize(cudaStream_t s) { note(s == 0 ? "wait" : "wait for another"); return cudaSuccess; }
"""
BODY = """
import ctypes, importlib.util, json, os
spec = importlib.util.spec_from_file_location("qfg_lib", os.path.join({root!r}, "qwen38_flash_ops_b200", "_lib.py"))
L = importlib.util.module_from_spec(spec)
spec.loader.exec_module(L)
lib, fake = L.load(), ctypes.CDLL({fake!r})
fake.fake_log.restype = ctypes.c_char_p
logs = {{}}
def made(name, create):
    fake.fake_clear()
    h = ctypes.c_void_p()
    assert create(ctypes.byref(h)) == 0 and h.value, (name, lib.qfg_last_error())
    logs[name] = fake.fake_log().decode().split("\\n")[:-1]
scales = (ctypes.c_float * 500)(*[1.0] * 500)
made("rotation", lambda h: lib.qfg_qk_norm_rope_create((ctypes.c_double * 32)(*[0.5] * 32), None, 32, 64, 0, 1.0, 1e-6, 0.0, h))
made("no rotation", lambda h: lib.qfg_qk_norm_rope_create(None, None, 0, 64, 0, 1.0, 1e-6, 0.0, h))
made("scales", lambda h: lib.qfg_quant_gemm_create(scales, 500, L.QFG_BFLOAT16, h))
made("no scales", lambda h: lib.qfg_quant_gemm_create(None, 0, L.QFG_BFLOAT16, h))
print(json.dumps(logs))
"""


def test_copies_are_waited_for(tmp_path):
    source, so = tmp_path / "shim.c", str(tmp_path / "libfake_cuda.so")
    source.write_text(SHIM)
    inc = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")
    subprocess.check_call(["gcc", "-shared", "-fPIC", "-O1", "-I" + inc, "-I" + HERE, "-Wl,-soname,libcublas.so.12", "-o", so, str(source)])
    r = subprocess.run([sys.executable, "-c", BODY.format(root=ROOT, fake=so)], env={**os.environ, "LD_PRELOAD": so}, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]
    logs = json.loads(r.stdout)
    assert logs["rotation"] == logs["scales"] == ["copy", "wait"] and logs["no rotation"] == logs["no scales"] == []
