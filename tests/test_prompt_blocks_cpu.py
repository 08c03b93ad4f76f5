"""PromptAttention has a block for every tile of queries, however the rows are split into sequences: its grids against a CUDA runtime that runs nothing (fake_cuda.c)."""
import json
import os
import subprocess
import sys
from functools import lru_cache

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CALLS = [(rows, seqs) for rows in (1, 2, 3, 127, 128, 129, 255, 256, 257, 300, 385, 640, 1000) for seqs in (1, 2, 3, 5, 9, 40)] + [(8192, 1), (8192, 7), (100000, 33), (3, 65536), (70000, 65536)]
BODY = """
import ctypes, importlib.util, json, os
spec = importlib.util.spec_from_file_location("qfg_lib", os.path.join({root!r}, "qwen38_flash_ops_b200", "_lib.py"))
L = importlib.util.module_from_spec(spec)
spec.loader.exec_module(L)
lib, fake = L.load(), ctypes.CDLL({fake!r})
fake.fake_log.restype = ctypes.c_char_p
P, grids = 1 << 20, []  # P: an address nothing reads
for dim in (64, 128):
    for heads in (1, 8):
        for rows, seqs in {calls!r}:
            fake.fake_clear()
            assert lib.qfg_prompt_attention(L.QFG_BFLOAT16, P, heads * dim, rows, heads, P, dim, P, dim, rows, 1, dim, P, P, seqs, 1, 0.1, P, None, None) == 0
            (line,) = fake.fake_log().decode().splitlines()
            grids.append([dim, heads, rows, seqs, [int(n) for n in line.split("grid=")[1].split()[0].split(",")]])
print(json.dumps(grids))
"""


@lru_cache(None)
def most_tiles(rows, seqs, tile):
    """The largest sum of ceil(n_i / tile) over all n_1 + ... + n_seqs = rows, tried out."""
    if seqs == 1:
        return -(-rows // tile)
    return max(-(-n // tile) + most_tiles(rows - n, seqs - 1, tile) for n in {0, 1, rows, *range(1, rows + 1, tile)} if n <= rows)


def test_the_largest_sum_of_tiles():
    """The formula below, against trying."""
    for tile in (4, 7):
        for rows in range(1, 30):
            for seqs in range(1, 7):
                full = max(sum(-(-n // tile) for n in split) for split in splits(rows, seqs))
                assert full == most_tiles(rows, seqs, tile) == formula(rows, seqs, tile)


def splits(rows, seqs):
    if seqs == 1:
        yield (rows,)
        return
    for n in range(rows + 1):
        for rest in splits(rows - n, seqs - 1):
            if rest[0] <= n:  # each split once, in falling order
                yield (n, *rest)


def formula(rows, seqs, tile):
    some = min(rows, seqs)  # sequences that are not empty: a row each, and the others in whole tiles
    return some + (rows - some) // tile


def test_blocks_are_enough(tmp_path):
    so = str(tmp_path / "libfake_cuda.so")
    inc = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")
    subprocess.check_call(["gcc", "-shared", "-fPIC", "-O1", "-I" + inc, "-Wl,-soname,libcublas.so.12", "-o", so, os.path.join(HERE, "fake_cuda.c")])
    r = subprocess.run([sys.executable, "-c", BODY.format(root=ROOT, fake=so, calls=CALLS)], env={**os.environ, "LD_PRELOAD": so}, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]
    grids = json.loads(r.stdout)
    assert len(grids) == 4 * len(CALLS)
    for dim, heads, rows, seqs, grid in grids:
        tile = 128 if dim == 64 else 256
        need = formula(rows, seqs, tile)  # rows / tile + seqs, which the host has at hand, is more by at most seqs / tile
        assert grid[1] == 1 and heads * need <= grid[0] <= heads * (need + -(-min(rows, seqs) // tile)), (dim, heads, rows, seqs, grid)
