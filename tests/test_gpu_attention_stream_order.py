"""Heads, caches and attention see what the kernels before them in the stream wrote, although their blocks may be placed before those have ended, and are done with
their inputs before the kernels behind them write: copies and a late writer ahead of each call, and chains of calls with nothing waited for."""
import pytest
import torch
from test_gpu_stream_order import _Early, _rand

from _attention import new_cache
from qwen38_flash_ops_b200 import CacheAttention, CacheRead, CacheWrite, KvCache, PromptAttention, QkNormRope, QuantGemm, RowQuant

pytestmark = pytest.mark.gpu


def _whole(*v):
    return torch.tensor(v, dtype=torch.int32).cuda()


def _bits(t):
    return t.contiguous().view(torch.uint8)


def _held(cache):
    return [cache.k.clone(), cache.k_scale.clone(), cache.v.clone(), cache.v_scale.clone()]


def _call(kind, reads):
    """A call that reads a [8, 2560] BF16 buffer as `reads`: buffer -> outputs."""
    rows = lambda b, dim: b.reshape(-1, 2, dim)  # [80, 2, 128] and the like
    numbers = lambda b: b[0].view(torch.int32)
    if kind in ("heads", "few heads"):
        n = 80 if kind == "heads" else 6
        other, w, at, slots, op = _rand(1, n, 2, 128), _rand(2, 128), torch.arange(n).cuda(), torch.arange(n).cuda(), QkNormRope(128)

        def call(b):
            cache, x = new_cache("nvfp4", 3, 2, 128), rows(b, 128)[:n]
            given = {"q": other, "k": other, "v": other, "weight": w, "positions": at, "slots": slots}
            given[reads] = {"weight": b[7, :128], "positions": numbers(b)[:n], "slots": numbers(b)[:n].long() % 96}.get(reads, x)
            if reads == "slots":
                given[reads] = torch.sort(given[reads]).values  # made by torch: an ordinary kernel ahead, and equal slots would race
                given[reads] = torch.where(torch.diff(given[reads], prepend=given[reads][:1] - 1) > 0, given[reads], -1)
            out = op(given["q"], given["k"], given["positions"], given["weight"], given["weight"], given["v"], cache, given["slots"], True)
            return [*out, *_held(cache)]

        return call
    if kind == "write":
        other, slots = _rand(3, 80, 2, 128), torch.arange(80).cuda()

        def call(b):
            cache = new_cache("e4m3", 3, 2, 128)
            CacheWrite()(*((rows(b, 128), other) if reads == "k" else (other, rows(b, 128))), cache, slots)
            return _held(cache)

        return call
    # a cache whose codes are the buffer, or another one
    codes, others = lambda b: b.view(torch.uint8).reshape(10, 2, 32, 64), [_rand(4 + i, 8, 2560) for i in range(2)]
    scale = torch.randint(40, 72, (10, 2, 32, 8), generator=torch.Generator().manual_seed(5), dtype=torch.uint8).cuda().view(torch.float8_e4m3fn)

    def cache_of(b):
        k, v = (codes(b) if reads == name else codes(o) for name, o in zip(("codes k", "codes v"), others))
        return KvCache.of(k, scale, v, scale, 0.05, 0.05)

    if kind == "read":
        table, offsets = torch.arange(10).int().view(2, 5).cuda(), _whole(0, 150, 300)
        return lambda b: CacheRead()(cache_of(b), numbers(b)[:10].view(2, 5) % 10 if reads == "table" else table, offsets, 300)
    if kind in ("attend", "attend uncut"):
        most = 5 if kind == "attend" else 1
        table, n, q = torch.arange(2 * most).int().view(2, most).cuda(), _whole(32 * most, 32 * most - 9), _rand(6, 2, 6, 128)

        def call(b):
            other_q = rows(b, 128)[:6].reshape(2, 6, 128) if reads == "q" else q
            lengths = numbers(b)[:2] % (32 * most) if reads == "lengths" else n
            return CacheAttention()(other_q, cache_of(b), table, lengths, lse=True)

        return call
    dim = 64 if kind == "prompt 64" else 128
    other, at = [_rand(7 + i, 8, 2560) for i in range(3)], _whole(0, 7, 10240 // dim)  # every row is of a sequence
    return lambda b: PromptAttention()(*(rows(b if reads == name else o, dim) for name, o in zip("qkv", other)), at, lse=True)


CALLS = ([(k, r) for k in ("heads", "few heads") for r in ("q", "k", "v", "weight", "positions", "slots")] + [("write", r) for r in "kv"] +
         [("read", r) for r in ("codes k", "codes v", "table")] + [(k, r) for k in ("attend", "attend uncut") for r in ("q", "codes k", "codes v", "lengths")] +
         [(k, r) for k in ("prompt 64", "prompt 128") for r in "qkv"])


@pytest.mark.parametrize("case", CALLS, ids="-".join)
def test_behind_a_predecessor_that_released_its_dependents(cuda, case):
    early, call, buffer = _Early(), _call(*case), _rand(920, 8, 2560)
    alone = []
    for i in range(2):
        early(i, buffer)
        torch.cuda.synchronize()
        alone.append([o.clone() for o in call(buffer)])
        torch.cuda.synchronize()
    assert any(not torch.equal(_bits(a), _bits(b)) for a, b in zip(*alone))  # the two inputs tell
    got = []
    for i in range(12):
        early(i, buffer)
        got.append(call(buffer))
        if i % 3 == 2:
            torch.cuda.synchronize()
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(_bits(p), _bits(q)) for p, q in zip(alone[i % 2], g)), i


@pytest.mark.parametrize("case", CALLS, ids="-".join)
def test_inputs_written_just_before(cuda, case):
    call, sources = _call(*case), [_rand(950 + i, 8, 2560) for i in range(6)]
    alone = []
    for s in sources:
        alone.append([o.clone() for o in call(s)])
        torch.cuda.synchronize()
    buffer, delay, got = torch.empty_like(sources[0]), torch.empty(1 << 24, device="cuda"), []
    for s in sources:
        delay.fill_(1.0)  # the copy behind it is in the stream before it is done
        buffer.copy_(s)
        got.append(call(buffer))
    torch.cuda.synchronize()
    for a, g in zip(alone, got):
        assert all(torch.equal(_bits(p), _bits(q)) for p, q in zip(a, g))


@pytest.mark.parametrize("form", ["nvfp4", "e4m3"])
@pytest.mark.parametrize("most", [1, 40])  # pages: sequences that are never cut, and such as are
def test_steps_in_a_row(cuda, most, form):
    """Heads into the cache, attention over it, its rows in eight bits and their product, the cache read back; then the next step over the same slots, table and lengths."""
    seqs, heads, kv, dim = 3, 8, 2, 128
    rope, attend, rows8, gemm, read = QkNormRope(dim), CacheAttention(), RowQuant(), QuantGemm(out_dtype=torch.float32), CacheRead()
    w, w8 = _rand(1, dim), torch.randint(-127, 128, (heads * dim, 640), generator=torch.Generator().manual_seed(2)).to(torch.int8).cuda()
    inputs = [(_rand(10 + i, seqs, heads, dim), _rand(40 + i, seqs, kv, dim), _rand(70 + i, seqs, kv, dim)) for i in range(12)]
    first = _rand(100, seqs * most * 32, kv, dim)

    def run(wait):
        cache = new_cache(form, seqs * most, kv, dim)
        table, n, at = torch.arange(seqs * most).int().view(seqs, most).cuda(), torch.full((seqs,), most * 32 - 14, dtype=torch.int32).cuda(), torch.arange(seqs).cuda() * 100
        offsets = _whole(0, 20, 50, 60)
        CacheWrite()(first, first, cache, torch.arange(seqs * most * 32).cuda())
        outs = []
        for q, k, v in inputs:
            slots = table[:, -1].long() * 32 + (n.long() - 1) % 32
            wait()
            q = rope(q, k, at, w, w, v, cache, slots)
            wait()
            y, lse = attend(q, cache, table, n, lse=True)
            wait()
            x8, s = rows8(y.view(seqs, -1))
            wait()
            z = gemm(x8, s, w8)
            wait()
            kv_rows = read(cache, table, offsets, 60)
            wait()
            CacheWrite()(k, v, cache, slots + 1)  # over what has just been read
            wait()
            outs += [y, lse, z, *kv_rows]
            n.add_(1), at.add_(7), table.copy_(table.roll(1, 0))
            wait()
        return [*outs, *_held(cache)]

    want = run(torch.cuda.synchronize)
    for _ in range(4):
        got = run(lambda: None)
        torch.cuda.synchronize()
        assert all(torch.equal(_bits(a), _bits(b)) for a, b in zip(want, got))


def test_prompts_in_a_row(cuda):
    """Heads, a prompt over them, its rows in eight bits, over the same tensors again and again."""
    rows, heads, kv, dim = 300, 8, 2, 128
    rope, prompt, rows8 = QkNormRope(dim), PromptAttention(), RowQuant()
    w, at, offsets = _rand(1, dim), torch.arange(rows).cuda(), _whole(0, 129, 300)
    sources = [_rand(10 + i, rows, heads + 2 * kv, dim) for i in range(6)]
    both, out = torch.empty_like(sources[0]), torch.empty(rows, heads, dim, device="cuda").bfloat16()

    def run(wait):
        outs = []
        for s in sources:
            both.copy_(s)
            wait()
            q, k = rope(both[:, :heads], both[:, heads:-kv], at, w, w)
            wait()
            prompt(q, k, both[:, -kv:], offsets, out=out)
            wait()
            outs += rows8(out.view(rows, -1))
            wait()
        return outs

    want = [o.clone() for o in run(torch.cuda.synchronize)]
    for _ in range(4):
        got = run(lambda: None)
        torch.cuda.synchronize()
        assert all(torch.equal(_bits(a), _bits(b)) for a, b in zip(want, got))
