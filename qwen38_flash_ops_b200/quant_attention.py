"""An attention block in eight bits over a quantised cache, made of the package's operators: norm with the residual's addition, q / k / v projection, norm and
rotation of heads with the write into the cache, attention, output projection.  With QuantMlp it makes a decoder layer.

    python -m qwen38_flash_ops_b200.quant_attention [--rows 8] [--context 4000] [--hidden 5120] [--heads 64] [--kv-heads 8] [--head-dim 128] [--cache nvfp4]

makes one of random weights, runs a prompt and a step over it, compares the step with the same block without a cache and without quantisation, and times it.
"""
from __future__ import annotations

import torch

from .attention import CacheAttention, KvCache, PromptAttention, QkNormRope, _table, _whole_numbers, _workspace_bytes
from .ops import QuantGemm, RmsNormQuant, RowQuant


class QuantAttention:
    """(y, h) = block(x, residual, positions, slots, ...): h = x + residual is the residual stream that goes on, y = out(attention(q, k, v)) of its norm.

    `qkv` [hidden, (heads + 2 * kv_heads) * head_dim] holds the columns of queries, keys, values; `out` [heads * head_dim, hidden]; both torch.int8 or both
    torch.float8_e4m3fn, either dimension contiguous, with a scale per column.  q_weight and k_weight [head_dim] are the heads' norms (or None).  `rope` is a
    QkNormRope and `cache` a KvCache, which is this layer's own.

    x, residual [tokens, hidden] in BF16; positions as the QkNormRope takes them; slots int64 [tokens]: where the tokens go in the cache.
    A prompt: offsets int32 [sequences + 1], the tokens' sequences, which attend to themselves, with keys and values that no cache has rounded; heads of 64 or 128
    channels.  A step: table and lengths, as CacheAttention takes them; the tokens are the last ones of as many sequences, equally many of each.  A call that is refused
    has written nothing into the cache."""

    def __init__(self, norm_weight, qkv, qkv_scale, out, out_scale, heads: int, kv_heads: int, rope: QkNormRope, cache: KvCache, q_weight=None, k_weight=None,
                 eps: float = 1e-6, weight_offset: float = 0.0, scale: float | None = None):
        dim = cache.head_dim
        if qkv.dtype != out.dtype or qkv.shape[1] != (heads + 2 * kv_heads) * dim or tuple(out.shape) != (heads * dim, qkv.shape[0]) or cache.kv_heads != kv_heads:
            raise ValueError("QuantAttention: qkv is [hidden, (heads + 2 * kv_heads) * head_dim] and out [heads * head_dim, hidden], of one type, and the cache has kv_heads")
        if rope.head_dim != dim:
            raise ValueError(f"QuantAttention: the cache has heads of {dim} channels, the QkNormRope of {rope.head_dim}")
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, dim
        self.norm_weight, self.qkv, self.out, self.q_weight, self.k_weight, self.cache = norm_weight, qkv, out, q_weight, k_weight, cache
        self._rope, self._device = rope, cache.k.get_device()
        self._norm = RmsNormQuant(eps=eps, weight_offset=weight_offset, dtype=qkv.dtype)
        self._rows = RowQuant(dtype=qkv.dtype)
        self._qkv, self._out = QuantGemm(w_scale=qkv_scale), QuantGemm(w_scale=out_scale)
        self._prompt, self._step = PromptAttention(scale=scale), CacheAttention(scale=scale)

    def _check_step(self, rows, table, lengths):
        _, _, seqs, most = _table("QuantAttention", table, self.cache)
        tokens = rows // max(1, seqs)
        if _whole_numbers("QuantAttention", "lengths", lengths, (torch.int32,), 1).shape[0] != seqs or tokens * seqs != rows:
            raise ValueError(f"QuantAttention: there must be a length for each of {seqs} sequences, and equally many tokens")
        _workspace_bytes(self.cache, seqs, tokens, self.heads, most)

    def __call__(self, x, residual, positions, slots, table=None, lengths=None, offsets=None):
        if (offsets is None) == (table is None) or (table is None) != (lengths is None):
            raise ValueError("QuantAttention: a prompt has offsets, a step a table and lengths")
        rows, dim = x.shape[0], self.head_dim
        # What the operators behind the cache's write would refuse.  Ordinary arguments have passed in a microsecond (the sizes are well within those that a step's counting sets).
        if offsets is not None:
            if dim == 256:
                raise ValueError("QuantAttention: prompts have heads of 64 or 128 channels")
            plain = offsets.dtype == torch.int32 and offsets.dim() == 1 and offsets.is_contiguous() and offsets.get_device() == self._device
            if offsets.numel() < 1 or not (plain or _whole_numbers("QuantAttention", "offsets", offsets, (torch.int32,), 1) is offsets):
                raise ValueError("QuantAttention: there must be one offset more than sequences")
        else:
            seqs, tokens = lengths.shape[0] if lengths.dim() == 1 else -1, 0
            if seqs > 0:
                tokens = rows // seqs
            if not (table.dtype == lengths.dtype == torch.int32 and table.dim() == 2 and table.shape[0] == seqs and tokens * seqs == rows and table.is_contiguous() and
                    lengths.is_contiguous() and table.get_device() == lengths.get_device() == self._device and seqs <= 65536 and tokens <= 1024 and
                    table.numel() * self.cache.page <= 1 << 22):
                self._check_step(rows, table, lengths)
        rows8, scale, h = self._norm(x, self.norm_weight, residual)
        both = self._qkv(rows8, scale, self.qkv).view(rows, self.heads + 2 * self.kv_heads, dim)
        q, k, v = both[:, :self.heads], both[:, self.heads:-self.kv_heads], both[:, -self.kv_heads:]
        if offsets is not None:
            q, k = self._rope(q, k, positions, self.q_weight, self.k_weight, v, self.cache, slots, True)
            y = self._prompt(q, k, v, offsets)
        else:
            q = self._rope(q, k, positions, self.q_weight, self.k_weight, v, self.cache, slots)
            y = self._step(q.view(seqs, tokens, self.heads, dim), self.cache, table, lengths)
        rows8, scale = self._rows(y.view(rows, self.heads * dim))
        return self._out(rows8, scale, self.out), h


def main() -> None:
    import argparse

    from .packing_torch import quantize_fp8_per_column_torch, quantize_int8_per_column_torch

    p = argparse.ArgumentParser(description="a step of an attention block in eight bits against its unquantised form")
    p.add_argument("--rows", type=int, default=8, help="sequences, of one token each")
    p.add_argument("--context", type=int, default=4000, help="tokens of each sequence ahead of the step")
    p.add_argument("--hidden", type=int, default=5120)
    p.add_argument("--heads", type=int, default=64)
    p.add_argument("--kv-heads", type=int, default=8)
    p.add_argument("--head-dim", type=int, default=128)
    p.add_argument("--dtype", choices=("int8", "e4m3"), default="int8")
    p.add_argument("--cache", choices=("nvfp4", "e4m3"), default="nvfp4")
    a = p.parse_args()
    gen = torch.Generator(device="cuda").manual_seed(0)
    randn = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    quantise = quantize_int8_per_column_torch if a.dtype == "int8" else quantize_fp8_per_column_torch
    heads, kv, dim, rows, context, page = a.heads, a.kv_heads, a.head_dim, a.rows, a.context, 64
    w1, w2 = randn(a.hidden, (heads + 2 * kv) * dim) * 0.02, randn(heads * dim, a.hidden) * 0.02
    (q1, s1), (q2, s2) = quantise(w1), quantise(w2)
    g, ones = (1 + 0.2 * randn(a.hidden)).bfloat16(), torch.ones(dim, device="cuda").bfloat16()
    most = -(-(context + 1) // page)
    cache = KvCache(rows * most, kv, dim, page, torch.uint8 if a.cache == "nvfp4" else torch.float8_e4m3fn)
    rope = QkNormRope(dim, base=1000000.0)
    block = QuantAttention(g, q1, s1.cpu().numpy(), q2, s2.cpu().numpy(), heads, kv, rope, cache, ones, ones)
    table = torch.arange(rows * most, device="cuda", dtype=torch.int32).view(rows, most)
    slot = lambda seq, token: table[seq, token // page].long() * page + token % page
    # the contexts, all of the tokens alike in kind, as one packed prompt a sequence
    keys, values = [], []
    for i in range(rows):
        x, at = randn(context, a.hidden).bfloat16(), torch.arange(context, device="cuda")
        offsets = torch.tensor([0, context], dtype=torch.int32, device="cuda")
        zero = torch.zeros_like(x)
        block(x, zero, at, slot(torch.full_like(at, i), at), offsets=offsets)
        f = x.float()
        both = (f * torch.rsqrt((f * f).mean(-1, keepdim=True) + 1e-6) * g.float() @ w1).view(context, -1, dim)
        keys.append(rope(both[:, :1].contiguous(), both[:, heads:-kv].contiguous(), at, ones.float(), ones.float())[1])
        values.append(both[:, -kv:])
    x, residual = randn(rows, a.hidden).bfloat16(), torch.zeros(rows, a.hidden, device="cuda").bfloat16()
    at, seq = torch.full((rows,), context, device="cuda"), torch.arange(rows, device="cuda")
    lengths = torch.full((rows,), context + 1, device="cuda", dtype=torch.int32)
    step = lambda: block(x, residual, at, slot(seq, at), table=table, lengths=lengths)
    y, _ = step()
    f = x.float()
    both = (f * torch.rsqrt((f * f).mean(-1, keepdim=True) + 1e-6) * g.float() @ w1).view(rows, -1, dim)
    q, k = rope(both[:, :heads].contiguous(), both[:, heads:-kv].contiguous(), at, ones.float(), ones.float())
    want = []
    for i in range(rows):
        ki, vi = torch.cat([keys[i], k[i:i + 1]]), torch.cat([values[i], both[i:i + 1, -kv:]])
        s = torch.einsum("hgd,nhd->hgn", q[i].view(kv, -1, dim), ki) / dim ** 0.5
        want.append(torch.einsum("hgn,nhd->hgd", torch.softmax(s, -1), vi).reshape(-1))
    want = torch.stack(want) @ w2
    print(f"relative difference from the unquantised block: {((y.float() - want).norm() / want.norm()).item():.4f}")
    for _ in range(3):
        step()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(50):
        step()
    end.record()
    torch.cuda.synchronize()
    print(f"{start.elapsed_time(end) / 50 * 1e3:.1f} us a step, {rows} sequences of {context} tokens, {a.hidden} -> {heads} and {kv} heads of {dim}, {a.dtype}, {a.cache} cache")


if __name__ == "__main__":
    main()
