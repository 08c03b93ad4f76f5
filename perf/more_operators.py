"""The operators between a block's projections, for timing and comparison: the norm and rotation of query and key heads with the
write into a quantised cache, that cache written and read back, attention of the last tokens over it, and attention over whole prompts.

Heads are those of the package's q / k / v projection (5120 -> 8192 + 1024 + 1024: 64 query and 8 key heads of 128), and others.
Keys have channels of very different size, as a model's do.  A case is a dict:

  op        heads | cache | decode | prompt
  source    bf16 | f16: the type of queries, keys and values
  q_heads, kv_heads, dim
  form      nvfp4 | e4m3 | none: what the cache holds ("none", heads: no cache, the keys are returned)
  tokens    heads: rows; cache: new tokens of each sequence; decode: the last tokens of each sequence, that attend
  seqs      sequences; the i-th one's length is a fixed part of `length`, between a tenth of it and all
  length    the longest sequence
  page      tokens of a cache page
  axes      heads: positions for each token, 1 or 3 (time, height, width)
  rotary    heads: channels of a head that are rotated
  pairs     heads: neighbours are rotated together, else the halves of the rotated part
  prefix    prompt: keys of each sequence that lie ahead of its queries
  causal    prompt

A cache holds pages of one head each: NVFP4, codes [pages, kv_heads, page, dim / 2] with an E4M3 scale for each 16 channels; E4M3
with an FP32 scale for each token and head.
"""
import math

import torch

own = False

_SOURCE = {"bf16": torch.bfloat16, "f16": torch.float16}
_EPS = 1e-6
_BASE = 1000000.0
_K_UNIT, _V_UNIT = 0.5, 0.125  # what a 1 in a cache of four bits stands for
_LEAST = 2.0 ** -40            # an E4M3 row's scale is no smaller


def _heads(name, tokens, q_heads=64, kv_heads=8, dim=128, source="bf16", form="e4m3", axes=1, rotary=128, pairs=False, page=64):
    c = {"op": "heads", "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "source": source, "form": form, "axes": axes, "rotary": rotary,
         "pairs": pairs, "page": page}
    return {"name": name, **c} if name else c


def _cache(name, seqs, length, tokens, form, kv_heads=8, dim=128, source="bf16", page=64):
    c = {"op": "cache", "seqs": seqs, "length": length, "tokens": tokens, "form": form, "kv_heads": kv_heads, "dim": dim, "source": source, "page": page}
    return {"name": name, **c} if name else c


def _decode(name, seqs, length, tokens, form, q_heads=64, kv_heads=8, dim=128, source="bf16", page=64):
    c = {"op": "decode", "seqs": seqs, "length": length, "tokens": tokens, "form": form, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "source": source,
         "page": page}
    return {"name": name, **c} if name else c


def _prompt(name, seqs, length, prefix=0, q_heads=64, kv_heads=8, dim=128, source="bf16", causal=True):
    c = {"op": "prompt", "seqs": seqs, "length": length, "prefix": prefix, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "source": source, "causal": causal}
    return {"name": name, **c} if name else c


def listed():
    return [
        # a decode step of eight sequences: latency
        _heads("heads_decode", 8),
        # a prompt chunk of text and images, positions by time, height and width
        _heads("heads_prompt_axes", 4096, axes=3),
        # wide heads of which a quarter is rotated, neighbours together, an odd number of tokens, no cache
        _heads("heads_partial_f16", 509, 24, 4, 256, "f16", "none", 1, 64, True),
        # sequences of a few hundred tokens, one new token each, read back to be moved elsewhere
        _cache("cache_step_e4m3", 16, 300, 1, "e4m3", page=32),
        # a chunk of a long prompt is written, and the prompt so far is read back for the next chunk's attention
        _cache("cache_chunk_nvfp4", 1, 10007, 2048, "nvfp4"),
        # one user's next token: latency
        _decode("decode_one_nvfp4", 1, 1000, 1, "nvfp4"),
        # a serving batch of very different lengths
        _decode("decode_batch_nvfp4", 64, 8192, 1, "nvfp4"),
        # drafted tokens checked together
        _decode("decode_draft_nvfp4", 16, 4001, 4, "nvfp4", 32, 8, source="f16", page=32),
        # few very long contexts
        _decode("decode_long_e4m3", 2, 131072, 1, "e4m3", page=128),
        # a short question: latency
        _prompt("prompt_short", 1, 77),
        # chunks of several prompts in one call, behind what their caches hold
        _prompt("prompt_packed_f16", 11, 640, 300, 24, 8, 64, "f16"),
        # a whole long prompt, the largest
        _prompt("prompt_long", 1, 8192),
    ]


def _log_int(rng, lo, hi, step=1):
    v = lo * (hi / lo) ** rng.random()
    return max(lo, min(hi, int(round(v / step)) * step))


def _plain_cost(c):
    """Elements that the plain form makes: what bounds its time and memory."""
    if c["op"] == "prompt":
        return sum(_lengths(c)) * sum(n + c["prefix"] for n in _lengths(c)) * c["q_heads"]
    if c["op"] == "heads":
        return c["tokens"] * (c["q_heads"] + 2 * c["kv_heads"]) * c["dim"]
    return c["seqs"] * c["length"] * c["kv_heads"] * c["dim"]


def draw(rng):
    most = {m: max(work(c)[m] for c in listed()) for m in ("bytes", "flops")}
    limit = {}
    for c in listed():
        limit[c["op"]] = max(limit.get(c["op"], 0), _plain_cost(c))
    while True:
        op = rng.choice(["heads"] * 2 + ["cache"] * 2 + ["decode"] * 5 + ["prompt"] * 3)
        source, form = rng.choice(["bf16", "bf16", "f16"]), rng.choice(["nvfp4", "nvfp4", "e4m3"])
        kv_heads, group, page = rng.choice([1, 2, 4, 8, 8, 20]), rng.choice([1, 2, 3, 4, 5, 8, 8, 12, 16]), rng.choice([32, 64, 64, 96, 256])
        dim = rng.choice([64, 128, 128, 128, 256])
        if op == "heads":
            c = _heads(None, rng.choice([rng.randint(1, 16), _log_int(rng, 1, 8192)]), group * kv_heads, kv_heads, dim, source, rng.choice(["e4m3", "none"]),
                       rng.choice([1, 3]), rng.choice([r for r in (32, 64, 128, 256) if r <= dim]), rng.random() < 0.4, page)
        elif op == "cache":
            length = _log_int(rng, 1, 32768)
            c = _cache(None, rng.choice([1, rng.randint(1, 64)]), length, rng.choice([1, _log_int(rng, 1, length)]), form, kv_heads, dim, source, page)
        elif op == "decode":
            c = _decode(None, rng.choice([1, rng.randint(1, 8), _log_int(rng, 1, 256)]), _log_int(rng, 16, 131072), rng.choice([1, 1, 1, 2, 3, 4, 8]), form,
                        group * kv_heads, kv_heads, dim, source, page)
        else:
            c = _prompt(None, rng.choice([1, 1, rng.randint(1, 24)]), _log_int(rng, 1, 16384), rng.choice([0, 0, _log_int(rng, 1, 4096)]), group * kv_heads, kv_heads,
                        rng.choice([64, 128, 128]), source, rng.random() < 0.8)
        w = work(c)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and _plain_cost(c) <= limit[op]:
            return c


def _lengths(c):
    """The sequences' lengths: the first is the longest, the others any part of it from a tenth."""
    return [max(1, int(c["length"] * (1 - 0.9 * ((i * 0.6180339887) % 1)))) for i in range(c["seqs"])]


# ------------------------------------------------------------------------------ inputs
def _rows(gen, rows, heads, dim, spread, source):
    """Heads whose channels differ in size, the same ones for every token."""
    channel = torch.exp(spread * torch.randn(heads, dim, generator=gen, device="cuda"))
    return (torch.randn(rows, heads, dim, generator=gen, device="cuda") * channel).to(source)


def _table(gen, case, spare=3):
    """Pages of each sequence, in any order over the cache: int32 [seqs, most], and how many the cache has."""
    most = -(-case["length"] // case["page"])
    pages = case["seqs"] * most + spare
    order = torch.randperm(pages, generator=gen, device="cuda")[:case["seqs"] * most]
    return order.view(case["seqs"], most).to(torch.int32), pages


def _slots(table, page, seq, token):
    """Where tokens of sequences lie in the cache: page times its size, and the place in it."""
    return table[seq, token // page].long() * page + token % page


def _offsets(lengths):
    return torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device="cuda")


def _owner(offsets, rows):
    """For each packed row its sequence, and its place in it."""
    at = torch.arange(rows, device=offsets.device)
    seq = torch.searchsorted(offsets[1:].long(), at, right=True)
    return seq, at - offsets.long()[seq]


def _empty_cache(form, pages, kv_heads, page, dim):
    shape = (pages, kv_heads, page)
    if form == "e4m3":
        return [torch.zeros(*shape, dim, device="cuda").to(torch.float8_e4m3fn), torch.zeros(*shape, device="cuda")]
    return [torch.zeros(*shape, dim // 2, dtype=torch.uint8, device="cuda"), torch.zeros(*shape, dim // 16, device="cuda").to(torch.float8_e4m3fn)]


def _filled(gen, form, pages, kv_heads, page, dim, unit, spread):
    """A cache's keys or values: every page holds something, as a cache in use does."""
    part = max(1, (1 << 26) // (kv_heads * page * dim))
    channel = torch.exp(spread * torch.randn(kv_heads, 1, dim, generator=gen, device="cuda"))
    made = [_quantised(torch.randn(min(part, pages - p), kv_heads, page, dim, generator=gen, device="cuda") * channel, form, unit) for p in range(0, pages, part)]
    return [torch.cat([m[0] for m in made]), torch.cat([m[1] for m in made])]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 1000 + 37)
    op, source, dim, kv_heads = case["op"], _SOURCE[case["source"]], case["dim"], case["kv_heads"]
    st = {"case": case, "op": op}
    randn = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    if op == "heads":
        tokens = case["tokens"]
        st["q"], st["k"] = _rows(gen, tokens, case["q_heads"], dim, 0.5, source), _rows(gen, tokens, kv_heads, dim, 0.5, source)
        st["v"] = _rows(gen, tokens, kv_heads, dim, 0.3, source)
        st["q_weight"], st["k_weight"] = (1 + 0.2 * randn(dim)).to(source), (1 + 0.2 * randn(dim)).to(source)
        start = torch.randint(0, 100000, (case["axes"], 1), generator=gen, device="cuda")
        st["positions"] = start + torch.arange(tokens, device="cuda") // torch.tensor([[1], [24], [1]], device="cuda")[:case["axes"]]
        st["positions"] = st["positions"][0] if case["axes"] == 1 else st["positions"]
        pairs = case["rotary"] // 2
        st["sections"] = [pairs] if case["axes"] == 1 else [pairs - 2 * (3 * pairs // 8), 3 * pairs // 8, 3 * pairs // 8]
        if case["form"] != "none":
            pages = -(-tokens // case["page"]) + 3
            st["slots"] = torch.randperm(pages * case["page"], generator=gen, device="cuda")[:tokens]
            st["k_cache"], st["v_cache"] = (_empty_cache(case["form"], pages, kv_heads, case["page"], dim) for _ in range(2))
    elif op == "prompt":
        lengths = _lengths(case)
        st["q"] = _rows(gen, sum(lengths), case["q_heads"], dim, 0.2, source)
        rows = sum(lengths) + len(lengths) * case["prefix"]
        st["k"], st["v"] = _rows(gen, rows, kv_heads, dim, 0.2, source), _rows(gen, rows, kv_heads, dim, 0.3, source)
        st["q_offsets"], st["k_offsets"] = _offsets(lengths), _offsets([n + case["prefix"] for n in lengths])
    else:
        lengths = _lengths(case)
        st["table"], pages = _table(gen, case)
        st["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        st["k_cache"] = _filled(gen, case["form"], pages, kv_heads, case["page"], dim, _K_UNIT, 0.4)
        st["v_cache"] = _filled(gen, case["form"], pages, kv_heads, case["page"], dim, _V_UNIT, 0.3)
        if op == "decode":
            st["q"] = randn(case["seqs"], case["tokens"], case["q_heads"], dim).to(source)
        else:
            new = [min(n, case["tokens"]) for n in lengths]
            seq, at = _owner(_offsets(new), sum(new))
            at = at + (st["lengths"].long() - torch.tensor(new, device="cuda"))[seq]  # a sequence's last tokens
            st["slots"] = _slots(st["table"], case["page"], seq, at)
            st["k"], st["v"] = _rows(gen, sum(new), kv_heads, dim, 0.4, source), _rows(gen, sum(new), kv_heads, dim, 0.3, source)
            st["offsets"], st["rows"] = _offsets(lengths), sum(lengths)
    if own:  # the nodes that a program makes once, and its cache
        import qwen38_flash_ops_b200 as framework

        if "k_cache" in st:
            st["cache"] = framework.KvCache.of(*st["k_cache"], *st["v_cache"], k_unit=_K_UNIT, v_unit=_V_UNIT)
        if op == "heads":
            st["node"] = framework.QkNormRope(dim, rotary_dim=case["rotary"], base=_BASE, sections=st["sections"], interleaved=case["pairs"], eps=_EPS)
        elif op == "cache":
            st["node"], st["back"] = framework.CacheWrite(), framework.CacheRead(dtype=source)
        else:
            st["node"] = framework.CacheAttention() if op == "decode" else framework.PromptAttention(causal=case["causal"])
    return st


# ------------------------------------------------------------------------------ plain forms
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _codes(v):
    """The E2M1 code nearest to each value; half-way values go to the even code."""
    a = v.abs()
    code = (a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    return (code + 8 * torch.signbit(v)).to(torch.uint8)


def _quantised(y, form, unit):
    """FP32 rows [..., dim] -> what a cache holds of them."""
    if form == "e4m3":
        scale = (y.abs().amax(dim=-1) / 448).clamp(min=_LEAST)
        return (y / scale[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn), scale
    blocks = y.unflatten(-1, (-1, 16))
    scale = (blocks.abs().amax(dim=-1) / (6 * unit)).clamp(max=448.0).to(torch.float8_e4m3fn).float().clamp(min=2.0 ** -9)
    code = _codes(blocks / (scale * unit)[..., None]).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, scale.to(torch.float8_e4m3fn)


def _values(held, scale, form, unit):
    """What a cache's rows stand for, in FP32."""
    if form == "e4m3":
        return held.float() * scale[..., None]
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=held.device)
    v = torch.stack([table[(held & 15).int()], table[(held >> 4).int()]], dim=-1).flatten(-2)
    return (v.unflatten(-1, (-1, 16)) * (scale.float() * unit)[..., None]).flatten(-2)


def _put(cache, rows, slots, form, unit):
    """Rows [tokens, kv_heads, dim] into their slots."""
    page = cache[0].shape[2]
    for to, what in zip(cache, _quantised(rows.float(), form, unit)):
        to.view(torch.uint8 if to.element_size() == 1 else to.dtype)[slots // page, :, slots % page] = what.view(torch.uint8) if what.element_size() == 1 else what


def _gathered(cache, table, form, unit):
    """FP32 [seqs, kv_heads, tokens, dim] of all pages of the table."""
    v = _values(cache[0][table.long()], cache[1].view(torch.uint8)[table.long()].view(torch.float8_e4m3fn) if form == "nvfp4" else cache[1][table.long()], form, unit)
    return v.transpose(1, 2).flatten(2, 3)


def _plain_heads(st):
    c = st["case"]
    half = c["rotary"] // 2
    freq = _BASE ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    if c["axes"] == 1:
        angle = st["positions"].double()[:, None] * freq
    else:
        axis = torch.repeat_interleave(torch.arange(3, device="cuda"), torch.tensor(st["sections"], device="cuda"))
        angle = st["positions"].double()[axis].t() * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def rotated(x, weight):
        f = x.float()
        f = f * torch.rsqrt((f * f).mean(dim=-1, keepdim=True) + _EPS) * weight.float()
        turned, rest = f[..., :c["rotary"]], f[..., c["rotary"]:]
        a, b = (turned[..., 0::2], turned[..., 1::2]) if c["pairs"] else (turned[..., :half], turned[..., half:])
        a, b = a * cos - b * sin, b * cos + a * sin
        turned = torch.stack([a, b], dim=-1).flatten(-2) if c["pairs"] else torch.cat([a, b], dim=-1)
        return torch.cat([turned, rest], dim=-1)

    q, k = rotated(st["q"], st["q_weight"]).to(st["q"].dtype), rotated(st["k"], st["k_weight"])
    if c["form"] == "none":
        return [q, k.to(st["k"].dtype)]
    _put(st["k_cache"], k, st["slots"], c["form"], _K_UNIT)
    _put(st["v_cache"], st["v"], st["slots"], c["form"], _V_UNIT)
    return [q, *st["k_cache"], *st["v_cache"]]


def _plain_cache(st):
    c = st["case"]
    _put(st["k_cache"], st["k"], st["slots"], c["form"], _K_UNIT)
    _put(st["v_cache"], st["v"], st["slots"], c["form"], _V_UNIT)
    seq, at = _owner(st["offsets"], st["rows"])
    return [_gathered(cache, st["table"], c["form"], unit)[seq, :, at].to(st["k"].dtype) for cache, unit in ((st["k_cache"], _K_UNIT), (st["v_cache"], _V_UNIT))]


def _plain_softmax(s):
    """Over the last dimension; rows that see nothing get no weight."""
    p = torch.exp(s - s.amax(dim=-1, keepdim=True).clamp(min=-3e38))
    return p / p.sum(dim=-1, keepdim=True).clamp(min=1e-37)


def _plain_decode(st):
    c = st["case"]
    k, v = _gathered(st["k_cache"], st["table"], c["form"], _K_UNIT), _gathered(st["v_cache"], st["table"], c["form"], _V_UNIT)
    q = st["q"].float().unflatten(2, (c["kv_heads"], -1)).permute(0, 2, 1, 3, 4)  # [seqs, kv_heads, tokens, group, dim]
    s = (q.flatten(2, 3) @ k.transpose(2, 3)).unflatten(2, (c["tokens"], -1)) / math.sqrt(c["dim"])
    sees = st["lengths"].long()[:, None] - c["tokens"] + 1 + torch.arange(c["tokens"], device="cuda")
    s = torch.where(torch.arange(k.shape[2], device="cuda") < sees[:, None, :, None, None], s, -math.inf)
    y = (_plain_softmax(s).flatten(2, 3) @ v).unflatten(2, (c["tokens"], -1))
    return [y.permute(0, 2, 1, 3, 4).flatten(2, 3).to(st["q"].dtype)]


def _plain_prompt(st):
    c = st["case"]
    q, k, v = (st[n].float().transpose(0, 1) for n in ("q", "k", "v"))
    group = c["q_heads"] // c["kv_heads"]
    (q_seq, q_at), (k_seq, k_at) = _owner(st["q_offsets"], q.shape[1]), _owner(st["k_offsets"], k.shape[1])
    seen = q_seq[:, None] == k_seq
    if c["causal"]:
        seen = seen & (k_at <= q_at[:, None] + c["prefix"])
    s = (q.unflatten(0, (-1, group)).flatten(1, 2) @ k.transpose(1, 2)).unflatten(1, (group, -1)) / math.sqrt(c["dim"])
    p = _plain_softmax(s.masked_fill_(~seen, -math.inf))
    return [(p.flatten(1, 2) @ v).unflatten(1, (group, -1)).flatten(0, 1).transpose(0, 1).to(st["q"].dtype)]


def run(st):
    op = st["op"]
    if not own:
        return {"heads": _plain_heads, "cache": _plain_cache, "decode": _plain_decode, "prompt": _plain_prompt}[op](st)
    if op == "heads":
        if st["case"]["form"] == "none":
            return list(st["node"](st["q"], st["k"], st["positions"], st["q_weight"], st["k_weight"]))
        q = st["node"](st["q"], st["k"], st["positions"], st["q_weight"], st["k_weight"], st["v"], st["cache"], st["slots"])
        return [q, *st["k_cache"], *st["v_cache"]]
    if op == "cache":
        st["node"](st["k"], st["v"], st["cache"], st["slots"])
        return list(st["back"](st["cache"], st["table"], st["offsets"], st["rows"]))
    if op == "decode":
        return [st["node"](st["q"], st["cache"], st["table"], st["lengths"])]
    return [st["node"](st["q"], st["k"], st["v"], st["q_offsets"], st["k_offsets"])]


# ------------------------------------------------------------------------------ in 64 bits
def _exact_scale(y):
    return torch.maximum(y.abs().max(dim=-1).values, torch.tensor(448 * _LEAST, dtype=torch.float64, device=y.device)) / 448


def _exact_held(cache, form, unit):
    """What all of a cache stands for."""
    if form == "e4m3":
        return cache[0].double() * cache[1].double().unsqueeze(-1)
    nibble = torch.cat([(cache[0] & 15).unsqueeze(-1), (cache[0] >> 4).unsqueeze(-1)], dim=-1).reshape(*cache[0].shape[:-1], -1).int()
    size = nibble & 7  # exponent in the upper two bits, mantissa in the lowest
    value = torch.where(size < 2, size.double() / 2, (1 + (size & 1).double() / 2) * torch.exp2((size >> 1).double() - 1))
    value = torch.where(nibble > 7, -value, value)
    return value * torch.repeat_interleave(cache[1].double(), 16, dim=-1) * unit


def _exact_written(y, form, unit):
    """What a cache stands for of rows that were written to it: in four bits the nearest value of the block's scale, in eight bits the row itself, whose
    rounding is smaller than that of the output's type allows for."""
    if form == "e4m3":
        return y
    block = y.reshape(*y.shape[:-1], -1, 16)
    s = (block.abs().max(dim=-1).values / (6 * unit)).float().clamp(max=448.0).to(torch.float8_e4m3fn).double()
    s = torch.where(s == 0, 2.0 ** -9, s)[..., None] * unit
    a = block / s
    step = torch.where(a.abs() < 2, 0.5, torch.where(a.abs() < 4, 1.0, 2.0))
    return (torch.clamp(torch.round(a / step) * step, -6, 6) * s).reshape(y.shape)


def exact(case, seed):
    if case["op"] == "prompt" and _plain_cost(case) > 2 ** 33:
        return None
    st = prepare(case, seed)
    if case["op"] == "heads":
        pairs = case["rotary"] // 2
        at = st["positions"].double().reshape(case["axes"], -1)
        turn = torch.cat([at[i // pairs if case["axes"] == 1 else next(a for a in range(3) if i < sum(st["sections"][:a + 1]))][:, None]
                          * math.pow(_BASE, -i / pairs) for i in range(pairs)], dim=1)
        turn = torch.polar(torch.ones_like(turn), turn)[:, None]

        def one(x, weight):
            x = x.double()
            y = x / torch.sqrt(torch.mean(x ** 2, dim=-1, keepdim=True) + _EPS) * weight.double()
            first, second = (slice(0, case["rotary"], 2), slice(1, case["rotary"], 2)) if case["pairs"] else (slice(0, pairs), slice(pairs, case["rotary"]))
            z = torch.complex(y[..., first], y[..., second]) * turn
            y[..., first], y[..., second] = z.real, z.imag
            return y

        q, k = one(st["q"], st["q_weight"]), one(st["k"], st["k_weight"])
        if case["form"] == "none":
            return [q, k]
        out = [q]
        for y, cache in ((k, st["k_cache"]), (st["v"].double(), st["v_cache"])):  # the values before they are rounded to eight bits
            scale = _exact_scale(y)
            held, scales = cache[0].double(), cache[1].double()
            page, place = st["slots"] // case["page"], st["slots"] % case["page"]
            held[page, :, place], scales[page, :, place] = y / scale[..., None], scale
            out += [held, scales]
        return out
    if case["op"] == "cache":
        out = []
        rows = torch.cat([st["table"][i].long().repeat_interleave(case["page"])[:n] * case["page"] + torch.arange(n, device="cuda") % case["page"]
                          for i, n in enumerate(_lengths(case))])
        for name, unit in (("k", _K_UNIT), ("v", _V_UNIT)):
            all_rows = _exact_held(st[name + "_cache"], case["form"], unit).transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"])
            all_rows[st["slots"]] = _exact_written(st[name].double(), case["form"], unit)
            out.append(all_rows[rows])
        return out
    scale = 1 / math.sqrt(case["dim"])
    if case["op"] == "decode":
        k, v = (_exact_held(st[n], case["form"], u) for n, u in (("k_cache", _K_UNIT), ("v_cache", _V_UNIT)))
        y = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
        group = case["q_heads"] // case["kv_heads"]
        for i, n in enumerate(_lengths(case)):
            mine = st["table"][i].long()
            ki, vi = (t[mine].transpose(0, 1).reshape(case["kv_heads"], -1, case["dim"])[:, :n] for t in (k, v))
            for t in range(case["tokens"]):
                sees = n - case["tokens"] + 1 + t
                if sees > 0:
                    qt = st["q"][i, t].double().view(case["kv_heads"], group, -1)
                    y[i, t] = (torch.softmax(torch.einsum("hgd,hnd->hgn", qt, ki[:, :sees]) * scale, dim=-1) @ vi[:, :sees]).reshape(case["q_heads"], -1)
        return [y]
    y = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    a = b = 0
    for n in _lengths(case):
        m = n + case["prefix"]
        hidden = torch.ones(n, m, dtype=torch.bool, device="cuda").triu(case["prefix"] + 1)
        for h in range(case["q_heads"]):
            of = h // (case["q_heads"] // case["kv_heads"])
            s = torch.mm(st["q"][a:a + n, h].double(), st["k"][b:b + m, of].double().t()) * scale
            if case["causal"]:
                s[hidden] = -math.inf
            y[a:a + n, h] = torch.mm(torch.softmax(s, dim=-1), st["v"][b:b + m, of].double())
        a, b = a + n, b + m
    return [y]


def work(case):
    op, dim, kv_heads = case["op"], case["dim"], case["kv_heads"]
    row = {"e4m3": dim + 4, "nvfp4": dim * 9 // 16}.get(case.get("form"), 0) * kv_heads  # a token's keys, or values, in the cache
    if op == "heads":
        q = case["tokens"] * case["q_heads"] * dim * 2
        k = case["tokens"] * kv_heads * dim * 2
        fixed = 4 * dim + 8 * case["axes"] * case["tokens"]
        return {"bytes": 2 * q + fixed + (2 * k if case["form"] == "none" else 2 * k + case["tokens"] * (8 + 2 * row)), "flops": 0}
    lengths = _lengths(case)
    if op == "cache":
        new = sum(min(n, case["tokens"]) for n in lengths)
        pages = sum(-(-n // case["page"]) for n in lengths)
        return {"bytes": 2 * new * (kv_heads * dim * 2 + row + 4) + 2 * sum(lengths) * (row + kv_heads * dim * 2) + 4 * pages, "flops": 0}
    if op == "decode":
        pages = sum(-(-n // case["page"]) for n in lengths)
        seen = sum(max(0, n - t) for n in lengths for t in range(case["tokens"]))
        return {"bytes": 2 * sum(lengths) * row + 4 * pages + 4 * len(lengths) + 4 * case["seqs"] * case["tokens"] * case["q_heads"] * dim,
                "flops": 4 * seen * case["q_heads"] * dim}
    seen = sum(n * (n + 1) // 2 + n * case["prefix"] if case["causal"] else n * (n + case["prefix"]) for n in lengths)
    keys = sum(lengths) + len(lengths) * case["prefix"]
    return {"bytes": 4 * sum(lengths) * case["q_heads"] * dim + 4 * keys * kv_heads * dim + 8 * (len(lengths) + 1), "flops": 4 * seen * case["q_heads"] * dim}
