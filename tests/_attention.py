"""What the tests of heads, caches and attention share: caches in plain layout, and the formulas in 64 bits."""
import torch

from qwen38_flash_ops_b200 import KvCache

E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
FORMS = {"nvfp4": torch.uint8, "e4m3": torch.float8_e4m3fn}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2  # the most that a rounding is off, relative to the value


def new_cache(form, pages, heads, dim, page=32, k_unit=0.25, v_unit=0.0625):
    return KvCache(pages, heads, dim, page, FORMS[form], k_unit, v_unit)


def held(codes, scale, unit):
    """What a cache's rows stand for, in 64 bits on the host: [pages, heads, page, dim]."""
    codes, scale = codes.cpu(), scale.cpu()
    if codes.dtype == torch.float8_e4m3fn:
        return codes.double() * scale.double()[..., None]
    nibbles = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).long()
    value = E2M1[nibbles & 7] * torch.where(nibbles > 7, -1.0, 1.0)
    return value * scale.double().repeat_interleave(16, dim=-1) * unit


def quantised(y, form, unit):
    """64-bit rows [..., dim] -> (codes as a cache holds them, scales), by the definition."""
    if form == "e4m3":
        most = y.abs().amax(-1, keepdim=True)
        q = torch.where(most / 448 < 2.0 ** -40, y * 2.0 ** 40, y * 448 / most)
        return q.nan_to_num(0).float().to(torch.float8_e4m3fn), (most[..., 0] / 448).float().clamp(min=2.0 ** -40)
    blocks = y.unflatten(-1, (-1, 16))
    scale = (blocks.abs().amax(-1) / (6 * unit)).float().clamp(max=448.0).to(torch.float8_e4m3fn).double().clamp(min=2.0 ** -9)
    a = (blocks / (scale * unit)[..., None]).clamp(-6, 6)
    step = torch.where(a.abs() < 2, 0.5, torch.where(a.abs() < 4, 1.0, 2.0)).double()
    size = (a / step).round().abs() * step  # half-way values go to the even code: codes are steps of 0.5 up to 2, of 1 up to 4, of 2
    code = torch.searchsorted(E2M1, size) + torch.where(torch.signbit(a), 8, 0)
    code = code.flatten(-2).to(torch.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4, scale.float().to(torch.float8_e4m3fn)


def same_bits(a, b):
    a, b = a.cpu().contiguous(), b.cpu().contiguous()
    if a.element_size() == 1:
        return torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    return torch.equal(a, b)


def same_codes(a, b, form):
    """The same values, code by code: the sign of a zero says nothing."""
    a, b = a.cpu().contiguous(), b.cpu().contiguous()
    if form == "nvfp4":
        a, b = (torch.stack([t & 15, t >> 4]) for t in (a, b))
        return torch.equal(torch.where(a == 8, 0, a), torch.where(b == 8, 0, b))
    return torch.equal(torch.where(a == 128, 0, a), torch.where(b == 128, 0, b))


def fill(cache, gen, spread=0.5):
    """Random keys and values in every row of a cache, quantised by the definition."""
    form = "nvfp4" if cache.dtype == torch.uint8 else "e4m3"
    for codes, scale, unit in ((cache.k, cache.k_scale, cache.k_unit), (cache.v, cache.v_scale, cache.v_unit)):
        rows = torch.randn(cache.pages, cache.kv_heads, cache.page, cache.head_dim, generator=gen, dtype=torch.float64)
        rows *= torch.exp(spread * torch.randn(cache.kv_heads, 1, cache.head_dim, generator=gen, dtype=torch.float64))
        c, s = quantised(rows, form, unit)
        codes.view(torch.uint8).copy_(c.view(torch.uint8))
        (scale.view(torch.uint8) if scale.element_size() == 1 else scale).copy_(s.view(torch.uint8) if s.element_size() == 1 else s)


def attention(q, k, v, seen, scale):
    """q [rows, dim], k and v [keys, dim] in 64 bits, seen [rows]: how many of the keys each row sees.  (y, sum of |weight v|, log of the sum of exponentials)"""
    s = (q @ k.t()) * scale
    s = s.masked_fill(torch.arange(k.shape[0])[None] >= seen[:, None], -float("inf"))
    lse = torch.logsumexp(s, -1) if k.shape[0] else torch.full((q.shape[0],), -float("inf"), dtype=torch.float64)
    w = torch.where(torch.isinf(lse)[:, None], 0.0, torch.exp(s - torch.where(torch.isinf(lse), 0.0, lse)[:, None]))
    return w @ v, w @ v.abs(), lse
