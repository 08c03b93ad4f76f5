"""The operators of an eight-bit block, for timing and comparison: the norm and the activation that write eight-bit rows with
a scale each, the product of such rows with an eight-bit weight, and an MLP made of them.

Shapes are those of the package's workloads, tests and benchmark (a K = 5120 model: attention outputs 5120, q / k / v 10240,
gate and up 34816, down 17408 -> 5120), and ragged ones.  Activations have channels of very different size, as a model's do;
weights are N(0, 0.02^2), quantised per column.  A case is a dict:

  op        norm | act | gemm | mlp
  dtype     e4m3 | int8: the eight-bit type.  The cases that return eight-bit rows use e4m3, whose tensors hold the values
            themselves; int8 rows are what the products and the MLP are made of.
  rows, k   rows, and their length (gemm, mlp: the inner dimension of the product)
  n         gemm: output columns; mlp: the width of the gated layer
  source    norm, act: the type of the input, bf16 | f16 | f32
  residual  norm: a residual stream is added first, and returned
  gated     act: swish(x) * u, else x alone
  order     gemm, mlp: the weight is stored with its columns ("n") or its inner dimension ("k") contiguous
"""
import torch

own = False

_EIGHT = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}
_SOURCE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_EPS = 1e-6
_TINY = 2.0 ** -100  # a row's largest value counts as no smaller than this, so that a scale is never zero


def _norm(name, rows, k, source="bf16", residual=True, dtype="e4m3"):
    c = {"op": "norm", "dtype": dtype, "rows": rows, "k": k, "source": source, "residual": residual}
    return {"name": name, **c} if name else c


def _act(name, rows, k, source="bf16", gated=True, dtype="e4m3"):
    c = {"op": "act", "dtype": dtype, "rows": rows, "k": k, "source": source, "gated": gated}
    return {"name": name, **c} if name else c


def _gemm(name, dtype, rows, k, n, order, op="gemm"):
    c = {"op": op, "dtype": dtype, "rows": rows, "k": k, "n": n, "order": order}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one decoded token: the norm ahead of a block, with the residual stream
        _norm("decode_norm", 1, 5120),
        # a prompt chunk
        _norm("prefill_norm", 4096, 5120),
        # rows of an odd length that begin off every vector boundary, no residual, another type
        _norm("odd_norm_f16", 333, 2561, "f16", False),
        # four speculated tokens: the gated activation between an MLP's products
        _act("decode_act", 4, 17408),
        # a prompt chunk of it
        _act("prefill_act", 2048, 17408),
        # one decoded token: attention's output projection, the smallest product
        _gemm("decode_o_proj_int8", "int8", 1, 5120, 5120, "n"),
        # eight speculated tokens: q, k and v as one weight, stored the way checkpoints store it
        _gemm("decode_qkv_e4m3", "e4m3", 8, 5120, 10240, "k"),
        # a batch of sequences decoded together: the MLP's down projection
        _gemm("batch_down_int8", "int8", 64, 17408, 5120, "k"),
        # odd in every size: neither operand's rows begin on a vector boundary
        _gemm("odd_int8", "int8", 77, 2561, 5117, "n"),
        # the ragged tail of a prompt
        _gemm("tail_qkv_e4m3", "e4m3", 509, 5120, 10240, "n"),
        # a prompt chunk: gate and up, the largest
        _gemm("prefill_gate_up_int8", "int8", 4096, 5120, 34816, "k"),
        # a whole MLP block over eight decoded tokens: norm, product, gated activation, product
        _gemm("decode_mlp_int8", "int8", 8, 5120, 17408, "n", op="mlp"),
    ]


def _log_int(rng, lo, hi, step=1):
    v = lo * (hi / lo) ** rng.random()
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    most = {m: max(work(c)[m] for c in listed()) for m in ("bytes", "flops")}
    while True:
        op = rng.choice(["norm"] * 3 + ["act"] * 2 + ["gemm"] * 6 + ["mlp"])
        rows = rng.choice([rng.randint(1, 16), _log_int(rng, 1, 8192)])
        step = rng.choice([1, 16, 128])
        k = _log_int(rng, 128, 17408, step)
        if op == "norm":
            c = _norm(None, rows, k, rng.choice(["bf16", "bf16", "f16", "f32"]), rng.random() < 0.6)
        elif op == "act":
            c = _act(None, rows, k, rng.choice(["bf16", "bf16", "f16", "f32"]), rng.random() < 0.7)
        elif op == "gemm":
            c = _gemm(None, rng.choice(["int8", "e4m3"]), rows, k, _log_int(rng, 128, 34816, step), rng.choice(["n", "k"]))
        else:
            c = _gemm(None, rng.choice(["int8", "e4m3"]), min(rows, 512), k, _log_int(rng, 128, 17408, max(step, 8)), rng.choice(["n", "k"]), op="mlp")
        w = work(c)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
            return c


# ------------------------------------------------------------------------------ inputs
def _activations(gen, rows, k, spread):
    """Rows whose channels differ in size, as behind a transformer's layers: a few are many times the ordinary ones."""
    channel = torch.exp(spread * torch.randn(k, generator=gen, device="cuda"))
    return torch.randn(rows, k, generator=gen, device="cuda") * channel


def _quantised_rows(v, dtype):
    """Eight-bit values and the scale of each row."""
    eight, top = _EIGHT[dtype]
    scale = v.abs().amax(dim=-1).clamp(min=1e-8) / top
    v = v / scale[:, None]
    return (v.round() if dtype == "int8" else v.clamp(-top, top)).to(eight), scale


def _weight(gen, dtype, k, n, order):
    """An eight-bit weight [k, n], and the scale of each column."""
    q, scale = _quantised_rows(torch.randn(n, k, generator=gen, device="cuda") * 0.02, dtype)
    return q.t() if order == "k" else q.t().contiguous(), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 1000 + 29)
    op, dtype, rows, k = case["op"], case["dtype"], case["rows"], case["k"]
    st = {"op": op, "dtype": dtype}
    if op == "norm":
        source = _SOURCE[case["source"]]
        st["x"] = _activations(gen, rows, k, 0.5).to(source)
        st["weight"] = (1 + 0.2 * torch.randn(k, generator=gen, device="cuda")).to(source)
        st["residual"] = (4 * _activations(gen, rows, k, 0.7)).to(source) if case["residual"] else None
    elif op == "act":
        source = _SOURCE[case["source"]]
        st["x"] = _activations(gen, rows, k, 0.5).to(source)
        st["u"] = _activations(gen, rows, k, 0.5).to(source) if case["gated"] else None
    elif op == "gemm":
        st["x"], st["x_scale"] = _quantised_rows(_activations(gen, rows, k, 0.5), dtype)
        st["w"], st["w_scale"] = _weight(gen, dtype, k, case["n"], case["order"])
    else:
        st["x"] = _activations(gen, rows, k, 0.5).bfloat16()
        st["residual"] = (4 * _activations(gen, rows, k, 0.7)).bfloat16()
        st["weight"] = (1 + 0.2 * torch.randn(k, generator=gen, device="cuda")).bfloat16()
        st["up"] = _weight(gen, dtype, k, 2 * case["n"], case["order"])  # gate's columns, then up's
        st["down"] = _weight(gen, dtype, case["n"], k, case["order"])
    if own:  # the nodes that a program makes once, with its weights' scales
        from qwen38_flash_ops_b200 import QuantGemm, QuantMlp, RmsNormQuant, RowQuant

        eight = _EIGHT[dtype][0]
        if op == "norm":
            st["node"] = RmsNormQuant(eps=_EPS, dtype=eight)
        elif op == "act":
            st["node"] = RowQuant(dtype=eight)
        elif op == "gemm":
            st["node"] = QuantGemm(w_scale=st["w_scale"].cpu().numpy())
        else:
            st["node"] = QuantMlp(st["weight"], st["up"][0], st["up"][1].cpu().numpy(), st["down"][0], st["down"][1].cpu().numpy(), eps=_EPS)
    return st


# ------------------------------------------------------------------------------ plain forms
def _plain_rows(y, dtype):
    """FP32 rows -> the eight-bit values (as FP32) and the scale of each row."""
    top = _EIGHT[dtype][1]
    scale = y.abs().amax(dim=-1).clamp(min=_TINY) / top
    y = y / scale[:, None]
    return (y.round() if dtype == "int8" else y.clamp(-top, top).to(torch.float8_e4m3fn).float()), scale


def _plain_norm(x, weight, residual, dtype):
    """Root-mean-square norm of x + residual, which is rounded to its own type first: it is the stream that goes on."""
    h = x
    if residual is not None:
        h = (x.float() + residual.float()).to(x.dtype)
    f = h.float()
    y = f * torch.rsqrt((f * f).mean(dim=-1, keepdim=True) + _EPS) * weight.float()
    return (*_plain_rows(y, dtype), h)


def _plain_act(g, u, dtype):
    g = g.float()
    return _plain_rows(g if u is None else g / (1 + torch.exp(-g)) * u.float(), dtype)


def _plain_gemm(q, x_scale, w, w_scale):
    return ((q.float() @ w.float()) * x_scale[:, None] * w_scale).bfloat16()


def _run_plain(st):
    op, dtype = st["op"], st["dtype"]
    if op == "norm":
        q, scale, h = _plain_norm(st["x"], st["weight"], st["residual"], dtype)
        return [q.to(torch.float8_e4m3fn), scale] + ([] if st["residual"] is None else [h])
    if op == "act":
        q, scale = _plain_act(st["x"], st["u"], dtype)
        return [q.to(torch.float8_e4m3fn), scale]
    if op == "gemm":
        return [_plain_gemm(st["x"], st["x_scale"], st["w"], st["w_scale"])]
    q, scale, h = _plain_norm(st["x"], st["weight"], st["residual"], dtype)
    up = _plain_gemm(q, scale, *st["up"])
    half = up.shape[1] // 2
    q, scale = _plain_act(up[:, :half], up[:, half:], dtype)
    return [_plain_gemm(q, scale, *st["down"]), h]


def run(st):
    if not own:
        return _run_plain(st)
    node = st["node"]
    if st["op"] == "norm":
        return list(node(st["x"], st["weight"], st["residual"]))
    if st["op"] == "act":
        return list(node(st["x"], st["u"]))
    if st["op"] == "gemm":
        return [node(st["x"], st["x_scale"], st["w"])]
    return list(node(st["x"], st["residual"]))


# ------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    top = _EIGHT[case["dtype"]][1]

    def scales(y):
        return torch.maximum(y.abs().max(dim=-1).values, torch.tensor(_TINY, dtype=torch.float64, device=y.device)) / top

    def rounded(v):  # the values that eight bits hold, of a result in 64 bits
        return v.round() if case["dtype"] == "int8" else v.float().clamp(-top, top).to(torch.float8_e4m3fn).double()

    def normed(x, residual):
        h = x.double() if residual is None else x.double() + residual.double()
        kept = h if residual is None else h.to(x.dtype).double()  # the norm is defined on the stream as it is kept
        root = torch.sqrt(torch.mean(kept ** 2, dim=-1, keepdim=True) + _EPS)
        return kept / root * st["weight"].double(), h

    def gated(g, u):
        return g if u is None else g * torch.sigmoid(g) * u

    def product(q, scale, w, w_scale):
        return torch.mm(q, w.double()) * torch.outer(scale, w_scale.double())

    if case["op"] == "gemm":
        return [product(st["x"].double(), st["x_scale"].double(), st["w"], st["w_scale"])]
    # eight-bit rows: the values before they are rounded to eight bits
    if case["op"] == "norm":
        y, h = normed(st["x"], st["residual"])
        s = scales(y)
        return [y / s[:, None], s] + ([] if st["residual"] is None else [h])
    if case["op"] == "act":
        y = gated(st["x"].double(), None if st["u"] is None else st["u"].double())
        s = scales(y)
        return [y / s[:, None], s]
    y, h = normed(st["x"], st["residual"])
    s = scales(y)
    up = product(rounded(y / s[:, None]), s, *st["up"]).bfloat16().double()  # the first product's own output type
    y = gated(up[:, :case["n"]], up[:, case["n"]:])
    s = scales(y)
    return [product(rounded(y / s[:, None]), s, *st["down"]), h]


def work(case):
    op, rows, k = case["op"], case["rows"], case["k"]
    if op == "norm":
        size = 4 if case["source"] == "f32" else 2
        return {"bytes": rows * k * (size * (3 if case["residual"] else 1) + 1) + size * k + 4 * rows, "flops": 0}
    if op == "act":
        size = 4 if case["source"] == "f32" else 2
        return {"bytes": rows * k * (size * (2 if case["gated"] else 1) + 1) + 4 * rows, "flops": 0}
    n = case["n"]
    if op == "gemm":
        return {"bytes": rows * (k + 4 + 2 * n) + k * n + 4 * n, "flops": 2 * rows * k * n}
    # activations in and out (y and the residual stream), both weights with their scales, the norm's weight
    return {"bytes": rows * k * 8 + 3 * k * n + 4 * (2 * n + k) + 2 * k, "flops": 2 * rows * k * 3 * n}
