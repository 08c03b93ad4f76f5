"""An MLP block in eight bits, made of the package's operators: norm with the residual's addition, gate and up projection, gated
activation, down projection.

    python -m qwen38_flash_ops_b200.quant_mlp [--rows 8] [--hidden 5120] [--width 17408] [--dtype int8]

makes one of random weights, compares it with the same block on unquantised weights, and times it.
"""
from __future__ import annotations

import torch

from . import ops
from .ops import QuantGemm, RmsNormQuant, RowQuant, check


class QuantMlp:
    """(y, h) = mlp(x, residual): h = x + residual is the residual stream that goes on, y = down(swish(gate) * up) of its norm.

    `gate_up` [hidden, 2 * width] holds gate's columns, then up's, and `down` [width, hidden]; both torch.int8 or both
    torch.float8_e4m3fn, either dimension contiguous, with a scale per column.  Between the products the rows are quantised to the
    same type.  The four calls follow one another on the current stream and allocate their outputs as torch does.

    x and residual are BF16, FP16 or FP32, and h is of their type.  `out_dtype` (BF16 unless given, FP16 or FP32) is the type of y, and of gate and up
    between the products.

    Work that other threads put on that stream during a call must not write the weights: a product may fetch its first ones before the calls
    ahead of it have ended."""

    def __init__(self, norm_weight, gate_up, gate_up_scale, down, down_scale, eps: float = 1e-6, weight_offset: float = 0.0,
                 out_dtype: torch.dtype = torch.bfloat16):
        if gate_up.dtype != down.dtype or gate_up.shape[1] != 2 * down.shape[0] or gate_up.shape[0] != down.shape[1]:
            raise ValueError("QuantMlp: gate_up is [hidden, 2 * width] and down [width, hidden], of one type")
        self.width = down.shape[0]
        self.norm_weight, self.gate_up, self.down = norm_weight, gate_up, down
        self._norm = RmsNormQuant(eps=eps, weight_offset=weight_offset, dtype=gate_up.dtype)
        self._act = RowQuant(dtype=gate_up.dtype)
        self._gate_up = QuantGemm(w_scale=gate_up_scale, out_dtype=out_dtype)
        self._down = QuantGemm(w_scale=down_scale, out_dtype=out_dtype)

    def __call__(self, x: torch.Tensor, residual: torch.Tensor):
        r = ops._calls.quant_mlp(self._norm.eps, self._norm.weight_offset, self.norm_weight, self._gate_up._p, self.gate_up, self._down._p, self.down,
                                 self._down._code, x, residual)
        if r is not None:
            return r if r.__class__ is tuple else check(r)
        q, scale, h = self._norm(x, self.norm_weight, residual)
        both = self._gate_up(q, scale, self.gate_up)
        q, scale = self._act(both[..., :self.width], both[..., self.width:])
        return self._down(q, scale, self.down), h


def main() -> None:
    import argparse

    from .packing_torch import quantize_fp8_per_column_torch, quantize_int8_per_column_torch

    p = argparse.ArgumentParser(description="an MLP block in eight bits against its unquantised form")
    p.add_argument("--rows", type=int, default=8)
    p.add_argument("--hidden", type=int, default=5120)
    p.add_argument("--width", type=int, default=17408)
    p.add_argument("--dtype", choices=("int8", "e4m3"), default="int8")
    a = p.parse_args()
    gen = torch.Generator(device="cuda").manual_seed(0)
    randn = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    quantise = quantize_int8_per_column_torch if a.dtype == "int8" else quantize_fp8_per_column_torch
    w1, w2, g = randn(a.hidden, 2 * a.width) * 0.02, randn(a.width, a.hidden) * 0.02, 1 + 0.2 * randn(a.hidden)
    (q1, s1), (q2, s2) = quantise(w1), quantise(w2)
    mlp = QuantMlp(g.bfloat16(), q1, s1.cpu().numpy(), q2, s2.cpu().numpy())
    x, residual = randn(a.rows, a.hidden).bfloat16(), (4 * randn(a.rows, a.hidden)).bfloat16()
    y, h = mlp(x, residual)
    f = (x + residual).float()
    both = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + 1e-6) * g.bfloat16().float() @ w1
    want = torch.nn.functional.silu(both[:, :a.width]) * both[:, a.width:] @ w2
    print(f"relative difference from the unquantised block: {((y.float() - want).norm() / want.norm()).item():.4f}")
    for _ in range(3):
        mlp(x, residual)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(50):
        mlp(x, residual)
    end.record()
    torch.cuda.synchronize()
    print(f"{start.elapsed_time(end) / 50 * 1e3:.1f} us a call, {a.rows} rows, {a.hidden} x {a.width}, {a.dtype}")


if __name__ == "__main__":
    main()
