"""QuantGemm at the inner dimensions of the workloads, to FP32, with scales of one: what the sums themselves are.

INT8: the exact integer, rounded to FP32 once.

E4M3: an instruction adds 32 products to the sum so far.  Measured, and taken as the rule here: the 33 addends are cut off at 2^-25 of the largest one's power of two,
and the new sum to 24 bits, toward zero.  With S_j the exact sum behind step j and P_j the sum of the step's magnitudes, a step is off by at most
(2^-23 + 33 2^-25) max(|S_j-1|, |S_j|, P_j); the ranks that share K begin at zero each, and their sums are added in FP32."""
import pytest
import torch

from qwen38_flash_ops_b200 import QuantGemm

pytestmark = pytest.mark.gpu
_STEP = 2.0 ** -23 + 33 * 2.0 ** -25


def _inputs(dtype, m, k, n, order, positive):
    gen = torch.Generator(device="cuda").manual_seed(m + k + n)
    if dtype == torch.int8:
        make = lambda *s: torch.randint(0 if positive else -128, 128, s, generator=gen, device="cuda", dtype=torch.int16).to(torch.int8)
    else:
        def make(*s):
            v = torch.randn(*s, generator=gen, device="cuda") * 3
            return (v.abs() if positive else v).to(torch.float8_e4m3fn)
    x, w = make(m, k), make(n, k)
    return x, (w.t() if order == "k" else w.t().contiguous())


def _call(x, w, plan):
    op = QuantGemm(out_dtype=torch.float32)
    op.set_option("plan", plan)
    return op(x, torch.ones(x.shape[0], device="cuda"), w)


@pytest.mark.parametrize("positive", [False, True])
@pytest.mark.parametrize("m,k,n,order,plan", [(1, 5120, 5120, "n", ""), (8, 5120, 10240, "k", ""), (64, 17408, 5120, "k", ""), (509, 5120, 10240, "n", ""),
                                              (300, 17408, 1280, "n", "256,1,1,1"), (8, 17408, 5120, "n", "16,8,0,1"), (77, 17407, 1283, "n", "")])
def test_int8_sums_are_exact(cuda, m, k, n, order, plan, positive):
    x, w = _inputs(torch.int8, m, k, n, order, positive)
    assert torch.equal(_call(x, w, plan), (x.double() @ w.double()).float())


@pytest.mark.parametrize("positive", [False, True])
@pytest.mark.parametrize("m,k,n,order,plan", [(1, 5120, 5120, "n", "16,1,0,2"), (1, 5120, 5120, "n", "16,3,0,2"), (8, 5120, 10240, "k", "16,1,0,2"),
                                              (64, 17408, 1280, "k", "64,1,0,1"), (64, 17408, 1280, "k", "64,3,0,1"), (64, 17408, 1280, "n", "64,8,0,1"),
                                              (200, 17408, 640, "n", "224,1,1,1"), (77, 17407, 643, "n", "80,1,0,1"), (77, 17407, 643, "k", "80,4,0,1")])
def test_e4m3_sums(cuda, m, k, n, order, plan, positive):
    x, w = _inputs(torch.float8_e4m3fn, m, k, n, order, positive)
    got = _call(x, w, plan).double()
    xd, wd, ranks, blocks = x.double(), w.double(), int(plan.split(",")[1]), (k + 127) // 128
    total, tol = torch.zeros(m, n, dtype=torch.float64, device="cuda"), torch.zeros(m, n, dtype=torch.float64, device="cuda")
    for rank in range(ranks):
        sum_ = torch.zeros_like(total)
        for k0 in range(rank * blocks // ranks * 128, min(k, (rank + 1) * blocks // ranks * 128), 32):
            a, b = xd[:, k0:k0 + 32], wd[k0:k0 + 32]
            new = sum_ + a @ b
            tol += _STEP * torch.maximum(torch.maximum(sum_.abs(), new.abs()), a.abs() @ b.abs())
            sum_ = new
        total += sum_
        tol += 2.0 ** -23 * total.abs()
    assert ((got - total).abs() <= tol).all(), ((got - total).abs() / tol).max().item()
    # of a cut toward zero half an ulp, at most 2^-24, is lost on average, by a sum that grows evenly from zero: 544 / 2 steps of 2^-24, 2^-15.9 of it
    assert ((got - total).norm() <= 2.0 ** -15.9 * total.norm())
