"""QuantMlp: its types, and what a refused call leaves behind."""
import pytest
import torch

from qwen38_flash_ops_b200 import QfgError, QuantGemm, QuantMlp, RmsNormQuant, RowQuant, _lib, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("change", [
    dict(ldw1=255), dict(ldw2=63), dict(order1=2), dict(order2=2), dict(w1=None), dict(w2=None), dict(weight=None), dict(h=None), dict(ldx=63),
    dict(q_dtype=_lib.QFG_UINT8), dict(up_plan="64,2,1,1"), dict(down_plan="15,1,0,1"), dict(up_scales=255), dict(down_scales=63),
], ids=lambda c: "-".join(c))
def test_a_refused_block_writes_nothing(cuda, change):
    """The residual stream is updated where it lies, so that a call refused half way would add x to it a second time when it is made again."""
    lib = _lib.load()
    rows, hidden, width = 3, 64, 128
    up, down = (QuantGemm(w_scale=[1.0] * change.get(k, n)) for k, n in (("up_scales", 2 * width), ("down_scales", hidden)))
    for op, plan in ((up, change.get("up_plan")), (down, change.get("down_plan"))):
        if plan:
            op.set_option("plan", plan)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, stream = (torch.randn(rows, hidden, generator=gen, device="cuda").bfloat16() for _ in range(2))
    weight, y = torch.ones(hidden, device="cuda").bfloat16(), torch.full((rows, hidden), 7.0, device="cuda").bfloat16()
    w1, w2 = torch.ones(hidden, 2 * width, dtype=torch.int8, device="cuda"), torch.ones(width, hidden, dtype=torch.int8, device="cuda")
    workspace = torch.zeros(lib.qfg_quant_mlp_workspace_bytes(up._p, rows, hidden, width), dtype=torch.uint8, device="cuda")
    a = dict(dtype=_lib.QFG_BFLOAT16, x=x.data_ptr(), ldx=hidden, residual=stream.data_ptr(), ldr=hidden, weight=weight.data_ptr(), weight_dtype=_lib.QFG_BFLOAT16,
             offset=0.0, eps=1e-6, rows=rows, hidden=hidden, width=width, q_dtype=_lib.QFG_INT8, up=up._p, w1=w1.data_ptr(), ldw1=2 * width, order1=0, down=down._p,
             w2=w2.data_ptr(), ldw2=hidden, order2=0, workspace=workspace.data_ptr(), y=y.data_ptr(), h=stream.data_ptr(),
             stream=torch.cuda.current_stream().cuda_stream)
    a.update({k: v for k, v in change.items() if k in a})
    before, kept = stream.clone(), workspace.clone()
    torch.cuda.synchronize()
    assert lib.qfg_quant_mlp(*a.values()) != _lib.QFG_OK
    torch.cuda.synchronize()
    assert torch.equal(stream, before) and (y == 7.0).all() and torch.equal(workspace, kept)


@pytest.mark.parametrize("eight", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,hidden,width", [(1, 256, 512), (7, 640, 264), (300, 512, 384), (5, 129, 77)])
def test_types(cuda, monkeypatch, eight, dtype, out_dtype, rows, hidden, width):
    """Rows and outputs of every type, against the four calls, and against the definition with the bounds of test_mlp: what eight bits move."""
    gen = torch.Generator(device="cuda").manual_seed(rows + hidden)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    top = 127.0 if eight == torch.int8 else 448.0

    def quantised(k, n):
        w = rand(k, n) * 0.05
        s = w.abs().amax(0) / top
        q = w / s
        return (q.round() if eight == torch.int8 else q).to(eight), s

    (q1, s1), (q2, s2) = quantised(hidden, 2 * width), quantised(width, hidden)
    g, x, r = (1 + 0.2 * rand(hidden)).to(dtype), rand(rows, hidden).to(dtype), rand(rows, hidden).to(dtype)
    mlp = QuantMlp(g, q1, s1.cpu().numpy(), q2, s2.cpu().numpy(), out_dtype=out_dtype)
    y, h = mlp(x, r)
    assert y.dtype == out_dtype and h.dtype == dtype and y.shape == h.shape == x.shape
    q, scale, h4 = RmsNormQuant(dtype=eight)(x, g, r)
    both = QuantGemm(w_scale=s1.cpu().numpy(), out_dtype=out_dtype)(q, scale, q1)
    q, scale = RowQuant(dtype=eight)(both[:, :width], both[:, width:])
    assert torch.equal(y, QuantGemm(w_scale=s2.cpu().numpy(), out_dtype=out_dtype)(q, scale, q2)) and torch.equal(h, h4)
    d = (x + r).double()
    both = d / torch.sqrt((d * d).mean(-1, keepdim=True) + 1e-6) * g.double() @ (q1.double() * s1.double())
    a, b = both[:, :width], both[:, width:]
    want = (a * torch.sigmoid(a) * b) @ (q2.double() * s2.double())
    assert ((y.double() - want).norm() / want.norm()).item() < (0.03 if eight == torch.int8 else 0.12)
    monkeypatch.setattr(ops._calls, "quant_mlp", lambda *args: None)  # the way through Python
    assert all(torch.equal(a, b) for a, b in zip(mlp(x, r), (y, h)))


def test_the_type_of_outputs_is_checked(cuda):
    w1, w2 = torch.zeros(64, 96, dtype=torch.int8, device="cuda"), torch.zeros(48, 64, dtype=torch.int8, device="cuda")
    with pytest.raises(QfgError, match="out_dtype"):
        QuantMlp(torch.ones(64, device="cuda"), w1, None, w2, None, out_dtype=torch.int8)
