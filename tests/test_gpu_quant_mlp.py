"""QuantMlp: what a refused call leaves behind."""
import pytest
import torch

from qwen38_flash_ops_b200 import QuantGemm, _lib

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
