"""Attention's backward pass at every head_dim, within the bounds of test_gpu_attn_bwd.py."""
import pytest

import test_gpu_attn_bwd as base

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", range(8, 129, 8))
@pytest.mark.parametrize("layout,cus", [("bhsd", 0), ("bshd", 4096)])
def test_every_head_dim(gpu, dtype, D, layout, cus, monkeypatch):
    monkeypatch.setitem(base.ops.TUNING, "cu_count", cus)
    t = base.inputs(gpu, 1, 2, 150, 131, D, 37, dtype, layout)
    base.close(base.call(*t), *base.bounds(*t))
    q, k, v, k2, v2, dout, out, lse = t
    framed = [base.framed(x)[0] for x in (q, k, v, k2, v2, dout, out)]   # NaN beside the tensors' columns
    base.close(base.call(*framed, lse), *base.bounds(*t))
