"""Gradients of keys and values alone, in launches that have whole tiles beside tiles in parts, within the bounds of test_gpu_attn_bwd.py."""
import pytest
import torch

import test_gpu_attn_bwd as base
from train_host import KEYS_ONLY

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", KEYS_ONLY)
def test_whole_tiles_beside_parts(gpu, kw, monkeypatch):
    monkeypatch.setitem(base.ops.TUNING, "cu_count", kw["cus"])
    t = base.inputs(gpu, 1, kw["H"], kw["Sq"], kw["Sk"], kw["D"], kw["Sk2"], kw["dtype"], "bshd")
    got = base.call(*t, need_q=False)
    want, far = base.bounds(*t)
    assert got[0] is None
    base.close(got[1:], want[1:], far[1:])
    results = [base.framed(torch.zeros_like(x)) for x in (t[1], t[2]) + ((t[3], t[4]) if kw["Sk2"] else ())]
    again = base.call(*t, need_q=False, **{n: r[0] for n, r in zip(("dk", "dv", "dk2", "dv2"), results)})
    for a, b, (inner, big) in zip(got[1:], again[1:], results):
        assert torch.equal(a, b) and b is inner and int(big.isnan().sum()) == big.numel() - inner.numel()
