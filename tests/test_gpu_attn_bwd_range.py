"""Attention's backward pass where rows differ in size, and where some are not finite.

Bars are those of test_gpu_attn_bwd.py.  fp16's probabilities are rounded times 2^15 and its numbers end at 2^-24: those below 2^-29 are off by up to 2^-40, which
moves a gradient of v by at most 2^-40 of its head's sizes of dout."""
import math

import pytest
import torch

import test_gpu_attn_bwd as base
from oracle import grad_oracle as O

pytestmark = pytest.mark.gpu


def loud(gpu, Sq, Sk, D, sizes, value=None, q_size=2.0, Sk2=0):
    """fp16 inputs whose rows of dout have the first of `sizes`, but for one of each of the others; `value` is a number of one row of v."""
    r = lambda n, S: base.rand(gpu, n, 1, 2, S, D)  # noqa: E731
    q, k, v, dout = q_size * r(1, Sq), r(2, Sk), r(3, Sk), sizes[0] * r(4, Sq)
    for i, size in enumerate(sizes[1:]):
        row = (i + 1) * Sq // len(sizes) + 3
        dout[:, :, row] *= size / sizes[0]
    if value is not None:
        v[:, :, Sk // 3, 5] = value
    k2, v2 = (r(5, Sk2).half(), r(6, Sk2).half()) if Sk2 else (None, None)
    q, k, v, dout = (t.half() for t in (q, k, v, dout))
    kk, vv = (torch.cat((k, k2), 2), torch.cat((v, v2), 2)) if Sk2 else (k, v)
    out, lse = O.attn_fwd(q, kk, vv, D ** -0.5)
    return q, k, v, k2, v2, dout, out.half(), lse.float()


@pytest.mark.parametrize("Sq,Sk,D,sizes,value,q_size,Sk2", [
    (300, 16384, 64, (1.0, 1000.0, 4000.0), None, 2.0, 0),
    (300, 16384, 128, (1.0, 1000.0, 4000.0), 50.0, 2.0, 0),
    (256, 4096, 64, (0.03, 1000.0), None, 2.0, 0),
    (60, 16384, 64, (0.1, 3000.0), None, 2.0, 0),
    (500, 700, 128, (0.03, 30.0, 1000.0), 1000.0, 2.0, 90),
    (20, 50, 64, (0.1, 3000.0), 1000.0, 2.0, 0),
    (40, 16384, 40, (0.1, 3000.0), 30000.0, 2.0, 0),
    (200, 3000, 72, (0.1, 10.0, 3000.0), 300.0, 2.0, 100),
    (60, 500, 64, (0.1, 3000.0), None, 10.0, 0),
    (150, 5000, 96, (0.1, 3000.0), None, 8.0, 0),
])
def test_fp16_rows_of_other_sizes(gpu, Sq, Sk, D, sizes, value, q_size, Sk2):
    """No row of dout and no value takes the bits of another's gradient."""
    t = loud(gpu, Sq, Sk, D, sizes, value, q_size, Sk2)
    want, far = base.bounds(*t)
    lost = 2.0 ** -40 * t[5].double().abs().sum(2, keepdim=True)
    far = [f + lost if i in (2, 4) else f for i, f in enumerate(far)]
    base.close(base.call(*t), want, far)


@pytest.mark.parametrize("cus", [1, 4096])
def test_fp16_rows_of_other_sizes_in_parts(gpu, cus, monkeypatch):
    monkeypatch.setitem(base.ops.TUNING, "cu_count", cus)
    t = loud(gpu, 700, 900, 64, (0.1, 20.0, 3000.0), 100.0, 2.0, 60)
    got = base.call(*t)
    base.close(got, *base.bounds(*t))
    assert all(torch.equal(a, b) for a, b in zip(got, base.call(*t)))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [64, 72, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_row_that_is_not_finite(gpu, dtype, D, bad):
    """In dout it reaches that query's dq, all dk and one column of dv of its head; in v that key's dk and all dq.  The rest has the bits that it has without."""
    t = base.inputs(gpu, 1, 3, 150, 100, D, 0, dtype)
    clean = base.call(*t)
    base.close(clean, *base.bounds(*t))
    q, k, v, _, _, dout, out, lse = t
    other = [i for i in range(3) if i != 1]

    def check(got, broken):
        """`broken`: for each gradient what of head 1 is not finite."""
        for g, c, b in zip(got, clean, broken):
            mask = torch.zeros_like(g[0, 1], dtype=torch.bool)
            if b is not None:
                mask[b] = True
            assert torch.equal(g[:, other], c[:, other])
            assert not bool(g[0, 1][mask].isfinite().any()) and torch.equal(g[0, 1][~mask], c[0, 1][~mask])

    every = slice(None)
    d = dout.clone()
    d[0, 1, 70, 5] = bad
    check(base.call(q, k, v, None, None, d, out, lse), (70, every, (every, 5)))
    w = v.clone()
    w[0, 1, 33, 5] = bad
    check(base.call(q, k, w, None, None, dout, out, lse), (every, 33, None))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D,layout", [(64, "bhsd"), (72, "bshd"), (128, "bshd")])
@pytest.mark.parametrize("rows", [[70], [149], [0, 63, 64, 148, 149], list(range(64, 128)), list(range(150))])
@pytest.mark.parametrize("cus", [0, 4096])
def test_what_rows_hold_that_attended_nothing(gpu, dtype, D, layout, rows, cus, monkeypatch):
    """Rows of q, dout and out whose log-sum-exp is -infinity need not be finite: the gradients have the bits that they have over any numbers there, those rows' own are zeros."""
    monkeypatch.setitem(base.ops.TUNING, "cu_count", cus)
    q, k, v, k2, v2, dout, out, lse = t = base.inputs(gpu, 1, 2, 150, 100, D, 30, dtype, layout)
    lse[:, 1, rows] = -math.inf
    clean = base.call(*t)
    base.close(clean, *base.bounds(*t))
    for bad in ((math.nan,) * 3, (1.0, math.inf, 1.0), (-math.inf, 1.0, math.nan), (1.0, math.nan, math.inf)):
        fill = [x.clone() for x in (q, dout, out)]
        for x, b in zip(fill, bad):
            if b != 1.0:
                x[:, 1, rows] = b
        got = base.call(fill[0], k, v, k2, v2, fill[1], fill[2], lse)
        assert all(torch.equal(a, b) for a, b in zip(got, clean))
        assert not got[0][:, 1, rows].any()
