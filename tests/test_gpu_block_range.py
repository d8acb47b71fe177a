"""Rows whose mean square does not fit fp32: finite elements beyond about 2^63.  An infinite deviation makes the normalised row zero, as
1 / sqrt(inf) does in fp32 PyTorch, and leaves the rows beside it alone; NaN stays where the row itself holds one or an infinity."""
import pytest
import torch

from xdit_amd import block_ops

pytestmark = pytest.mark.gpu


def randn(gpu, *s, seed=0):
    return torch.randn(*s, generator=torch.Generator(device=gpu).manual_seed(seed), device=gpu)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("S,C", [(6, 64), (6, 1160), (2000, 640), (1500, 2560), (9, 8192)])
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_norm_of_rows_beyond_the_range(gpu, dtype, S, C, norm):
    x = randn(gpu, 1, S, C).to(dtype)
    y = randn(gpu, 1, S, C, seed=1).to(dtype)
    shift = randn(gpu, 1, C, seed=2).to(dtype)
    k = dict(shift=shift, norm=norm, y_norm="rms", return_stats=True)
    h0, n0, st0 = block_ops.gated_norm(x, y=y, **k)
    keep = torch.arange(S, device=gpu) % 3 != 1
    x[0, 1::3] *= 1e20
    h, n, st = block_ops.gated_norm(x, y=y, **k)
    assert torch.isfinite(n.float()).all() and torch.equal(n[0, ~keep], shift.expand(S, C)[~keep]) and (st[0, ~keep, 1] == 0).all()
    assert torch.equal(n[0, keep], n0[0, keep]) and torch.equal(st[0, keep], st0[0, keep])
    y[0, 1::3] *= 1e20                                    # the branch's norm: its row adds nothing
    h2, n2, st2 = block_ops.gated_norm(randn(gpu, 1, S, C).to(dtype), y=y, **k)
    assert torch.equal(h2[0, ~keep], randn(gpu, 1, S, C).to(dtype)[0, ~keep]) and torch.equal(n2[0, keep], n0[0, keep])
    dn = randn(gpu, 1, S, C, seed=3).to(dtype)
    g = block_ops.gated_norm_backward(dn, dn, h, st, y=y, norm=norm, y_norm="rms", shift=shift)
    assert torch.equal(g["dx"][0, ~keep], dn[0, ~keep]) and torch.isfinite(g["dx"].float()).all()
    _, (q, scale) = block_ops.gated_norm(x, y=y, shift=shift, norm=norm, y_norm="rms", fp8=True)
    assert torch.isfinite(q.float()).all() and torch.isfinite(scale).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [8, 64, 128, 512])
def test_rotation_of_rows_beyond_the_range(gpu, dtype, D):
    q = randn(gpu, 1, 3, 50, D).to(dtype)
    freq, pairs = block_ops.rope_frequencies((D,), device=gpu)
    pos = torch.arange(50, device=gpu).view(50, 1)
    w = randn(gpu, D, seed=4)
    ref, _ = block_ops.axes_rope(q, None, pos, freq, pairs, norm=True, q_weight=w)
    q[:, 1, 7] *= 1e20
    y, _ = block_ops.axes_rope(q, None, pos, freq, pairs, norm=True, q_weight=w)
    keep = torch.ones(1, 3, 50, dtype=torch.bool, device=gpu)
    keep[:, 1, 7] = False
    assert torch.equal(y[keep], ref[keep]) and (y[~keep] == 0).all()
    dq, _, dw, _ = block_ops.axes_rope_backward(ref, None, pos, freq, pairs, q=q, norm=True, q_weight=w)
    assert (dq[~keep] == 0).all() and torch.isfinite(dq.float()).all() and torch.isfinite(dw).all()


def test_infinities_and_nan_keep_to_their_row(gpu):
    """An RMS row with an infinity: the infinity over itself is NaN, the rest of the row zero; with a NaN: all of it."""
    x = randn(gpu, 1, 5, 256).bfloat16()
    ref = block_ops.gated_norm(x, norm="rms")[1]
    x[0, 1, 9], x[0, 3, 11] = float("inf"), float("nan")
    n = block_ops.gated_norm(x, norm="rms")[1]
    assert torch.equal(n[0, [0, 2, 4]], ref[0, [0, 2, 4]]) and torch.isnan(n[0, 3].float()).all()
    assert torch.isnan(n[0, 1, 9].float()) and (n[0, 1].float().nan_to_num(0) == 0).all() and int(torch.isnan(n[0, 1].float()).sum()) == 1
