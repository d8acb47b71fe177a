"""Calls of many rows, where a wavefront holds a row, and parts of many rows a workgroup: the bars are those of few rows."""
import pytest
import torch

from oracle import block_oracle as O
from test_gpu_block_norm import F32, close, problem
from xdit_amd import block_ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,S,C", [(1, 1030, 8), (2, 613, 136), (3, 401, 504), (1, 1153, 512), (2, 555, 520), (1, 1500, 1152), (2, 700, 1544), (1, 1031, 2040), (2, 517, 2056), (1, 1201, 2560), (1, 1030, 2568), (2, 530, 2984)])
def test_many_rows_against_oracle(gpu, dtype, B, S, C):
    for norm, y_norm, mods, affine in (("layer", None, "wide", False), ("rms", "rms", "same", True), ("layer", "layer", "wide", True), ("rms", None, "same", False)):
        k = problem(gpu, B, S, C, dtype, mods, affine=affine)
        if y_norm is None:
            k.pop("y_weight", None)
        rh, rn, rs, size = O.gated_norm(norm=norm, y_norm=y_norm, eps=1e-5, y_eps=1e-4, residual_scale=0.7, **k)
        h, n, st = block_ops.gated_norm(norm=norm, y_norm=y_norm, eps=1e-5, y_eps=1e-4, residual_scale=0.7, return_stats=True, **k)
        close(n, rn, size)
        close(h, rh, rh.abs().amax(-1, keepdim=True) + k["x"].double().abs())
        close(st[..., 1::2].contiguous(), rs[..., 1::2], rs[..., 1::2])
        close(st[..., 0::2].contiguous(), rs[..., 0::2], torch.stack([rh.abs().amax(-1), k["y"].double().abs().amax(-1)], -1))


def test_variants_of_many_rows(gpu):
    """No y, no norm, (B, C) and batch-broadcast modulation, strided rows, h in place, rows that are not finite, the same bits again."""
    B, S, C = 2, 811, 1160
    k = problem(gpu, B, S, C, torch.bfloat16)
    x, y = k["x"], k["y"]
    close(block_ops.gated_norm(x, scale=k["scale"], norm="rms")[1], *O.gated_norm(x, scale=k["scale"], norm="rms")[1:4:2])
    rh, _, _, size = O.gated_norm(x, y=y, gate=k["gate"], norm=None)
    close(block_ops.gated_norm(x, y=y, gate=k["gate"], norm=None)[0], rh, size)
    kk = dict(gate=k["gate"][:, 0], scale=k["scale"][:, 0], shift=k["shift"][:1], y=y)
    rh, rn, _, size = O.gated_norm(x, **kk)
    wide = torch.randn(B, S, 2 * C + 8, device=gpu).bfloat16()
    wide[..., 8:8 + C] = x
    keep = wide.clone()
    xs = wide[..., 8:8 + C]
    h, n = block_ops.gated_norm(xs, **kk)
    close(n, rn, size)
    h2, n2 = block_ops.gated_norm(xs, out_h=xs, **kk)
    assert h2 is xs and torch.equal(h2, h) and torch.equal(n2, n)
    assert torch.equal(wide[..., :8], keep[..., :8]) and torch.equal(wide[..., 8 + C:], keep[..., 8 + C:])
    bad = torch.zeros(S, dtype=torch.bool, device=gpu)
    bad[[0, 5, 400, S - 1]] = True
    broken = x.clone()
    broken[1, bad, 3] = float("nan")
    n3 = block_ops.gated_norm(broken, **kk)[1]
    assert torch.equal(n3[0], n[0]) and torch.equal(n3[1, ~bad], n[1, ~bad]) and torch.isnan(n3[1, bad].float()).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,S,C,y", [(1, 1100, 8, False), (2, 613, 200, True), (1, 1203, 1160, True), (2, 519, 2056, False), (1, 1100, 2600, True), (1, 1050, 1544, False), (1, 9001, 4104, True), (3, 5003, 3600, False)])
def test_fp8_output_of_many_rows(gpu, dtype, B, S, C, y):
    """Also parts of 16 rows and more of a workgroup, whose scales leave together, and what is left of them."""
    k = problem(gpu, B, S, C, dtype, y=y, affine=False)
    _, rn, _, size = O.gated_norm(**k)
    _, (q, sc) = block_ops.gated_norm(fp8=True, **k)
    assert q.dtype == torch.float8_e4m3fn and sc.shape == (B, S, (C + 127) // 128)
    top = O.block_scales(rn.view(-1, C), 1).view(sc.shape)
    assert bool(((sc.double() - top).abs() <= 2.0 ** -23 * top + F32 * size.amax() / 448).all())
    full = O.spread(sc.double().reshape(B * S, -1), 1, B * S, C).view(B, S, C)
    err = (q.double() * full - rn).abs()
    assert bool((err <= 2.0 ** -4 * rn.abs() * 1.001 + 2.0 ** -10 * full + 2 * F32 * size).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,S,C,per_token", [(2, 2100, 1536, False), (1, 3001, 2056, False), (1, 1301, 5128, True), (3, 901, 520, True), (1, 5003, 8, False)])
def test_gradients_of_many_rows(gpu, dtype, B, S, C, per_token):
    """The chain of a column sum: rows of a part over its teams, teams, runs of parts, runs: far below a sixteenth of the rows and 80."""
    k = problem(gpu, B, S, C, dtype, "wide", per_token)
    opt = dict(norm="layer", y_norm="rms", residual_scale=0.7)
    h, _, st = block_ops.gated_norm(return_stats=True, **opt, **k)
    k.pop("x")
    dh, dn = (torch.randn(h.shape, generator=torch.Generator(device=gpu).manual_seed(s), device=gpu).to(dtype) for s in (1, 2))
    ref, big = O.gated_norm_backward(dh, dn, h, st, **opt, **k)
    got = block_ops.gated_norm_backward(dh, dn, h, st, **opt, **k)
    assert set(got) == set(ref)
    chain = (B * S / 16 + 80) * 2.0 ** -24
    for name in got:
        close(got[name], ref[name], big[name], F32 if name in ("dx", "dy") else chain + F32)
