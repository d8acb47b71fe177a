"""The norms around a block with their gate, residual and modulation, against the float64 oracle.

Bars: a result is rounded once to its dtype (half a unit: 2^-8, 2^-11 or 2^-24 of its value) and computed in fp32 before that.
A row's statistics come from sums of up to 8192 terms (at most 32 additions in a chain of a thread, 8 across lanes and wavefronts),
and an element from a dozen operations, so fp32 errors stay below 64 units of 2^-24 of the largest terms involved, which the
oracle returns.  A column sum adds its rows in a chain of (rows of a part) + (parts) additions, each off by at most 2^-24 of the
sum of the terms' sizes.
"""
import pytest
import torch

from oracle import block_oracle as O
from xdit_amd import block_ops

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
F32 = 64 * 2.0 ** -24


def close(got, ref, size, factor=F32):
    assert got.shape == ref.shape, (got.shape, ref.shape)
    err = (got.double() - ref).abs()
    bound = HALF[got.dtype] * ref.abs() * 1.01 + TINY[got.dtype] + factor * size
    assert bool((err <= bound).all()), (err - bound).max().item()


def problem(gpu, B, S, C, dtype, mods="wide", per_token=False, y=True, affine=True, seed=0, batch1=False):
    g = torch.Generator(device=gpu).manual_seed(seed + B * 1000003 + S * 1009 + C)
    rn = lambda *s: torch.randn(*s, generator=g, device=gpu)  # noqa: E731
    md = torch.float32 if mods == "wide" else dtype
    ms = (B, S, C) if per_token else (B, 1, C)
    k = dict(x=(2 * rn(B, S, C) + 0.5).to(dtype), scale=(0.4 * rn(*ms)).to(md), shift=rn(*ms).to(md))
    if y:
        k.update(y=(rn(B, S, C) * 3 - 1).to(dtype), gate=rn(*ms).to(md))
    if affine:
        k.update(weight=(1 + 0.3 * rn(C)).to(dtype), bias=rn(C).to(dtype))
        if y:
            k["y_weight"] = (1 + 0.3 * rn(C)).to(dtype)
    return k


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,S,C", [(1, 1, 8), (2, 3, 136), (1, 5, 1152), (3, 2, 2048), (1, 4, 2056), (2, 2, 5120), (1, 3, 8192), (1, 700, 640)])
def test_forward_against_oracle(gpu, dtype, B, S, C):
    for norm, y_norm, mods, per_token, affine in (("layer", None, "wide", False, False), ("rms", "rms", "same", False, True),
                                                  ("layer", "layer", "wide", True, True), ("rms", None, "same", True, False)):
        k = problem(gpu, B, S, C, dtype, mods, per_token, affine=affine)
        if y_norm is None:
            k.pop("y_weight", None)
        rh, rn, rs, size = O.gated_norm(norm=norm, y_norm=y_norm, eps=1e-5, y_eps=1e-4, residual_scale=0.7, **k)
        h, n, st = block_ops.gated_norm(norm=norm, y_norm=y_norm, eps=1e-5, y_eps=1e-4, residual_scale=0.7, return_stats=True, **k)
        assert h.dtype == n.dtype == dtype
        close(n, rn, size)
        close(h, rh, rh.abs().amax(-1, keepdim=True) + k["x"].double().abs())
        close(st[..., 1::2].contiguous(), rs[..., 1::2], rs[..., 1::2])
        close(st[..., 0::2].contiguous(), rs[..., 0::2], torch.stack([rh.abs().amax(-1), k["y"].double().abs().amax(-1)], -1))


@pytest.mark.gpu
def test_forward_variants(gpu):
    """What may be left out: y, the norm, modulation; (B, C) modulation; a batch-broadcast one; strided rows; h in place."""
    B, S, C = 2, 37, 1160
    k = problem(gpu, B, S, C, torch.bfloat16)
    x, y = k["x"], k["y"]
    h, n = block_ops.gated_norm(x, scale=k["scale"], norm="rms")
    assert h is x
    close(n, *O.gated_norm(x, scale=k["scale"], norm="rms")[1:4:2])
    h, n = block_ops.gated_norm(x, y=y, gate=k["gate"], norm=None)
    rh, _, _, size = O.gated_norm(x, y=y, gate=k["gate"], norm=None)
    assert n is None
    close(h, rh, size)
    kk = dict(gate=k["gate"][:, 0], scale=k["scale"][:, 0], shift=k["shift"][:1], y=y)
    rh, rn, _, size = O.gated_norm(x, **kk)
    wide = torch.randn(B, S, 2 * C + 8, device=gpu).bfloat16()
    wide[..., 8:8 + C] = x
    keep = wide.clone()
    xs = wide[..., 8:8 + C]
    h, n = block_ops.gated_norm(xs, **kk)
    close(n, rn, size)
    h2, n2 = block_ops.gated_norm(xs, out_h=xs, **kk)       # the residual stream in place, its neighbours untouched
    assert h2 is xs and torch.equal(h2, h) and torch.equal(n2, n)
    assert torch.equal(wide[..., :8], keep[..., :8]) and torch.equal(wide[..., 8 + C:], keep[..., 8 + C:])
    e = block_ops.gated_norm(x[:, :0], scale=k["scale"])
    assert e[1].shape == (B, 0, C)
    # a row of equal values has no deviation: eps alone keeps it finite
    flat = torch.full((1, 2, 256), 3.0, device=gpu)
    assert torch.equal(block_ops.gated_norm(flat)[1], torch.zeros_like(flat))
    # a large mean costs the variance no digits
    off = (torch.randn(1, 4, 1024, device=gpu) + 4096).contiguous()
    close(block_ops.gated_norm(off)[1], *O.gated_norm(off)[1:4:2])


@pytest.mark.gpu
def test_non_finite_rows_stay_by_themselves(gpu):
    k = problem(gpu, 1, 6, 512, torch.bfloat16)
    h0, n0 = block_ops.gated_norm(**k)
    k["x"][0, 2, 7] = float("nan")
    k["x"][0, 4, 9] = float("inf")
    h, n = block_ops.gated_norm(**k)
    bad = torch.tensor([2, 4], device=gpu)
    good = torch.tensor([0, 1, 3, 5], device=gpu)
    assert torch.equal(n[0, good], n0[0, good]) and not torch.isfinite(n[0, bad].float()).all(-1).any()
    q, s = block_ops.gated_norm(fp8=True, **k)[1]
    assert torch.isfinite(s[0, good]).all() and torch.isnan(s[0, 2]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,S,C", [(1, 1, 8), (2, 33, 1152), (1, 7, 200), (1, 3, 5120), (2, 130, 8192)])
def test_fp8_output(gpu, dtype, B, S, C):
    """Scales within fp32 rounding of the oracle's, every value within half an e4m3 step (2^-4 of it, or 2^-10 of the scale) of n."""
    k = problem(gpu, B, S, C, dtype, y=False)
    _, rn, _, size = O.gated_norm(**k)
    _, (q, sc) = block_ops.gated_norm(fp8=True, **k)
    assert q.dtype == torch.float8_e4m3fn and sc.shape == (B, S, (C + 127) // 128)
    top = O.block_scales(rn.view(-1, C), 1).view(sc.shape)
    assert bool(((sc.double() - top).abs() <= 2.0 ** -23 * top + F32 * size.amax() / 448).all())
    full = O.spread(sc.double().reshape(B * S, -1), 1, B * S, C).view(B, S, C)
    err = (q.double() * full - rn).abs()
    assert bool((err <= 2.0 ** -4 * rn.abs() * 1.001 + 2.0 ** -10 * full + 2 * F32 * size).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,S,C", [(1, 1, 8), (2, 3, 136), (1, 77, 1152), (3, 40, 2048), (1, 19, 2056), (2, 17, 5120), (1, 5, 8192), (1, 1500, 640)])
def test_backward_against_oracle(gpu, dtype, B, S, C):
    g = torch.Generator(device=gpu).manual_seed(C)
    for norm, y_norm, mods, per_token, affine in (("layer", None, "wide", False, False), ("rms", "rms", "same", False, True),
                                                  ("layer", "layer", "wide", True, True), ("rms", None, "same", True, False)):
        k = problem(gpu, B, S, C, dtype, mods, per_token, affine=affine)
        if y_norm is None:
            k.pop("y_weight", None)
        opt = dict(norm=norm, y_norm=y_norm, residual_scale=0.7)
        h, _, st = block_ops.gated_norm(return_stats=True, **opt, **k)
        k.pop("x")
        dh = torch.randn(h.shape, generator=g, device=gpu).to(dtype)
        dn = torch.randn(h.shape, generator=g, device=gpu).to(dtype)
        for a, b in ((dh, dn), (None, dn), (dh, None)):
            ref, big = O.gated_norm_backward(a, b, h, st, **opt, **k)
            if b is None:
                for name in ("dscale", "dshift", "dweight", "dbias"):
                    ref.pop(name, None)
            got = block_ops.gated_norm_backward(a, b, h, st, **opt, **k)
            assert set(got) == set(ref), (set(got), set(ref))
            chain = (min(B * S, 16 + B * S // 1024 + B * S // 16) + 64) * 2.0 ** -24
            for name in got:
                close(got[name], ref[name], big[name], F32 if name in ("dx", "dy") else chain + F32)
    again = block_ops.gated_norm_backward(dh, dn, h, st, **opt, **k)
    once = block_ops.gated_norm_backward(dh, dn, h, st, **opt, **k)
    assert all(torch.equal(again[n], once[n]) for n in again)      # a fixed order of summation


@pytest.mark.gpu
def test_backward_against_differences(gpu):
    """Central differences of a weighted sum of h and n along random directions, in fp32.  The step of 2^-7 leaves a truncation
    error of about its square (6e-5) and a rounding error of 2^-24 sqrt(terms) / step (a few 1e-4): bar 2e-3 of the sum of the sizes."""
    k = problem(gpu, 2, 6, 264, torch.float32)
    opt = dict(norm="layer", y_norm="rms", residual_scale=0.7)
    ch, cn = torch.randn_like(k["x"]), torch.randn_like(k["x"])
    h, _, st = block_ops.gated_norm(return_stats=True, **opt, **k)
    kk = {n: t for n, t in k.items() if n != "x"}
    grads = block_ops.gated_norm_backward(ch, cn, h, st, **opt, **kk)

    def loss(**over):
        a, b = block_ops.gated_norm(**opt, **{**k, **over})
        return (a.double() * ch).sum().item() + (b.double() * cn).sum().item()

    step = 2.0 ** -7
    for name, t in k.items():
        d = torch.randn_like(t)
        num = (loss(**{name: t + step * d}) - loss(**{name: t - step * d})) / (2 * step)
        prod = grads["d" + name].double() * d
        assert abs(num - prod.sum().item()) <= 2e-3 * prod.abs().sum().item(), (name, num, prod.sum().item())


@pytest.mark.gpu
def test_on_another_stream_and_in_a_graph(gpu):
    k = problem(gpu, 2, 50, 1152, torch.bfloat16)
    opt = dict(norm="rms", y_norm="rms")
    h, n, st = block_ops.gated_norm(return_stats=True, **opt, **k)
    kk = {m: t for m, t in k.items() if m != "x"}
    ref = block_ops.gated_norm_backward(h, n, h, st, **opt, **kk)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = block_ops.gated_norm(return_stats=True, **opt, **k)
        b = block_ops.gated_norm_backward(a[0], a[1], a[0], a[2], **opt, **kk)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a[1], n) and all(torch.equal(ref[m], b[m]) for m in ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        block_ops.gated_norm_backward(h, n, h, st, **opt, **kk)   # scratch of this stream exists before the capture
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            c = block_ops.gated_norm(return_stats=True, **opt, **k)
            d = block_ops.gated_norm_backward(c[0], c[1], c[0], c[2], **opt, **kk)
    for _ in range(3):
        k["x"].mul_(-0.5)
        want = block_ops.gated_norm(return_stats=True, **opt, **k)
        wgrad = block_ops.gated_norm_backward(want[0], want[1], want[0], want[2], **opt, **kk)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c[1], want[1]) and all(torch.equal(d[m], wgrad[m]) for m in wgrad)


@pytest.mark.gpu
def test_refusals(gpu):
    x = torch.zeros(2, 3, 64, device=gpu, dtype=torch.bfloat16)
    m = torch.zeros(2, 1, 64, device=gpu)
    f = block_ops.gated_norm
    for bad in (lambda: f(x[0]), lambda: f(x, norm="batch"), lambda: f(x, gate=m), lambda: f(x, y_norm="rms"), lambda: f(x, y=x.float()),
                lambda: f(x, scale=m[:, :, :32]), lambda: f(x, scale=m.half()), lambda: f(x, norm=None, scale=m),
                lambda: f(x, scale=m, shift=m.bfloat16()), lambda: f(x, weight=m[0, 0].half()), lambda: f(x, weight=m), lambda: f(x.cpu()[..., ::2]),
                lambda: f(x, eps=float("nan")), lambda: f(x, residual_scale=float("inf")), lambda: f(x[..., 1:57]), lambda: f(x.double()),
                lambda: f(x, y=x, out_h=x.float()), lambda: f(x, y=x, out_h=torch.zeros(1, 1, 64, device=gpu, dtype=x.dtype).expand(2, 3, 64))):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
    with pytest.raises(NotImplementedError):
        f(torch.zeros(1, 1, 8200, device=gpu))
    with pytest.raises(NotImplementedError):
        f(torch.zeros(1, 1, 12, device=gpu))
    h, n, st = f(x, y=x, gate=m, scale=m, return_stats=True)
    b = block_ops.gated_norm_backward
    per = m.expand(2, 3, 64)
    for bad in (lambda: b(None, None, h, st), lambda: b(h, n, h, st[..., :3]), lambda: b(h, n, h, st, gate=m), lambda: b(h, n, h, st, norm=None),
                lambda: b(h, n, h, st, y=x, gate=m[:1]), lambda: b(h, n, h, st, scale=m, shift=per), lambda: b(h, n.float(), h, st)):
        with pytest.raises(ValueError):
            bad()


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError):
        block_ops.gated_norm(torch.zeros(1, 2, 64))


@pytest.mark.gpu
@pytest.mark.parametrize("S,C", [(40, 1160), (1500, 640), (1100, 2304), (9, 8192)])
def test_fp8_output_beside_the_quantiser(gpu, S, C):
    """fp32 n is the unrounded one, so the quantiser's result from it can be had.  Scales: a product with 1 / 448 against a division, two roundings
    against one, 3 * 2^-24.  Values: the hardware's reciprocal (a unit, 2^-23) and a product against a division, and the scale's difference: 7 * 2^-24;
    only quotients that close to the middle of two e4m3 numbers may differ, by one step."""
    k = problem(gpu, 2, S, C, torch.float32)
    n = block_ops.gated_norm(**k)[1]
    q, s = block_ops.gated_norm(fp8=True, **k)[1]
    rq, rs = block_ops.fp8_block_quant(n)
    assert bool(((s.double() - rs.double()).abs() <= 3 * 2.0 ** -24 * 1.001 * rs.double()).all())
    other = q.view(torch.uint8) != rq.view(torch.uint8)
    a, b = q.double()[other], rq.double()[other]
    quotient = (n.double() / rs.double().repeat_interleave(128, -1)[..., :C])[other]
    assert bool(((a - b).abs() <= a.abs().maximum(b.abs()) / 8 + 2.0 ** -9 * 1.001).all())
    assert bool((((a + b) / 2 - quotient).abs() <= 8 * 2.0 ** -24 * quotient.abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,S,C,per_token", [(1, 600, 3080, False), (2, 301, 4096, False), (1, 601, 4088, True), (300, 1, 136, False), (150, 3, 1032, True), (2100, 1, 64, False)])
def test_gradients_of_two_teams_and_of_many_batch_entries(gpu, dtype, B, S, C, per_token):
    """Rows that fill a workgroup's LDS with two teams' sums, and entries of one to three tokens.  A column sum adds at most 16 rows of a team, 16 teams, its
    entry's parts in 64 runs and, for what the entries share, B totals."""
    k = problem(gpu, B, S, C, dtype, "wide", per_token)
    opt = dict(norm="layer", y_norm="rms", residual_scale=0.7)
    h, n, st = block_ops.gated_norm(return_stats=True, **opt, **k)
    rh, rn, _, size = O.gated_norm(**opt, **k)
    close(n, rn, size)
    k.pop("x")
    dh, dn = (torch.randn(h.shape, generator=torch.Generator(device=gpu).manual_seed(s), device=gpu).to(dtype) for s in (1, 2))
    ref, big = O.gated_norm_backward(dh, dn, h, st, **opt, **k)
    got = block_ops.gated_norm_backward(dh, dn, h, st, **opt, **k)
    for name in got:
        close(got[name], ref[name], big[name], F32 if name in ("dx", "dy") else (16 + 16 + 10 + B) * 2.0 ** -24 + F32)
