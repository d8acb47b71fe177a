"""The rotation of q and k by positions on several axes, with its RMSNorm, against the float64 oracle.

Bars: one rounding to the dtype (2^-8, 2^-11 or 2^-24 of the value) behind fp32 arithmetic.  An element is two products of
values of at most the pair's size with a sine and a cosine; those come from an angle reduced in fp64 and then rounded to fp32
(2^-25 of half a turn, times pi) by a function good to 2 units, the norm's statistic from at most 512 squares: 32 units of 2^-24 of
the row's largest element cover them.  The gains' gradients add the rows in chains of (rows of a wavefront) + (workgroups / 32) + 40.
"""
import pytest
import torch

from oracle import block_oracle as O
from xdit_amd import block_ops

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
F32 = 32 * 2.0 ** -24


def close(got, ref, size, factor=F32):
    assert got.shape == ref.shape
    err = (got.double() - ref).abs()
    bound = HALF[got.dtype] * ref.abs() * 1.01 + TINY[got.dtype] + factor * size
    assert bool((err <= bound).all()), (err - bound).max().item()


def problem(gpu, B, S, H, Hk, D, axes, dtype, layout, pos="grid"):
    g = torch.Generator(device=gpu).manual_seed(B + S * 7 + H * 31 + D)
    rn = lambda *s: torch.randn(*s, generator=g, device=gpu)  # noqa: E731
    make = lambda h: (rn(B, S, h, D).to(dtype).transpose(1, 2) if layout == "bshd" else rn(B, h, S, D).to(dtype))  # noqa: E731
    inv, pairs = block_ops.rope_frequencies(axes, device=gpu)
    i = torch.arange(S, device=gpu)
    p = torch.stack([i // 64, i // 8 % 8 - 4, i % 8 - 4, i][:len(axes)], 1)
    if pos == "float":
        p = p.float() * 0.37 - 2.5
    elif pos == "int32":
        p = p.int()
    elif pos == "batch":
        p = torch.stack([p * (b + 1) for b in range(B)]).float()
    elif pos == "far":
        p = p * 100003
    return make(H), make(Hk), p, inv, pairs, (1 + 0.3 * rn(D)), (1 + 0.3 * rn(D))


CASES = [(1, 1, 1, 1, 8, (8,)), (2, 5, 3, 3, 128, (16, 56, 56)), (1, 70, 40, 10, 128, (44, 42, 42)), (2, 33, 5, 1, 64, (16, 24, 24)), (1, 19, 16, 16, 72, (0, 36, 36)),
         (1, 21, 7, 7, 96, (32, 32, 24)), (1, 40, 2, 9, 128, (16, 24, 24)), (1, 9, 3, 2, 512, (128, 128, 128, 128)), (1, 6, 70, 70, 256, (8, 8, 8))]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rope", ["interleaved", "split_half"])
@pytest.mark.parametrize("case", CASES)
def test_against_oracle(gpu, dtype, rope, case):
    B, S, H, Hk, D, axes = case
    for n, (layout, pos, norm, wide) in enumerate((("bshd", "grid", True, False), ("bhsd", "float", False, False), ("bshd", "batch", True, True), ("bhsd", "int32", True, None))):
        q, k, p, inv, pairs, qw, kw = problem(gpu, B, S, H, Hk, D, axes, dtype, layout, pos)
        qw, kw = (None, None) if not norm or wide is None else (qw, kw) if wide else (qw.to(dtype), kw.to(dtype))
        f = inv if n != 1 else inv.float()
        opt = dict(norm=norm, q_weight=qw, k_weight=kw, eps=1e-5, rope=rope)
        yq, yk = block_ops.axes_rope(q, k, p, f, pairs, **opt)
        dq, dk = torch.randn_like(yq).transpose(2, 3).contiguous().transpose(2, 3).contiguous(), torch.randn_like(yk)
        got = block_ops.axes_rope_backward(dq, dk, p, f, pairs, q=q, k=k, **opt)
        for x, w, y, d, dx, dw in ((q, qw, yq, dq, got[0], got[2]), (k, kw, yk, dk, got[1], got[3])):
            ref = O.axes_rope(x, w, p, f, pairs, norm, 1e-5, rope)
            pre = O.axes_rope(x, w, p * 0, f, pairs, norm, 1e-5, rope)
            assert y.is_contiguous() and y.dtype == dtype
            close(y, ref, pre.abs().amax(-1, keepdim=True))
            rdx, rdw, sx, sw = O.axes_rope_backward(d, x, w, p, f, pairs, norm, 1e-5, rope)
            close(dx, rdx, sx)
            assert (dw is None) == (w is None)
            if dw is not None:
                close(dw, rdw, sw, F32 + (x.shape[1] * S * B / 4 + 40) * 2.0 ** -24)


@pytest.mark.gpu
def test_large_positions_keep_their_angle(gpu):
    """Positions of several millions: the angle is reduced in fp64, so fp32 tensors keep their bar."""
    q, k, p, inv, pairs, _, _ = problem(gpu, 1, 64, 2, 2, 128, (44, 42, 42), torch.float32, "bhsd", "far")
    y, _ = block_ops.axes_rope(q, k, p, inv, pairs)
    close(y, O.axes_rope(q, None, p, inv, pairs, False, 0, "interleaved"), q.double().abs().amax(-1, keepdim=True))


@pytest.mark.gpu
def test_identities(gpu):
    """Position 0 leaves bits alone, backward undoes forward, rotating in place and into given tensors gives the same bits,
    agreement with the table-driven rotation."""
    q, k, p, inv, pairs, qw, kw = problem(gpu, 1, 77, 3, 3, 128, (16, 56, 56), torch.bfloat16, "bshd")
    y, z = block_ops.axes_rope(q, k, p * 0, inv, pairs)
    assert torch.equal(y, q) and torch.equal(z, k)
    qf = q.float()
    y, none = block_ops.axes_rope(qf, None, p, inv, pairs)
    assert none is None
    back = block_ops.axes_rope_backward(y, None, p, inv, pairs)
    assert back[1:] == (None, None, None)
    close(back[0], qf.double(), 2 * qf.double().abs().amax(-1, keepdim=True))
    ref = block_ops.axes_rope(q, k, p, inv, pairs, norm=True, q_weight=qw, k_weight=kw)
    out = torch.full((1, 3, 100, 128), 7.0, device=gpu, dtype=q.dtype)
    a, b = q.clone(), out[:, :, 9:86]
    block_ops.axes_rope(a, k, p, inv, pairs, norm=True, q_weight=qw, k_weight=kw, out_q=a, out_k=b)
    assert torch.equal(a, ref[0]) and torch.equal(b, ref[1]) and bool((out[:, :, :9] == 7).all()) and bool((out[:, :, 86:] == 7).all())
    from xdit_amd import prologue
    axis = torch.tensor([a for a, n in enumerate(pairs) for _ in range(n)], device=gpu)
    phi = (p.double()[:, axis] * inv).float().repeat_interleave(2, 1)
    table = prologue.apply_rotary_emb(qf, (phi.cos(), phi.sin()))
    mine, _ = block_ops.axes_rope(qf, None, p, inv, pairs)
    assert (table - mine).abs().max().item() <= 2e-6 * qf.abs().max().item()   # the table's fp32 angles are off by 2^-24 of up to 33 radians


@pytest.mark.gpu
def test_gradient_against_differences(gpu):
    """Central differences in fp32 along random directions: truncation about step^2 = 6e-5, rounding 2^-24 sqrt(terms) / step."""
    q, k, p, inv, pairs, qw, kw = problem(gpu, 1, 9, 2, 3, 64, (16, 24, 24), torch.float32, "bhsd")
    opt = dict(norm=True, eps=1e-6, rope="split_half")
    cq, ck = torch.randn_like(q), torch.randn_like(k)
    grads = block_ops.axes_rope_backward(cq, ck, p, inv, pairs, q=q, k=k, q_weight=qw, k_weight=kw, **opt)
    arg = dict(q=q, k=k, q_weight=qw, k_weight=kw)

    def loss(**over):
        a = {**arg, **over}
        y, z = block_ops.axes_rope(a["q"], a["k"], p, inv, pairs, q_weight=a["q_weight"], k_weight=a["k_weight"], **opt)
        return (y.double() * cq).sum().item() + (z.double() * ck).sum().item()

    step = 2.0 ** -7
    for (name, t), grad in zip(arg.items(), grads):
        d = torch.randn_like(t)
        num = (loss(**{name: t + step * d}) - loss(**{name: t - step * d})) / (2 * step)
        prod = grad.double() * d
        assert abs(num - prod.sum().item()) <= 2e-3 * prod.abs().sum().item(), name


@pytest.mark.gpu
def test_bad_rows_stay_by_themselves_and_repeat(gpu):
    q, k, p, inv, pairs, qw, kw = problem(gpu, 1, 50, 6, 6, 128, (44, 42, 42), torch.bfloat16, "bshd")
    opt = dict(norm=True, q_weight=qw, k_weight=kw)
    ref = block_ops.axes_rope(q, k, p, inv, pairs, **opt)
    g = block_ops.axes_rope_backward(*ref, p, inv, pairs, q=q, k=k, **opt)
    g2 = block_ops.axes_rope_backward(*ref, p, inv, pairs, q=q, k=k, **opt)
    assert all(torch.equal(a, b) for a, b in zip(g, g2))
    q[0, 3, 7, 5] = float("nan")
    y, z = block_ops.axes_rope(q, k, p, inv, pairs, **opt)
    bad = ~(y == ref[0]).all(-1)
    assert bad.sum().item() == 1 and bad[0, 3, 7] and torch.equal(z, ref[1])
    zero = torch.zeros(1, 1, 2, 64, device=gpu)       # a row of zeros has no direction: eps keeps it at zero
    assert torch.equal(block_ops.axes_rope(zero, None, p[:2], *block_ops.rope_frequencies((16, 24, 24), device=gpu), norm=True)[0], zero)
    empty = block_ops.axes_rope(q[:, :, :0], k[:, :, :0], p[:0], inv, pairs)
    assert empty[0].shape == (1, 6, 0, 128)


@pytest.mark.gpu
def test_refusals(gpu):
    q, k, p, inv, pairs, qw, kw = problem(gpu, 2, 8, 2, 2, 128, (16, 56, 56), torch.bfloat16, "bhsd")
    f = block_ops.axes_rope
    for bad in (lambda: f(q[0], k, p, inv, pairs), lambda: f(q, k.float(), p, inv, pairs), lambda: f(q, k[:, :, :4], p, inv, pairs), lambda: f(q, k, p[:4], inv, pairs),
                lambda: f(q, k, p[:, :2], inv, pairs), lambda: f(q, k, p.double(), inv, pairs), lambda: f(q, k, p, inv[:3], pairs), lambda: f(q, k, p, inv.half(), pairs),
                lambda: f(q, k, p, inv, (64,)), lambda: f(q, k, p, inv, pairs, rope="wan"), lambda: f(q, k, p, inv, pairs, q_weight=qw),
                lambda: f(q, k, p, inv, pairs, norm=True, q_weight=qw[:64]), lambda: f(q, None, p, inv, pairs, k_weight=kw, norm=True), lambda: f(q, k, p.t().contiguous().t(), inv, pairs),
                lambda: f(q[..., ::2], k, p, inv, pairs), lambda: f(q, k, p, inv, pairs, norm=True, eps=-1.0), lambda: f(q, k, p, inv, pairs, out_q=q[:, :1].expand(2, 2, 8, 128)),
                lambda: block_ops.axes_rope_backward(q, k, p, inv, pairs, norm=True), lambda: block_ops.rope_frequencies((3, 4))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        f(q, k, p, *block_ops.rope_frequencies((2, 4, 4), device=gpu))
    with pytest.raises(RuntimeError):
        f(q.cpu(), k.cpu(), p.cpu(), inv.cpu(), pairs)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_no_rotated_pairs_leave_the_norm(gpu, dtype):
    q, k, p, _, _, qw, kw = problem(gpu, 2, 9, 3, 2, 72, (0, 36, 36), dtype, "bshd")
    inv, pairs = block_ops.rope_frequencies((0, 0, 0), device=gpu)
    opt = dict(norm=True, q_weight=qw, k_weight=kw, eps=1e-5)
    y, z = block_ops.axes_rope(q, k, p, inv, pairs, **opt)
    for x, w, got in ((q, qw, y), (k, kw, z)):
        ref = O.axes_rope(x, w, p, inv, pairs, True, 1e-5, "interleaved")
        close(got, ref, ref.abs().amax(-1, keepdim=True))
    got = block_ops.axes_rope_backward(y, z, p, inv, pairs, q=q, k=k, **opt)
    for x, w, d, dx in ((q, qw, y, got[0]), (k, kw, z, got[1])):
        rdx, _, sx, _ = O.axes_rope_backward(d, x, w, p, inv, pairs, True, 1e-5, "interleaved")
        close(dx, rdx, sx)
    assert torch.equal(block_ops.axes_rope(q, None, p, inv, pairs)[0], q)
