"""Attention's backward pass against its formula in float64, element by element, within the bounds that `oracle.grad_oracle.attn_bwd`
derives: half a step of the type (bf16 2^-8, fp16 2^-11, fp32 2^-24) for each of the roundings of P, dS and the result, and 2^-17 of the sizes
that a sum adds.  fp16 results below 2^-14 are multiples of 2^-24: 2^-25 more."""
import math

import pytest
import torch

from oracle import grad_oracle as O
from xdit_amd import attention_backend as AB
from xdit_amd import grad_ops, ops, ring, usp

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def rand(gpu, seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator(device=gpu).manual_seed(seed), device=gpu).to(dtype)


def inputs(gpu, B, H, Sq, Sk, D, Sk2=0, dtype="bf16", layout="bhsd", size=1.0, seed=0):
    dt = DT[dtype]

    def tensor(n, S, f=1.0):
        if layout == "bshd":
            return (f * rand(gpu, seed + n, B, S, H, D)).to(dt).transpose(1, 2)
        return (f * rand(gpu, seed + n, B, H, S, D)).to(dt)

    q, k, v, dout = tensor(1, Sq, 2.0), tensor(2, Sk), tensor(3, Sk), tensor(4, Sq, size)
    k2, v2 = (tensor(5, Sk2), tensor(6, Sk2)) if Sk2 else (None, None)
    kk, vv = (torch.cat((k, k2), 2), torch.cat((v, v2), 2)) if Sk2 else (k, v)
    out, lse = O.attn_fwd(q, kk, vv, D ** -0.5)
    return q, k, v, k2, v2, dout, out.to(dt), lse.float()


def bounds(q, k, v, k2, v2, dout, out, lse, dlse=None, scale=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    kk, vv = (torch.cat((k, k2), 2), torch.cat((v, v2), 2)) if k2 is not None else (k, v)
    half = torch.finfo(q.dtype).eps / 2
    (dq, dk, dv), (fq, fk, fv) = O.attn_bwd(dout, q, kk, vv, out, lse, scale, dlse, half if q.dtype != torch.float32 else 0.0)
    if q.dtype == torch.float16:
        fq, fk, fv = fq + 2.0 ** -25, fk + 2.0 ** -25, fv + 2.0 ** -25
    n = k.shape[2]
    if k2 is None:
        return (dq, dk, dv), (fq, fk, fv)
    return (dq, dk[:, :, :n], dv[:, :, :n], dk[:, :, n:], dv[:, :, n:]), (fq, fk[:, :, :n], fv[:, :, :n], fk[:, :, n:], fv[:, :, n:])


def close(got, want, far):
    for name, g, w, f in zip(("dq", "dk", "dv", "dk2", "dv2"), got, want, far):
        assert g.shape == w.shape
        over = (g.double() - w).abs() - f
        assert bool((over <= 0).all()), (name, float(over.max()), float(w.abs().max()))


def call(q, k, v, k2, v2, dout, out, lse, **kw):
    return grad_ops.attn_bwd(dout, q, k, v, out, lse, k2=k2, v2=v2, **kw)


SHAPES = [(1, 1, 64, 64, 0), (1, 2, 64, 256, 0), (2, 3, 130, 77, 0), (1, 1, 1, 1, 0), (1, 1, 1, 300, 0), (1, 2, 300, 1, 0), (1, 1, 257, 255, 1),
          (2, 2, 63, 65, 129), (1, 3, 513, 640, 31), (1, 1, 2, 2, 2)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [8, 32, 40, 64, 72, 80, 96, 104, 128])
def test_head_dims(gpu, dtype, D):
    t = inputs(gpu, 1, 2, 200, 150, D, 40, dtype, "bshd")
    close(call(*t), *bounds(*t))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("D,layout", [(128, "bhsd"), (64, "bshd")])
def test_lengths(gpu, dtype, shape, D, layout):
    B, H, Sq, Sk, Sk2 = shape
    t = inputs(gpu, B, H, Sq, Sk, D, Sk2, dtype, layout)
    close(call(*t), *bounds(*t))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("cus", [1, 7, 40, 4096])
def test_work_in_parts(gpu, dtype, cus, monkeypatch):
    """Launches planned for few and for many compute units: whole ranges, and ranges cut into parts that a second launch adds up."""
    monkeypatch.setitem(ops.TUNING, "cu_count", cus)
    for D, shape in ((128, (1, 2, 900, 500, 60)), (72, (1, 1, 50, 3000, 0)), (64, (1, 1, 3000, 50, 70))):
        B, H, Sq, Sk, Sk2 = shape
        t = inputs(gpu, B, H, Sq, Sk, D, Sk2, dtype)
        got = call(*t)
        close(got, *bounds(*t))
        assert all(torch.equal(a, b) for a, b in zip(got, call(*t)))   # the same bits again


def framed(t, rows=3, cols=8):
    """A tensor of t's values inside a larger one of NaN, and that one."""
    B, H, S, D = t.shape
    big = torch.full((B, H, S + 2 * rows, D + 2 * cols), math.nan, dtype=t.dtype, device=t.device)
    inner = big[:, :, rows:rows + S, cols:cols + D]
    inner.copy_(t)
    return inner, big


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("bf16", 72), ("fp16", 64), ("fp32", 40), ("fp32", 128)])
@pytest.mark.parametrize("cus", [0, 4096])
def test_nothing_outside_the_tensors_is_read_or_written(gpu, dtype, D, cus, monkeypatch):
    monkeypatch.setitem(ops.TUNING, "cu_count", cus)
    t = inputs(gpu, 2, 2, 190, 130, D, 35, dtype)
    want = call(*t)
    q, k, v, k2, v2, dout, out, lse = t
    fr = [framed(x)[0] for x in (q, k, v, k2, v2, dout, out)]
    wide = torch.full((2, 2, lse.shape[2] + 9), math.nan, device=gpu)
    wide[:, :, 4:-5] = lse
    results = [framed(torch.zeros_like(x)) for x in (q, k, v, k2, v2)]
    names = ("dq", "dk", "dv", "dk2", "dv2")
    got = call(*fr, wide[:, :, 4:-5], **{n: r[0] for n, r in zip(names, results)})
    for a, b, (inner, big) in zip(got, want, results):
        assert torch.equal(a, b) and a is inner
        assert int(big.isnan().sum()) == big.numel() - inner.numel()


def test_gradients_into_one_fused_buffer(gpu):
    """q, k, v as views of a projection's output, and their gradients as views of its gradient."""
    B, H, S, D = 2, 3, 140, 64
    qkv = rand(gpu, 1, B, S, 3, H, D, dtype=torch.bfloat16)
    q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
    out, lse = ops.attn_fwd(q, k, v)
    dout = rand(gpu, 2, B, S, H, D, dtype=torch.bfloat16).transpose(1, 2)
    want = grad_ops.attn_bwd(dout, q, k, v, out, lse)
    dqkv = torch.full_like(qkv, math.nan)
    dq, dk, dv = (dqkv[:, :, i].transpose(1, 2) for i in range(3))
    grad_ops.attn_bwd(dout, q, k, v, out, lse, dq=dq, dk=dk, dv=dv)
    assert all(torch.equal(a, b) for a, b in zip((dq, dk, dv), want))


def test_heads_that_share_keys(gpu):
    """Keys and values expanded over the heads (stride 0): every head has its own gradient."""
    q, k, v, _, _, dout, _, _ = inputs(gpu, 1, 4, 100, 90, 64)
    k, v = k[:, :1].expand(-1, 4, -1, -1), v[:, :1].expand(-1, 4, -1, -1)
    out, lse = O.attn_fwd(q, k, v, 64 ** -0.5)
    t = (q, k, v, None, None, dout, out.to(q.dtype), lse.float())
    close(call(*t), *bounds(*t))


@pytest.mark.parametrize("need_q,need_kv", [(True, False), (False, True)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_some_of_the_gradients(gpu, need_q, need_kv, dtype):
    t = inputs(gpu, 1, 2, 300, 200, 64, 50, dtype)
    every, some = call(*t), call(*t, need_q=need_q, need_kv=need_kv)
    assert [x is not None for x in some] == [need_q] + 4 * [need_kv]
    (want, far) = bounds(*t)   # the launches are cut up differently: each within its own bounds
    for got in (every, some):
        close(*zip(*((g, w, f) for g, w, f in zip(got, want, far) if g is not None)))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_gradient_of_the_log_sum_exp(gpu, dtype):
    t = inputs(gpu, 2, 2, 150, 100, 64, 20, dtype)
    dlse = rand(gpu, 9, 2, 2, 150)
    close(call(*t, dlse=dlse), *bounds(*t, dlse=dlse))
    turned = dlse.transpose(1, 2).contiguous().transpose(1, 2)   # other strides, and one value for all rows
    assert all(torch.equal(a, b) for a, b in zip(call(*t, dlse=dlse), call(*t, dlse=turned)))
    other = t[:7] + (t[7].transpose(1, 2).contiguous().transpose(1, 2),)
    assert all(torch.equal(a, b) for a, b in zip(call(*t, dlse=dlse), call(*other, dlse=dlse)))
    one = torch.tensor(0.5, device=gpu).expand(2, 2, 150)
    close(call(*t, dlse=one), *bounds(*t, dlse=one))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape", [(1, 1, 4100, 3, 0), (1, 1, 5, 4000, 0), (3, 1, 2500, 9, 2), (1, 2, 1000, 1100, 0)])
@pytest.mark.parametrize("D", [72, 128])
def test_few_tiles_for_the_whole_chip(gpu, shape, D, dtype):
    """Fewer tiles than XCDs, cut into many parts."""
    B, H, Sq, Sk, Sk2 = shape
    t = inputs(gpu, B, H, Sq, Sk, D, Sk2, dtype)
    close(call(*t), *bounds(*t))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_rows_that_attended_nothing(gpu, dtype):
    q, k, v, _, _, dout, out, lse = inputs(gpu, 1, 2, 150, 100, 64, 0, dtype)
    lse[:, 0, 10:20] = lse[:, 1, 149] = -math.inf
    t = (q, k, v, None, None, dout, out, lse)
    got = call(*t)
    close(got, *bounds(*t))
    assert not got[0][:, 0, 10:20].any() and not got[0][:, 1, 149].any()


@pytest.mark.parametrize("size", [2.0 ** -14, 2.0 ** -8, 1.0, 64.0, 1024.0])
def test_fp16_gradients_of_every_size(gpu, size):
    """P and dS are scaled with the size of dout: small gradients lose no bits beside the result's own."""
    t = inputs(gpu, 1, 2, 700, 1500, 64, 0, "fp16", size=size)
    close(call(*t), *bounds(*t))


def test_fp16_scores_stay_in_range(gpu):
    """dS near fp16's end: values of 500 that all add up, and a gradient of the log-sum-exp far above dout."""
    k, v = rand(gpu, 1, 1, 1, 2, 128).half(), torch.tensor([500.0, -500.0], device=gpu).view(1, 1, 2, 1).expand(1, 1, 2, 128).half().contiguous()
    q, dout = (0.1 * rand(gpu, 2, 1, 1, 64, 128)).half(), torch.full((1, 1, 64, 128), 0.98, dtype=torch.float16, device=gpu)
    out, lse = O.attn_fwd(q, k, v, 128 ** -0.5)
    t = (q, k, v, None, None, dout, out.half(), lse.float())
    close(call(*t), *bounds(*t))
    t = inputs(gpu, 1, 2, 70, 3, 64, 0, "fp16", size=1e-3)
    dlse = 50 * rand(gpu, 3, 1, 2, 70)
    close(call(*t, dlse=dlse), *bounds(*t, dlse=dlse))


def test_large_logits(gpu):
    """Rows whose probability is one key's."""
    q, k, v, _, _, dout, _, _ = inputs(gpu, 1, 2, 200, 190, 64)
    q = 30 * q
    out, lse = O.attn_fwd(q, k, v, 64 ** -0.5)
    t = (q, k, v, None, None, dout, out.to(q.dtype), lse.float())
    close(call(*t), *bounds(*t))


def test_not_a_number_stays_in_its_rows(gpu):
    """An infinity or a NaN in one query's gradient reaches that query's dq and all of dk and dv of its head, and no other head."""
    q, k, v, k2, v2, dout, out, lse = inputs(gpu, 1, 3, 150, 100, 64)
    clean = call(q, k, v, k2, v2, dout, out, lse)
    dout = dout.clone()
    dout[0, 1, 70, 5] = math.nan
    dq, dk, dv = call(q, k, v, k2, v2, dout, out, lse)
    for h in (0, 2):
        assert all(torch.equal(a[:, h], b[:, h]) for a, b in zip((dq, dk, dv), clean))
    rest = [i for i in range(150) if i != 70]
    assert torch.equal(dq[0, 1, rest], clean[0][0, 1, rest]) and bool(dq[0, 1, 70].isnan().all()) and bool(dv[0, 1, :, 5].isnan().all())


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("fp16", 64), ("fp32", 72)])
def test_chunks_of_a_ring(gpu, dtype, D):
    """With the whole ring's output and log-sum-exp a chunk of keys has its own dk and dv, and the chunks' dq add up."""
    t = inputs(gpu, 1, 2, 200, 360, D, 0, dtype)
    q, k, v, _, _, dout, out, lse = t
    (dq, dk, dv), (fq, fk, fv) = bounds(*t)
    parts = [call(q, k[:, :, s], v[:, :, s], None, None, dout, out, lse) for s in (slice(0, 120), slice(120, 240), slice(240, 360))]
    close([sum(p[0].double() for p in parts)], [dq], [fq + 3 * torch.finfo(q.dtype).eps * sum(p[0].double().abs() for p in parts)])
    close([torch.cat([p[i] for p in parts], 2) for i in (1, 2)], [dk, dv], [fk, fv])


@pytest.mark.parametrize("scale", [0.01, 1.0])
def test_softmax_scale(gpu, scale):
    q, k, v, _, _, dout, _, _ = inputs(gpu, 1, 2, 100, 130, 64)
    out, lse = O.attn_fwd(q, k, v, scale)
    t = (q, k, v, None, None, dout, out.to(q.dtype), lse.float())
    close(call(*t, softmax_scale=scale), *bounds(*t, scale=scale))


def test_long_rows(gpu):
    """A whole head of 17776 tokens, probed row by row."""
    t = inputs(gpu, 1, 1, 4000, 17776, 64, 0, "bf16")
    close(call(*t), *bounds(*t))


def test_offsets_beyond_32_bits(gpu):
    """Heads that lie more than 2^32 bytes apart."""
    H, S, D = 3, 200, 64
    far = (1 << 31) + 512   # elements between heads, 2^32 bytes and more
    store = [torch.empty(2 * far + S * D, dtype=torch.bfloat16, device=gpu) for _ in range(2)]
    q, k, v, _, _, dout, out, lse = inputs(gpu, 1, H, S, S, D)
    want = grad_ops.attn_bwd(dout, q, k, v, out, lse)

    def spread(x, buf):
        y = buf.as_strided((1, H, S, D), (3 * far, far, D, 1))
        return y.copy_(x) if x is not None else y

    a = spread(k, store[0])
    got = grad_ops.attn_bwd(dout, q, a, v, out, lse, dk=spread(None, store[1]))
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_other_stream_and_replayed_graph(gpu):
    t = inputs(gpu, 1, 2, 500, 300, 64, 50, "fp16")
    want = call(*t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(*t)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):   # two graphs of the same call, side by side with eager ones
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call(*t)
        graphs.append((g, out))
    q = t[0].clone()
    for n in range(4):
        t[0].copy_(q * (1 + n))
        eager = call(*t)
        for g, out in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:   # bit by bit: under the log-sum-exp of other queries P overflows from the second pass on
            assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(out, eager))
        assert n or all(x.isfinite().all() for x in eager)


# ---- through the attention calls -----------------------------------------------------------------------


def leaves(*ts):
    return [t.detach().clone().requires_grad_() for t in ts]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_gradient_of_the_attention_call(gpu, dtype):
    t = inputs(gpu, 1, 2, 150, 100, 64, 0, dtype)
    q, k, v, _, _, dout, _, _ = t
    plain, lse = ops.attn_fwd(q, k, v)
    lq, lk, lv = leaves(q, k, v)
    o = usp.attention(lq, lk, lv)
    assert torch.equal(o, plain)
    got = torch.autograd.grad(o, (lq, lk, lv), dout)
    assert all(torch.equal(a, b) for a, b in zip(got, grad_ops.attn_bwd(dout, q, k, v, plain, lse)))
    # one operand, a gradient expanded from a scalar, the log-sum-exp alone
    o, l = AB._mi355_attn_call(q, lk, v, 0.0, False)
    (dk,) = torch.autograd.grad(o.sum() + l.square().sum(), (lk,))
    ones = torch.ones_like(plain)
    assert torch.equal(dk, grad_ops.attn_bwd(ones, q, k, v, plain, lse, dlse=2 * lse, need_q=False)[1])
    o, l = AB._mi355_attn_call(lq, k, v, 0.0, False)
    (dq,) = torch.autograd.grad(l.sum(), (lq,))
    assert torch.equal(dq, grad_ops.attn_bwd(torch.zeros_like(plain), q, k, v, plain, lse, dlse=torch.ones_like(lse), need_kv=False)[0])
    with torch.no_grad():
        assert not usp.attention(lq, lk, lv).requires_grad


@pytest.mark.parametrize("strategy", ["rear", "front"])
@pytest.mark.parametrize("chunks", [1, 4])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_gradient_of_joint_attention_and_of_the_ring(gpu, strategy, chunks, dtype):
    """USP with text tokens, in one call and as a ring: the outputs of the calls without gradients, and the formula's gradients."""
    D = 64
    q, k, v, k2, v2, _, _, _ = inputs(gpu, 1, 2, 160, 160, D, 40, dtype)
    q2 = rand(gpu, 30, 1, 2, 40, D, dtype=q.dtype)
    ts = (q, k, v, q2, k2, v2)
    joint = dict(zip(("joint_query", "joint_key", "joint_value"), (q2, k2, v2)), joint_strategy=strategy, ring_chunks=chunks)
    plain = usp.USP(q, k, v, **joint)
    lq, lk, lv, lq2, lk2, lv2 = ls = leaves(*ts)
    o = usp.USP(lq, lk, lv, joint_query=lq2, joint_key=lk2, joint_value=lv2, joint_strategy=strategy, ring_chunks=chunks)
    assert torch.equal(o, plain)
    dout = rand(gpu, 31, *o.shape, dtype=o.dtype)
    got = torch.autograd.grad(o, ls, dout)
    qq = torch.cat((q, q2) if strategy == "rear" else (q2, q), 2)
    _, lse = ops.attn_fwd(qq, k, v, k2=k2, v2=v2)
    (dq, *dkv), (fq, *fkv) = bounds(qq, k, v, k2, v2, dout, o.detach(), lse)
    n = 160 if strategy == "rear" else 40
    dq, fq = ((x[:, :, :n], x[:, :, n:]) for x in (dq, fq))
    if strategy == "front":
        dq, fq = dq[::-1], fq[::-1]
    # the ring's own log-sum-exp: off by a few steps of 2^-24 of its size, which the bound of P covers
    close((got[0], got[1], got[2], got[4], got[5]), (dq[0], *dkv), (fq[0], *fkv))
    close((got[3],), (dq[1],), (fq[1],))


def ring_call(**joint):
    """The ring over four chunks, with joint keys as `joint` says -> a function of (q, k, v, joint key, joint value)."""
    def f(q, k, v, k2, v2, order=None, chunks=4):
        kw = dict(joint_key=k2, joint_value=v2, **joint) if joint else None
        return usp.ring_attn(usp._get_attention_function(), q, k, v, joint_attn_kwargs=kw, ring_chunks=chunks, order=order)
    return f


def test_no_gradient_of_a_ring_is_lost(gpu):
    """Whichever one tensor asks for a gradient."""
    ts = [rand(gpu, i, 1, 2, 32, 64, dtype=torch.bfloat16) for i in range(5)]
    for chunks in (1, 4):
        for i in range(5):
            one = [t.clone().requires_grad_(j == i) for j, t in enumerate(ts)]
            o = ring_call(joint_strategy="front", total_steps=chunks)(*one, chunks=chunks)
            (g,) = torch.autograd.grad(o.square().sum(), one[i:i + 1])
            assert bool(g.any())


@pytest.mark.parametrize("joint", [dict(joint_strategy="front", step=1), dict(joint_strategy="rear", total_steps=9), dict(joint_strategy="none")])
def test_joint_keys_that_no_step_takes(gpu, joint):
    q, k, v, k2, v2, dout, _, _ = inputs(gpu, 1, 2, 60, 80, 64, 20)
    ls = leaves(q, k, v, k2, v2)
    got = torch.autograd.grad(ring_call(**joint)(*ls), ls, dout, allow_unused=True)
    want = torch.autograd.grad(ring_call()(*ls), ls[:3], dout)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[3] is None and got[4] is None


def test_ring_that_takes_a_chunk_twice(gpu):
    q, k, v, _, _, dout, _, _ = inputs(gpu, 1, 2, 60, 80, 64)
    ls = leaves(q, k, v)
    order = [0, 2, 2, 1]
    o = ring_call()(*ls, None, None, order=order)
    dq, dk, dv = torch.autograd.grad(o, ls, dout)
    kk, vv = (torch.cat([t.chunk(4, 2)[c] for c in order], 2) for t in (k, v))
    lse = ops.attn_fwd(q, kk, vv)[1]
    (wq, wk, wv), (fq, fk, fv) = bounds(q, kk, vv, None, None, dout, o.detach(), lse)
    close((dq,), (wq,), (fq,))
    for got, w, f in ((dk, wk, fk), (dv, wv, fv)):
        w, f = w.chunk(4, 2), f.chunk(4, 2)
        both = w[1] + w[2]
        close((got,), (torch.cat((w[0], w[3], both, torch.zeros_like(both)), 2),),
              (torch.cat((f[0], f[3], f[1] + f[2] + 2.0 ** -8 * both.abs(), torch.zeros_like(both)), 2),))   # and their sum's own rounding
    with pytest.raises(ValueError, match="order"):
        ring_call()(*ls, None, None, order=[0, 1, 2])


@pytest.mark.parametrize("joint", [{}, dict(joint_strategy="rear", total_steps=4)])
def test_compiled_ring_has_the_eager_gradient(gpu, joint):
    q, k, v, k2, v2, dout, _, _ = inputs(gpu, 1, 2, 60, 80, 64, 20)
    ls = leaves(q, k, v, *((k2, v2) if joint else ()))
    rest = () if joint else (None, None)
    eager = ring_call(**joint)(*ls, *rest)
    traced = torch.compile(ring_call(**joint), backend="aot_eager", fullgraph=True)(*ls, *rest)
    assert torch.equal(eager, traced)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(traced, ls, dout), torch.autograd.grad(eager, ls, dout)))


@pytest.mark.parametrize("call", [ring.flash_attn_forward, lambda q, k, v: ring.xdit_ring_flash_attn_func(q, k, v, group=ring.LocalRing(2), return_attn_probs=True)[:2]])
def test_compiled_ring_on_bshd_tensors(gpu, call):
    ls = leaves(*(rand(gpu, i, 1, 64, 2, 32, dtype=torch.bfloat16) for i in range(3)))
    dout, dlse = rand(gpu, 3, 1, 64, 2, 32, dtype=torch.bfloat16), rand(gpu, 4, 1, 2, 64)
    eager, traced = call(*ls), torch.compile(call, backend="aot_eager")(*ls)
    assert all(torch.equal(a, b) for a, b in zip(eager, traced))
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(traced, ls, (dout, dlse)), torch.autograd.grad(eager, ls, (dout, dlse))))


def test_second_gradients_are_refused(gpu):
    q, k, v, _, _, dout, _, _ = inputs(gpu, 1, 2, 20, 30, 64)
    for call in (usp.attention, lambda *t: ring_call()(*t[:1], *(x[:, :, :28] for x in t[1:]), None, None)):
        ls = leaves(q, k, v)
        (dq,) = torch.autograd.grad(call(*ls), ls[:1], dout, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(dq.sum(), ls[1:2])


@pytest.mark.parametrize("world", [1, 2])
@pytest.mark.parametrize("joint", [False, True])
def test_gradient_of_the_ring_on_bshd_tensors(gpu, world, joint):
    B, H, S, D = 2, 2, 128, 32
    q, k, v, jk, jv = (rand(gpu, i, B, S, H, D, dtype=torch.float16) for i in range(5))
    dout = rand(gpu, 9, B, S, H, D, dtype=torch.float16)
    kw = dict(joint_strategy="rear") if joint else {}
    ls = leaves(q, k, v, *((jk, jv) if joint else ()))
    if joint:
        kw.update(joint_tensor_key=ls[3], joint_tensor_value=ls[4])
    o, lse, _ = ring.xdit_ring_flash_attn_func(*ls[:3], group=ring.LocalRing(world), return_attn_probs=True, **kw)
    with torch.no_grad():
        assert torch.equal(o, ring.xdit_ring_flash_attn_func(*ls[:3], group=ring.LocalRing(world), **kw)) and o.is_contiguous()
    got = torch.autograd.grad(o, ls, dout)
    t = lambda x: None if x is None else x.transpose(1, 2)  # noqa: E731
    want, far = bounds(t(q), t(k), t(v), t(jk) if joint else None, t(jv) if joint else None, t(dout), t(o.detach()), lse)
    close([t(x) for x in got], want, far)
    layer = ring.xFuserLongContextAttention(ring_group=ring.LocalRing(world))
    if not joint:
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(layer(None, *ls), ls, dout), got))


def test_gradient_against_differences(gpu):
    """Along random directions, fp32: (L(x + h d) - L(x - h d)) / 2h.  L is a sum of 2 * 60 * 64 = 7680 outputs of size 1 times weights of size 1, off
    by about sqrt(7680) * 2^-21 = 4e-5, which 2h = 0.02 makes 2e-3; the third derivative's h^2 / 6 adds about 2e-5 of a size of 100.  Held to 1e-2."""
    q, k, v, _, _, _, _, _ = inputs(gpu, 1, 2, 60, 50, 64, 0, "fp32")
    w, wl = rand(gpu, 40, 1, 2, 60, 64), rand(gpu, 41, 1, 2, 60)

    def loss(q, k, v):
        o, l = AB._mi355_attn_call(q, k, v, 0.0, False)
        return (o.double() * w).sum() + (l.double() * wl).sum()

    ls = leaves(q, k, v)
    grads = torch.autograd.grad(loss(*ls), ls)
    h = 0.01
    for i in range(3):
        d = rand(gpu, 50 + i, *ls[i].shape)
        d /= d.norm()
        with torch.no_grad():
            moved = [[x + (s * h * d if j == i else 0) for j, x in enumerate((q, k, v))] for s in (1, -1)]
            slope = float(loss(*moved[0]) - loss(*moved[1])) / (2 * h)
        assert abs(slope - float((grads[i].double() * d).sum())) <= 1e-2


def test_compiled_call_has_the_eager_gradient(gpu):
    q, k, v, _, _, dout, _, _ = inputs(gpu, 1, 2, 100, 80, 64)
    eager, traced = leaves(q, k, v), leaves(q, k, v)
    want = torch.autograd.grad(usp.attention(*eager), eager, dout)
    f = torch.compile(usp.attention, backend="aot_eager", fullgraph=True)
    got = torch.autograd.grad(f(*traced), traced, dout)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(gpu):
    q, k, v, _, _, dout, out, lse = inputs(gpu, 1, 2, 64, 64, 64)
    with pytest.raises(ValueError, match="shape"):
        grad_ops.attn_bwd(dout, q[..., 1:], k[..., 1:], v[..., 1:], out, lse)
    with pytest.raises(ValueError):
        grad_ops.attn_bwd(dout.expand(1, 2, 64, 64)[:, :, :1].expand(1, 2, 64, 64), q, k, v, out, lse)   # rows on one another
    with pytest.raises(ValueError, match="overlap"):
        grad_ops.attn_bwd(dout, q, k, v, out, lse, dq=torch.empty_like(q)[:, :1].expand(1, 2, 64, 64))
    with pytest.raises(NotImplementedError):
        f8 = torch.float8_e4m3fn
        grad_ops.attn_bwd(dout.to(f8), q.to(f8), k.to(f8), v.to(f8), out.to(f8), lse)
    with pytest.raises(NotImplementedError, match="head_dim"):
        w = torch.zeros(1, 2, 64, 256, dtype=q.dtype, device=gpu)
        grad_ops.attn_bwd(w, w, w, w, w, lse)
