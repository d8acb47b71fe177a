"""The differentiable and module forms of the operators around the attention call, and a whole block made of them.

Bars.  float32 gradients are compared to float64 autograd of the formula: an element is off by less than 64 units of 2^-24 of its terms, and a
sum over up to 120 rows of terms of random sign by that of the sum of their sizes, about sqrt(120) = 11 times a typical sum: 64 * 11 * 2^-24 = 2^-14.5,
held to 2^-12 of the largest element.  A block's fp8 values are off by up to 1/16 of their size, 1/16/sqrt(3) = 0.036 in the root mean square.  Each branch
passes two of those steps and the softmax or activation between them (logits of a deviation of 1 move by 0.05), so what the block adds
is off by about sqrt(4 * 0.036^2 + 0.05^2) = 0.09: held to 0.12.  A gradient passes the four products once more: sqrt(2) * 0.09 = 0.13, held to 0.2.
"""
import importlib.util
import os

import pytest
import torch

from xdit_amd import block, block_ops, custom_ops  # noqa: F401

spec = importlib.util.spec_from_file_location("dit_block", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "dit_block.py"))
dit = importlib.util.module_from_spec(spec)
spec.loader.exec_module(dit)
pytestmark = pytest.mark.gpu


def near(got, ref):
    for a, b in zip(got, ref):
        assert a.shape == b.shape
        assert float((a.double() - b).abs().max()) <= 2.0 ** -12 * float(b.abs().max())


def rand(gpu, *shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator(device=gpu).manual_seed(seed + len(shape) + shape[-1]), device=gpu).to(dtype)


def norm64(x, y, gate, scale, shift, weight, bias, y_weight, kind, y_kind):
    def norm(t, k):
        t = t - t.mean(-1, keepdim=True) if k == "layer" else t
        return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6)
    rows = [t if t.ndim == 3 else t.unsqueeze(1) for t in (gate, scale, shift)]
    h = x + rows[0] * (norm(y, y_kind) * y_weight if y_kind else y * y_weight)
    return h, (norm(h, kind) * weight + bias) * (1 + rows[1]) + rows[2]


@pytest.mark.parametrize("kind,y_kind", [("layer", "rms"), ("rms", "layer")])
@pytest.mark.parametrize("mods", [((2, 1), (2, 1), (2, 1)), ((1, 1), (1,), (2, 60)), ((1, 60), (2, 60), (1, 1)), ((2,), (2, 60), (2,))])
def test_norm_gradients_with_broadcast_modulation(gpu, kind, y_kind, mods):
    C = 72
    shapes = [(2, 60, C), (2, 60, C), *((*m, C) for m in mods), (C,), (C,), (C,)]
    t = [rand(gpu, *s, seed=7 * i).requires_grad_() for i, s in enumerate(shapes)]
    x, y, gate, scale, shift, weight, bias, y_weight = t
    r = rand(gpu, 2, 60, C, seed=90), rand(gpu, 2, 60, C, seed=91)
    h, n = block.gated_norm(x, y, gate, scale, shift, weight, bias, kind, 1e-6, y_kind, y_weight, 1e-6)
    assert torch.equal(h, block_ops.gated_norm(*(v.detach() for v in (x, y, gate, scale, shift, weight, bias)), kind, 1e-6, y_kind, y_weight.detach(), 1e-6)[0])
    got = torch.autograd.grad((h, n), t, r)
    t64 = [v.detach().double().requires_grad_() for v in t]
    near(got, torch.autograd.grad(norm64(*t64, kind, y_kind), t64, [v.double() for v in r]))


def test_norm_gradients_of_one_result(gpu):
    """Only h, only n, no y, no norm; and a gradient that was expanded from a scalar."""
    x, y, g = (rand(gpu, 2, 9, 64, seed=i).requires_grad_() for i in range(3))
    s = rand(gpu, 2, 64, seed=5).requires_grad_()
    x64, y64, g64, s64 = (t.detach().double().requires_grad_() for t in (x, y, g, s))
    ln = lambda t: torch.nn.functional.layer_norm(t, (64,), eps=1e-6)  # noqa: E731
    for fn, ref, a, b in (
            (lambda: block.gated_norm(x, y, g, norm=None)[0].sum(), lambda: (x64 + g64 * y64).sum(), (x, y, g), (x64, y64, g64)),
            (lambda: block.gated_norm(x, y, g, s)[0].square().sum(), lambda: (x64 + g64 * y64).square().sum(), (x, y, g), (x64, y64, g64)),
            (lambda: block.gated_norm(x, y, scale=s)[1].pow(3).sum(), lambda: (ln(x64 + y64) * (1 + s64.unsqueeze(1))).pow(3).sum(), (x, y, s), (x64, y64, s64)),
            (lambda: (block.gated_norm(x, scale=s)[1].pow(3) + x).sum(), lambda: ((ln(x64) * (1 + s64.unsqueeze(1))).pow(3) + x64).sum(), (x, s), (x64, s64))):
        near(torch.autograd.grad(fn(), a), torch.autograd.grad(ref(), b))
    h, n = block.gated_norm(x, scale=s)
    assert torch.equal(h, x) and block.gated_norm(x, y, norm=None)[1] is None
    with pytest.raises(ValueError, match="no gradient"):
        block.gated_norm(x, fp8=True)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("rope", ["interleaved", "split_half"])
def test_rotation_gradients(gpu, norm, rope):
    B, H, Hk, S, D = 2, 3, 1, 20, 24
    freq, pairs = block.rope_frequencies((8, 8), device=gpu)
    pos = torch.stack([torch.arange(S, device=gpu) // 5, torch.arange(S, device=gpu) % 5 - 2], -1)
    q, k = rand(gpu, B, S, H, D).transpose(1, 2).requires_grad_(), rand(gpu, B, Hk, S, D, seed=3).requires_grad_()
    w = [rand(gpu, D, seed=s).requires_grad_() for s in (8, 9)] if norm else []
    r = rand(gpu, B, H, S, D, seed=11), rand(gpu, B, Hk, S, D, seed=12)
    oq, ok = block.axes_rope(q, k, pos, freq, pairs, norm, *(w or (None, None)), rope=rope)
    got = torch.autograd.grad((oq, ok), (q, k, *w), r)

    def turn(t, gain):
        if norm:
            t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * gain
        phi = torch.cat([pos[:, :1] * freq[:4], pos[:, 1:] * freq[4:]], -1)
        a, b = (t[..., 0:16:2], t[..., 1:16:2]) if rope == "interleaved" else (t[..., :8], t[..., 8:16])
        u, v = a * phi.cos() - b * phi.sin(), a * phi.sin() + b * phi.cos()
        return torch.cat([torch.stack((u, v), -1).flatten(-2) if rope == "interleaved" else torch.cat((u, v), -1), t[..., 16:]], -1)

    t64 = [t.detach().double().requires_grad_() for t in (q, k, *w)]
    out = turn(t64[0], t64[2] if norm else None), turn(t64[1], t64[3] if norm else None)
    near((oq, ok), [t.detach() for t in out])
    near(got, torch.autograd.grad(out, t64, [t.double() for t in r]))
    one, none = block.axes_rope(q, None, pos, freq, pairs, norm, w[0] if w else None, rope=rope)
    assert none is None and torch.equal(one, oq)
    near(torch.autograd.grad(one.sum(), q), torch.autograd.grad(turn(t64[0], t64[2] if norm else None).sum(), t64[0]))


def test_projection(gpu, tmp_path):
    lin = torch.nn.Linear(400, 208, device=gpu, dtype=torch.bfloat16)
    m = block.Fp8Linear.from_linear(lin, backward=True)
    x = rand(gpu, 2, 30, 400, dtype=torch.bfloat16)
    x8, xs = block_ops.fp8_block_quant(x)
    want = block_ops.fp8_block_matmul(x8, xs, m.weight, m.weight_scale, lin.bias.detach().float())
    assert torch.equal(m(x), want) and torch.equal(m((x8, xs)), want) and torch.equal(m(x.flatten(0, 1)), want.flatten(0, 1))
    assert m(x.float()).dtype == torch.float32
    # the gradient to x, also from an expanded one, is dy's product with the transposed weight
    v = x.clone().requires_grad_()
    dy = rand(gpu, 2, 30, 208, dtype=torch.bfloat16)
    d8, ds = block_ops.fp8_block_quant(dy)
    assert torch.equal(m(v), want)
    assert torch.equal(torch.autograd.grad(m(v), v, dy)[0], block_ops.fp8_block_matmul(d8, ds, m.weight_t, m.weight_t_scale))
    ones8, ones = block_ops.fp8_block_quant(torch.ones_like(dy))
    assert torch.equal(torch.autograd.grad(m(v).sum(), v)[0], block_ops.fp8_block_matmul(ones8, ones, m.weight_t, m.weight_t_scale))
    with pytest.raises(RuntimeError, match="transposed weight"):
        torch.autograd.grad(block.Fp8Linear.from_linear(lin)(v).sum(), v)
    # a model's change of type leaves the bytes and the scales, a saved state brings them back
    model = torch.nn.Sequential(m).half()
    assert m.weight.dtype == torch.float8_e4m3fn and m.weight_scale.dtype == m.bias.dtype == torch.float32
    torch.save(model.state_dict(), tmp_path / "m.pt")
    other = torch.nn.Sequential(block.Fp8Linear.from_linear(torch.nn.Linear(400, 208, device=gpu, dtype=torch.bfloat16), backward=True))
    assert not torch.equal(other(x), want)
    other.load_state_dict(torch.load(tmp_path / "m.pt", weights_only=True))
    assert torch.equal(other(x), want)
    assert torch.equal(m.cpu().weight_scale.to(gpu), other[0].weight_scale) and torch.equal(m.to(gpu)(x), want)


def test_registered_ops(gpu):
    """torch's own checks of schema, fake results and gradients' registration.  (Its schema check hashes the inputs with arithmetic that
    fp8 tensors do not have.)"""
    tests = ("test_schema", "test_faketensor", "test_autograd_registration")
    o = torch.ops.xdit_amd
    bf = torch.bfloat16
    x, y = rand(gpu, 2, 9, 200, dtype=bf), rand(gpu, 2, 9, 200, seed=1, dtype=bf)
    c, w = rand(gpu, 2, 1, 200, seed=2), rand(gpu, 200, seed=3, dtype=bf)
    for first in (x, x.clone().requires_grad_()):
        for args in ((first, y, c, c, c, w, w, w, "layer", 1e-6, "rms", 1e-6, 1.0), (first, None, None, c, None, None, None, None, "rms", 1e-6, "none", 1e-6, 1.0),
                     (first, y, c, None, None, None, None, None, "none", 1e-6, "none", 1e-6, 0.5)):
            torch.library.opcheck(o.gated_norm.default, args, test_utils=tests)
    torch.library.opcheck(o.gated_norm_fp8.default, (x, y, c, c, c, w, w, w, "layer", 1e-6, "rms", 1e-6, 1.0), test_utils=tests)
    st = o.gated_norm(x, y, c, c, c, w, w, w, "layer", 1e-6, "rms", 1e-6, 1.0)[2]
    for dh, dn in ((x, y), (None, y), (x, None)):
        torch.library.opcheck(o.gated_norm_backward.default, (dh, dn, x, st, y, c, c, c, w, w, w, "layer", "rms", 1.0), test_utils=tests)
    q, k = rand(gpu, 2, 9, 3, 64, dtype=bf).transpose(1, 2), rand(gpu, 2, 1, 9, 64, dtype=bf)
    freq, pairs = block.rope_frequencies((32, 32), device=gpu)
    pos, g = dit.grid_positions(1, 3, 3, gpu)[:, 1:].contiguous(), rand(gpu, 64, dtype=bf)
    for kk in (k, None):
        torch.library.opcheck(o.axes_rope.default, (q, kk, pos, freq, list(pairs), True, g, None if kk is None else g, 1e-6, "split_half"), test_utils=tests)
        torch.library.opcheck(o.axes_rope_backward.default, (q, kk, pos, freq, list(pairs), q, kk, True, g, None if kk is None else g, 1e-6, "split_half"), test_utils=tests)
    for t, rows in ((x, 1), (x[0], 1), (x[0], 128)):
        torch.library.opcheck(o.fp8_block_quant.default, (t, rows), test_utils=tests)
    m = block.Fp8Linear(rand(gpu, 144, 208, dtype=bf), backward=True)
    x8, xs = block_ops.fp8_block_quant(rand(gpu, 7, 208, dtype=bf))
    fake = ("test_faketensor", "test_autograd_registration")
    torch.library.opcheck(o.fp8_block_matmul.default, (x8, xs, m.weight, m.weight_scale, None, torch.float16, None), test_utils=fake)
    torch.library.opcheck(o.fp8_linear.default, (rand(gpu, 7, 208, dtype=bf), m.weight, m.weight_scale, m.weight_t, m.weight_t_scale, m.bias), test_utils=fake)


@pytest.mark.parametrize("grid,heads,head_dim,mlp,batch,dtype", [((1, 17, 13), 4, 64, 512, 2, torch.bfloat16), ((3, 5, 9), 5, 128, 1104, 1, torch.float16)])
def test_block(gpu, grid, heads, head_dim, mlp, batch, dtype):
    m = dit.DiTBlock(heads, head_dim, mlp, dtype, gpu)
    data = dit.inputs(grid, heads, head_dim, batch, dtype, gpu)
    assert dit.check(m, *data) <= 0.12
    with torch.no_grad():
        want = m(*data)
        assert torch.equal(m(*data), want)
        # compiled: one graph, the same bits
        assert torch.equal(torch.compile(lambda *a: block.gated_norm(*a)[1], backend="aot_eager", fullgraph=True)(data[0], data[0]), block.gated_norm(data[0], data[0])[1])
        up = lambda x: m.up(block.gated_norm(x, fp8=True)[1])  # noqa: E731
        assert torch.equal(torch.compile(up, backend="aot_eager", fullgraph=True)(data[0]), up(data[0]))
        # captured: every replay gives the eager result, with other work and new data between the replays
        x, mods, pos = (t.clone() for t in data)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            m(x, mods, pos)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = m(x, mods, pos)
        for i in range(4):
            x.copy_(data[0] * (1 + 0.5 * i))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, m(x, mods, pos))


def test_block_gradients(gpu):
    m = dit.DiTBlock(3, 64, 400, torch.bfloat16, gpu, train=True)
    data = dit.inputs((2, 7, 9), 3, 64, 2, torch.bfloat16, gpu)
    got = dit.check_gradients(m, *data)
    assert set(got) == {"x", "modulation", "q_gain", "k_gain"} and max(got.values()) <= 0.2, got
    # a compiled norm, rotation and projection: the same gradients
    x = data[0].clone().requires_grad_()

    def part(x):
        h, n = block.gated_norm(x, scale=data[1][:, :1])
        qkv = m.qkv(n).view(2, -1, 3, 3, 64)
        q, k = block.axes_rope(qkv[:, :, 0].transpose(1, 2), qkv[:, :, 1].transpose(1, 2), data[2], m.freq, m.pairs, True, m.q_gain, m.k_gain)
        return (q.float() * k.float()).sum()

    want = torch.autograd.grad(part(x), (x, m.q_gain, m.k_gain))
    for a, b in zip(torch.autograd.grad(torch.compile(part, backend="aot_eager", fullgraph=True)(x), (x, m.q_gain, m.k_gain)), want):
        assert torch.equal(a, b)


def test_graphs_of_one_stream_replayed_side_by_side(gpu, monkeypatch):
    """Two graphs captured on the same stream hold different scratch, and replays of them on two streams, beside eager calls on the
    stream of the capture, give the eager bits."""
    g = torch.Generator(device=gpu).manual_seed(3)
    rn = lambda *s: torch.randn(*s, generator=g, device=gpu)  # noqa: E731
    w, ws = block_ops.fp8_block_quant(rn(640, 4096) / 64, 128)
    h, dn, y = (rn(1, 3000, 640).bfloat16() for _ in range(3))
    scale, gate = rn(1, 640), rn(1, 640)
    st = block_ops.gated_norm(h, scale=scale, return_stats=True)[2]
    q, d, gain = rn(1, 5, 700, 128).bfloat16(), rn(1, 5, 700, 128).bfloat16(), rn(128)
    inv, pairs = block_ops.rope_frequencies((44, 42, 42), device=gpu)
    pos = torch.arange(2100, device=gpu).view(700, 3)

    def work(x):
        y8 = block_ops.fp8_block_matmul(*block_ops.fp8_block_quant(x), w, ws)
        n = block_ops.gated_norm_backward(None, dn * x[0, 0], h, st, y=y, gate=gate, scale=scale)
        r = block_ops.axes_rope_backward(d * x[0, 0], None, pos, inv, pairs, q=q, norm=True, q_weight=gain)
        return (y8, *(n[k] for k in sorted(n)), r[0], r[2])

    taken = []
    plain = block_ops._scratch
    monkeypatch.setattr(block_ops, "_scratch", lambda *a: taken.append(plain(*a)) or taken[-1])
    side, s1, s2 = (torch.cuda.Stream() for _ in range(3))
    xs = [rn(8, 4096).bfloat16() for _ in range(3)]
    want = [work(x) for x in xs]
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        work(xs[2])
    torch.cuda.synchronize()
    graphs, outs, held = [torch.cuda.CUDAGraph() for _ in range(2)], [], []
    for graph, x in zip(graphs, xs):
        del taken[:]
        with torch.cuda.graph(graph, stream=side):
            outs.append(work(x))
        held.append({t.data_ptr() for t in taken})
    del taken[:]
    with torch.cuda.stream(side):
        work(xs[2])
    held.append({t.data_ptr() for t in taken})
    assert all(held) and not held[0] & held[1] and not held[2] & (held[0] | held[1])
    for _ in range(5):
        for o in (*outs[0], *outs[1]):
            o.zero_()
        torch.cuda.synchronize()
        for _ in range(4):
            with torch.cuda.stream(s1):
                graphs[0].replay()
            with torch.cuda.stream(s2):
                graphs[1].replay()
            with torch.cuda.stream(side):
                eager = work(xs[2])
        torch.cuda.synchronize()
        for got, ref in zip((*outs, eager), want):
            assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_norm_of_nothing_has_the_statistics_of_absent_norms(gpu):
    x = torch.randn(2, 5, 64, device=gpu).bfloat16()
    torch.full((2, 5, 4), 7.0, device=gpu)
    want = torch.tensor([0.0, 1.0, 0.0, 1.0], device=gpu).expand(2, 5, 4)
    assert torch.equal(block_ops.gated_norm(x, norm=None, return_stats=True)[2], want)
    torch.full((2, 5, 4), 7.0, device=gpu)
    assert torch.equal(torch.ops.xdit_amd.gated_norm(x, *(None,) * 7, "none", 1e-6, "none", 1e-6, 1.0)[2], want)
    assert torch.equal(block_ops.gated_norm(x, y=x, norm=None, return_stats=True)[2], want)


def test_gradients_that_start_anywhere(gpu):
    """The gradient of a result that went into a concatenation is a part of that one's, at any element: the same bits as one by itself."""
    g = torch.Generator(device=gpu).manual_seed(9)
    rn = lambda *s: torch.randn(*s, generator=g, device=gpu)  # noqa: E731
    x = rn(1, 6, 128).bfloat16().requires_grad_()
    q = rn(1, 2, 6, 128).bfloat16().requires_grad_()
    pad, r = torch.zeros(3, device=gpu, dtype=torch.bfloat16), rn(6 * 128 * 2).bfloat16()
    freq, pairs = block.rope_frequencies((44, 42, 42), device=gpu)
    linear = block.Fp8Linear((rn(256, 128) / 11).bfloat16(), backward=True)
    pos = torch.arange(18, device=gpu).view(6, 3)
    for t, f in ((x, lambda: block.gated_norm(x, norm="rms")[1]), (q, lambda: block.axes_rope(q, None, pos, freq, pairs, norm=True)[0]), (x, lambda: linear(x))):
        y = f().flatten()
        (want,) = torch.autograd.grad(y, t, r[:y.numel()])
        cat = torch.cat([pad, f().flatten()])
        (got,) = torch.autograd.grad(cat, t, torch.cat([pad, r[:y.numel()]]))
        assert torch.equal(got, want)


def test_projection_of_strided_and_unaligned_activations(gpu):
    g = torch.Generator(device=gpu).manual_seed(10)
    linear = block.Fp8Linear(torch.randn(200, 128, generator=g, device=gpu) / 11)
    x = torch.randn(2, 128, 7, generator=g, device=gpu).bfloat16().transpose(1, 2)
    flat = torch.empty(x.numel() + 1, dtype=x.dtype, device=gpu)
    flat[1:] = x.contiguous().flatten()
    want = linear(x.contiguous())
    assert torch.equal(linear(x), want) and torch.equal(linear(flat[1:].view(2, 7, 128)), want) and torch.equal(linear(x.clone().requires_grad_()), want)


def test_projection_of_a_weight_in_a_flat_buffer(gpu):
    g = torch.Generator(device=gpu).manual_seed(12)
    flat = (torch.randn(96 * 128 + 8, generator=g, device=gpu) / 11).bfloat16()
    x = torch.randn(5, 128, generator=g, device=gpu).bfloat16()
    for at in (1, 4, 8):
        w = flat[at:at + 96 * 128].view(96, 128)
        assert torch.equal(block.Fp8Linear(w)(x), block.Fp8Linear(w.clone())(x))
        assert torch.equal(block.Fp8Linear(w.t().contiguous().t())(x), block.Fp8Linear(w.clone())(x))
