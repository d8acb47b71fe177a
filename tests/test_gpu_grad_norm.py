"""Norm and clipping of lists of gradients against float64.

Bars.  A norm is summed in 64 bits and rounded to fp32: off by 2^-24, and 2^-50 of the sums' own; held to 2^-23.  A clipped gradient is g times a
factor off by three roundings of fp32 (the norm's, the sum's with 1e-6, the quotient's), and rounded twice more (the product, the result's type): half a step
of its type plus 5 * 2^-24."""
import math

import pytest
import torch

from oracle import grad_oracle as O
from xdit_amd import grad_ops

pytestmark = pytest.mark.gpu
F = (torch.bfloat16, torch.float16, torch.float32)
EPS32 = 2.0 ** -24


def grads(gpu, sizes, dtypes=F, seed=0, offset=0):
    """Gradients of these sizes, each `offset` elements behind a 16-byte boundary."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        dt = dtypes[i % len(dtypes)]
        buf = torch.full((n + 32,), math.nan, dtype=dt, device=gpu)
        t = buf[16 + offset:16 + offset + n]
        t.copy_(torch.randn(n, generator=g, device=gpu) * 2.0 ** ((i % 9) - 4))
        out.append(t)
    return out


def norm_close(got, want):
    assert got.dtype == torch.float32 and got.shape == ()
    assert abs(float(got) - want) <= 2.0 ** -23 * want, (float(got), want)


def clip_close(got, src, norm, max_norm):
    for g, w in zip(got, O.clip(src, norm, max_norm)):
        far = (torch.finfo(g.dtype).eps / 2 + 5 * EPS32) * w.abs() + (2.0 ** -25 if g.dtype == torch.float16 else 2.0 ** -140)
        assert bool(((g.double() - w).abs() <= far).all())


LISTS = [[1], [7, 1, 8, 9], [0, 5, 0, 4096], [2048, 2047, 2049, 8192, 24576, 24577], [72, 72, 6912] * 28, [3, 100003, 17, 640, 1 << 20], [1] * 500, [300000]]


@pytest.mark.parametrize("sizes", LISTS)
@pytest.mark.parametrize("offset", [0, 1, 5])
@pytest.mark.parametrize("kind", [2, 1, math.inf])
def test_norm(gpu, sizes, offset, kind):
    gs = grads(gpu, sizes, offset=offset)
    norm_close(grad_ops.grad_norm(gs, kind), O.grad_norm(gs, kind))
    assert torch.equal(grad_ops.grad_norm(gs, kind), grad_ops.grad_norm(grad_ops.GradList(gs), kind))


@pytest.mark.parametrize("dtype", F)
def test_norm_of_many_elements(gpu, dtype):
    g = torch.Generator(device=gpu).manual_seed(1)
    t = torch.randn(50_000_003, generator=g, device=gpu).to(dtype)
    norm_close(grad_ops.grad_norm([t[1:], t[:1]]), O.grad_norm([t]))


def test_norm_beyond_the_squares_of_fp32(gpu):
    for size in (1e30, 1e-30):
        t = [torch.full((1000,), size, device=gpu), torch.full((9,), size, device=gpu, dtype=torch.bfloat16)]
        norm_close(grad_ops.grad_norm(t), O.grad_norm(t))
    assert float(grad_ops.grad_norm([torch.full((100,), 3e38, device=gpu)])) == math.inf


@pytest.mark.parametrize("kind", [2, 1, math.inf])
def test_norm_of_what_is_not_finite(gpu, kind):
    t = torch.ones(5000, device=gpu)
    t[4321] = math.inf
    assert float(grad_ops.grad_norm([t], kind)) == math.inf
    t[17] = math.nan
    assert math.isnan(float(grad_ops.grad_norm([t, torch.ones(3, device=gpu)], kind)))
    assert float(grad_ops.grad_norm([torch.empty(0, device=gpu)], kind)) == 0


@pytest.mark.parametrize("sizes", LISTS)
@pytest.mark.parametrize("offset", [0, 3])
@pytest.mark.parametrize("max_norm", [0.0, 0.25, 1e9])
def test_clip_in_place(gpu, sizes, offset, max_norm):
    gs = grads(gpu, sizes, offset=offset)
    src = [t.clone() for t in gs]
    n = grad_ops.clip_grads(gs, max_norm)
    want = O.grad_norm(src)
    norm_close(n, want)
    clip_close(gs, src, want, max_norm)
    if max_norm > want:
        assert all(torch.equal(a, b) for a, b in zip(gs, src))
    for t in gs:   # the elements around the tensor
        assert int(t._base.isnan().sum()) == 32


@pytest.mark.parametrize("to", F)
@pytest.mark.parametrize("offsets", [(0, 0), (1, 1), (0, 2), (3, 0)])
def test_clip_into_other_tensors(gpu, to, offsets):
    sizes = [72, 1, 0, 20000, 6911, 100003]
    src = grads(gpu, sizes, offset=offsets[0])
    keep = [t.clone() for t in src]
    dst = grads(gpu, sizes, dtypes=(to,), offset=offsets[1])
    n = grad_ops.clip_grads(grad_ops.GradList(src), 0.5, out=grad_ops.GradList(dst), norm_type=1)
    norm_close(n, O.grad_norm(src, 1))
    clip_close(dst, src, O.grad_norm(src, 1), 0.5)
    assert all(torch.equal(a, b) for a, b in zip(src, keep))
    for t in dst:
        assert int(t._base.isnan().sum()) == 32
    n = grad_ops.clip_grads(src, 1e9, out=dst)   # nothing to clip: copied all the same
    clip_close(dst, src, float(n), 1e9)


def test_clip_by_a_given_norm(gpu):
    gs = grads(gpu, [1000, 24])
    src = [t.clone() for t in gs]
    norm = torch.tensor([40.0], device=gpu)
    assert grad_ops.clip_grads(gs, 2.0, norm=norm) is norm
    clip_close(gs, src, 40.0, 2.0)


def test_clip_by_what_is_not_finite(gpu):
    gs = [torch.ones(100, device=gpu), torch.ones(9, device=gpu, dtype=torch.bfloat16)]
    grad_ops.clip_grads(gs, 1.0, norm=torch.tensor(math.inf, device=gpu))
    assert not any(t.any() for t in gs)
    grad_ops.clip_grads(gs, 1.0, norm=torch.tensor(math.nan, device=gpu))
    assert all(t.isnan().all() for t in gs)


def test_matches_torch_on_a_model(gpu):
    m = torch.nn.Sequential(torch.nn.Linear(300, 77), torch.nn.Linear(77, 5)).to(gpu)
    m(torch.ones(4, 300, device=gpu)).square().sum().backward()
    ours = [p.grad.clone() for p in m.parameters()]
    norm = torch.nn.utils.clip_grad_norm_(m.parameters(), 0.1)
    assert abs(float(grad_ops.clip_grads(ours, 0.1)) - float(norm)) <= 1e-6 * float(norm)
    for a, p in zip(ours, m.parameters()):
        assert bool(((a - p.grad).abs() <= 8 * EPS32 * p.grad.abs() + 1e-6 * p.grad.abs()).all())


@pytest.mark.parametrize("kind", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("sizes,mixed", [([3], False), ([72] * 84, False), ([2041] * 184, False), ([2041] * 185, False), ([300000, 7], False), ([2097000], False),
                                         ([2200000], False), ([50, 60], True), ([0, 5, 0], False)])
def test_norm_in_one_launch(gpu, sizes, mixed, kind):
    """Around the border between one launch and two, call after call: the same bits as in the clipping and in a graph, which take their sums another way."""
    gs = grads(gpu, sizes)
    gs = [t.bfloat16() if mixed and i else t.float() for i, t in enumerate(gs)]
    norms = [grad_ops.grad_norm(gs, kind) for _ in range(5)]
    norm_close(norms[0], O.grad_norm(gs, kind))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = grad_ops.grad_norm(gs, kind)
    graph.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        norms += [grad_ops.grad_norm(gs, kind) for _ in range(5)]
    torch.cuda.current_stream().wait_stream(side)
    clipped = grad_ops.clip_grads([t.clone() for t in gs], 1.0, norm_type=kind)
    assert all(torch.equal(n, norms[0]) for n in (*norms, captured, clipped))


def test_a_list_whose_tensors_move(gpu):
    t = [torch.ones(100, device=gpu), torch.ones(50, device=gpu)]
    g = grad_ops.GradList(t)
    norm_close(grad_ops.grad_norm(g), math.sqrt(150))
    t[1].data = torch.full((200,), 2.0, device=gpu)
    norm_close(grad_ops.grad_norm(g), math.sqrt(900))
    assert len(g) == 2 and g[1] is t[1]


def test_streams_and_replayed_graphs(gpu):
    gs = grads(gpu, [72, 72, 6912] * 60)
    src = [t.clone() for t in gs]
    out = [torch.empty_like(t, dtype=torch.float32) for t in gs]
    want = grad_ops.grad_norm(gs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = grad_ops.grad_norm(gs)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            n = grad_ops.clip_grads(gs, 0.5, out=out)
        graphs.append((g, n))
    for k in range(4):
        for t, s in zip(gs, src):
            t.copy_(s * (k + 1))
        eager = [torch.empty_like(t) for t in out]
        ne = grad_ops.clip_grads(gs, 0.5, out=eager)
        for g, n in graphs:
            for t in out:
                t.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(n, ne) and all(torch.equal(a, b) for a, b in zip(out, eager))


def test_refusals(gpu):
    a = torch.ones(8, device=gpu)
    for bad, kind in (([], ValueError), (a, ValueError), ([a, None], ValueError), ([torch.ones(4)], RuntimeError), ([a, torch.ones(4)], RuntimeError),
                      ([a.double()], ValueError), ([torch.ones(4, 4, device=gpu).t()], ValueError), ([a[:1].expand(4)], ValueError)):
        with pytest.raises(kind):
            grad_ops.grad_norm(bad)
    with pytest.raises(ValueError, match="norm_type"):
        grad_ops.grad_norm([a], 3)
    for out in ([a, a], [torch.ones(9, device=gpu)]):
        with pytest.raises(ValueError, match="out"):
            grad_ops.clip_grads([a], 1.0, out=out)
    for m in (-1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="max_norm"):
            grad_ops.clip_grads([a], m)
    for norm in (1.0, torch.ones(2, device=gpu), torch.ones((), device=gpu, dtype=torch.float64), torch.ones(())):
        with pytest.raises(ValueError, match="norm must"):
            grad_ops.clip_grads([a], 1.0, norm=norm)
    b = torch.ones(64, device=gpu)
    for src, dst in (([a, a], None), ([b[:32], b[16:48]], None), ([b[:32], b[32:]], [b[32:], b[:32]]), ([b[:32]], [b[4:36]]),
                     ([b[:16]], [b.view(torch.bfloat16)[:16]])):
        with pytest.raises(ValueError, match="overlaps"):
            grad_ops.clip_grads(src, 1.0, out=dst)
    assert bool((b == 1).all())
