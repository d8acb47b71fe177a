"""A training step of a block on the operators together: forward, attention's backward pass among the others, norm and clipping of the gradients.

Bars.  A gradient passes the block's fp8 values, off by 1/16/sqrt(3) = 0.036 in the root mean square, in four products forward and four backward, and the softmax
between them: sqrt(8 * 0.036^2 + 0.05^2) = 0.11 relative to float32, held to 0.2.  A norm that is recomputed from bf16 gradients after clipping has their
roundings, each off by at most 2^-8: held to 2^-8."""
import importlib.util
import os
import threading

import pytest
import torch

from oracle import grad_oracle as O
from xdit_amd import grad_ops, ops, usp

spec = importlib.util.spec_from_file_location("dit_block", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "dit_block.py"))
dit = importlib.util.module_from_spec(spec)
spec.loader.exec_module(dit)
pytestmark = pytest.mark.gpu


def setup(heads, head_dim, mlp, grid, batch=1):
    m = dit.DiTBlock(heads, head_dim, mlp, train=True)
    x, modulation, positions = dit.inputs(grid, heads, head_dim, batch)
    r = torch.randn(x.shape, generator=torch.Generator(device=x.device).manual_seed(3), device=x.device).to(x.dtype)
    return m, x, modulation.requires_grad_(), positions, r


@pytest.mark.parametrize("heads,head_dim,mlp,grid,batch", [(4, 64, 512, (1, 12, 11), 2), (2, 128, 1024, (3, 8, 10), 1), (4, 72, 640, (1, 9, 7), 1)])
def test_gradients_of_a_block(gpu, heads, head_dim, mlp, grid, batch):
    m, x, modulation, positions, _ = setup(heads, head_dim, mlp, grid, batch)
    far = dit.check_gradients(m, x, modulation.detach(), positions)
    assert set(far) == {"x", "modulation", "q_gain", "k_gain"} and max(far.values()) <= 0.2, far


def test_training_step(gpu):
    m, x, modulation, positions, r = setup(4, 64, 512, (1, 12, 11), 2)
    raw = torch.autograd.grad(m(x, modulation, positions), [modulation, m.q_gain, m.k_gain], r)
    want = O.grad_norm(raw)
    grads, norm = dit.training_step(m, x, modulation, positions, r, max_norm=0.5)
    assert abs(float(norm) - want) <= 2.0 ** -22 * want and want > 0.5
    assert abs(O.grad_norm(grads) - 0.5) <= 2.0 ** -8 * 0.5
    again, _ = dit.training_step(m, x, modulation, positions, r, max_norm=0.5)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))   # the same step gives the same bits
    with torch.no_grad():
        for p, g in zip((modulation, m.q_gain, m.k_gain), grads):
            p -= 0.01 * g
    _, after = dit.training_step(m, x, modulation, positions, r, max_norm=1e9)
    assert torch.isfinite(after) and not torch.equal(after, norm)


@pytest.mark.parametrize("own_streams", [True, False])
def test_two_threads_at_once(gpu, own_streams):
    """Steps of two threads, of other sizes, on streams of their own or on one: the results of one after the other."""
    def step(seed):
        g = torch.Generator(device=gpu).manual_seed(seed)
        q, k, v, dout = (torch.randn(1, 2 + seed, 500 + 100 * seed, 64, generator=g, device=gpu).half() for _ in range(4))
        leaves = [t.requires_grad_() for t in (q, k, v)]
        grads = list(torch.autograd.grad(usp.attention(*leaves), leaves, dout))
        norm = grad_ops.clip_grads(grads, 0.5)
        return [*grads, norm]

    want = [step(s) for s in (0, 1)]
    torch.cuda.synchronize()
    got, failed = [None, None], []

    def work(seed):
        try:
            with torch.cuda.stream(torch.cuda.Stream() if own_streams else torch.cuda.default_stream()):
                for _ in range(20):
                    got[seed] = step(seed)
                torch.cuda.current_stream().synchronize()
        except BaseException as e:
            failed.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for s in (0, 1) for a, b in zip(got[s], want[s]))


def test_attention_forward_and_backward_in_one_graph(gpu):
    """A captured step of the three calls, replayed on new inputs beside eager steps."""
    g = torch.Generator(device=gpu).manual_seed(0)
    q, k, v, dout = (torch.randn(1, 3, n, 64, generator=g, device=gpu).bfloat16() for n in (300, 200, 200, 300))
    out = [torch.empty(t.shape, dtype=torch.float32, device=gpu) for t in (q, k, v)]

    def step(dst):
        o, lse = ops.attn_fwd(q, k, v)
        return grad_ops.clip_grads(grad_ops.attn_bwd(dout, q, k, v, o, lse), 0.25, out=dst)

    graph = torch.cuda.CUDAGraph()
    step(out)
    with torch.cuda.graph(graph):
        norm = step(out)
    for i in range(4):
        for t in (q, k, v, dout):
            t.copy_(torch.randn(t.shape, generator=g, device=gpu))
        eager = [torch.empty_like(t) for t in out]
        want = step(eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(out, eager))
        assert abs(O.grad_norm(out) - 0.25) <= 2.0 ** -20
