"""What is written into given tensors counts as a change in place: autograd refuses to go on with what it saved before.  On the CPU, with C calls that do nothing."""
import contextlib

import pytest
import torch

from xdit_amd import block_ops, grad_ops, ops


class OnGpu(torch.Tensor):
    is_cuda = True


@pytest.fixture
def no_kernels(monkeypatch):
    class Lib:
        def __getattr__(self, name):
            return lambda a: 8 if name.endswith("workspace_bytes") else 0

    monkeypatch.setattr(ops, "_check4", lambda *a: None)
    for module in (grad_ops, block_ops):
        monkeypatch.setattr(module, "_stream", lambda device: 7)
        monkeypatch.setattr(module, "_on_device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(block_ops, "_capturing", lambda device, stream: False)
    monkeypatch.setattr(block_ops, "_SCRATCH", {})
    monkeypatch.setattr(grad_ops._lib, "lib", Lib)
    monkeypatch.setattr(ops._TLS, "block_plans", {}, raising=False)


def gpu(*shape):
    return torch.ones(*shape).as_subclass(OnGpu)


@pytest.mark.parametrize("kind", [list, grad_ops.GradList])
def test_clipping(no_kernels, kind):
    a, b, out = gpu(6), gpu(2, 3), [gpu(6), gpu(2, 3)]
    before = a._version, out[0]._version
    grad_ops.clip_grads(kind([a, b]), 1.0, out=kind(out))
    assert a._version == before[0] and all(t._version > before[1] for t in out)
    grad_ops.clip_grads(kind([a, b]), 1.0)
    assert a._version > before[0] and b._version > before[0]


def test_a_gradient_that_a_graph_has_saved(no_kernels):
    p = torch.ones(6, requires_grad=True)
    g = (p.detach() * 2).as_subclass(OnGpu)
    loss = (p * g).sum()   # saves g
    grad_ops.clip_grads([g], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_inference_tensors_have_no_versions(no_kernels):
    with torch.inference_mode():
        t = gpu(6)
    grad_ops.clip_grads([t], 1.0)


def test_gradients_of_attention(no_kernels):
    q, lse, dq = torch.zeros(1, 2, 8, 64), torch.zeros(1, 2, 8), torch.zeros(1, 2, 8, 64)
    grad_ops.attn_bwd(q, q, q, q, q, lse, dq=dq)
    assert dq._version == 1 and q._version == 0
    empty = torch.zeros(1, 2, 0, 64)
    grad_ops.attn_bwd(q, q, empty, empty, q, lse, dq=dq)
    assert dq._version > 1
