"""Host-side logic of a training step on the CPU: no kernels run, device calls are stubbed."""
import contextlib

import pytest
import torch
from torch.autograd import forward_ad

from xdit_amd import attention_backend as AB
from xdit_amd import block_ops, custom_ops, grad_ops, ops, ring, usp


@pytest.fixture
def calls(monkeypatch):
    """`grad_ops` on CPU tensors -> a list of (entry point, workspace address, workspace bytes) of the C calls."""
    class Calls(list):
        capturing = False
        need = 5000

    seen = Calls()

    class Lib:
        def __getattr__(self, name):
            if name.endswith("workspace_bytes"):
                return lambda a: seen.need

            def call(a):
                seen.append((name, getattr(a._obj, "workspace", None), getattr(a._obj, "workspace_bytes", 0)))
                return 0
            return call

    monkeypatch.setattr(ops, "_check4", lambda *a: None)
    for module in (grad_ops, block_ops):
        monkeypatch.setattr(module, "_stream", lambda device: 7)
        monkeypatch.setattr(module, "_on_device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(block_ops, "_capturing", lambda device, stream: seen.capturing)
    monkeypatch.setattr(block_ops, "_SCRATCH", {})
    monkeypatch.setattr(grad_ops._lib, "lib", Lib)
    monkeypatch.setattr(ops._TLS, "block_plans", {}, raising=False)
    return seen


def backward(S=8, **kw):
    q = torch.zeros(1, 2, S, 64)
    return grad_ops.attn_bwd(q, q, q, q, q, torch.zeros(1, 2, S), **kw)


def test_captured_calls_have_scratch_of_their_own(calls):
    backward()
    backward()
    (buf,) = block_ops._SCRATCH.values()
    assert calls[0][1] == calls[1][1] == buf.data_ptr() and calls[0][2] == 8192   # sizes go by powers of two
    calls.capturing = True
    backward()
    assert calls[2][1] != buf.data_ptr() and list(block_ops._SCRATCH.values())[0] is buf


def test_scratch_of_growing_calls(calls):
    """What outgrown buffers leave allocated stays below the last one's size."""
    sizes = []
    for n in range(1, 200):
        calls.need = 1000 * n
        backward(S=8 * n)
        sizes.append(calls[-1][2])
        assert sizes[-1] >= calls.need
    assert sum(set(sizes)) < 2 * max(sizes)


def test_norms_count_their_workgroups(calls, monkeypatch):
    """One counter a stream, never one of a captured call's; the norm and the clipping of a list differ in what they are given."""
    class OnGpu(torch.Tensor):
        is_cuda = True

    monkeypatch.setattr(grad_ops, "_capturing", lambda device, stream: calls.capturing)
    monkeypatch.setattr(grad_ops, "_COUNTERS", {})
    ts = [torch.zeros(6).as_subclass(OnGpu)]
    given = []
    run = grad_ops._launch
    monkeypatch.setattr(grad_ops, "_launch", lambda entry, a, *r, **k: (run(entry, a, *r, **k), given.append(getattr(a, "counter", None))))
    grad_ops.grad_norm(ts)
    grad_ops.grad_norm(ts, 1)
    (c,) = grad_ops._COUNTERS.values()
    assert given == [c.data_ptr()] * 2 and int(c) == 0
    calls.capturing = True
    grad_ops.grad_norm(ts)
    grad_ops.clip_grads(ts, 1.0)
    assert given[2:] == [None, None] and len(grad_ops._COUNTERS) == 1


def test_gradients_that_are_asked_for(calls):
    q = torch.zeros(1, 2, 8, 64)
    k2 = torch.zeros(1, 2, 3, 64)
    assert [t is not None for t in backward()] == [True] * 3
    assert [t is not None for t in backward(need_q=False)] == [False, True, True]
    got = backward(k2=k2, v2=k2, need_kv=False)
    assert [t is not None for t in got] == [True] + 4 * [False]
    for kw in (dict(need_q=False, need_kv=False), dict(dq=q, need_q=False), dict(dk2=k2), dict(dk=q, need_kv=False)):
        with pytest.raises(ValueError):
            backward(**kw)
    mine = torch.ones(1, 2, 8, 64)
    assert backward(dk=mine)[1] is mine


@pytest.mark.parametrize("Sq,Sk", [(0, 5), (5, 0), (0, 0)])
def test_nothing_to_attend(calls, Sq, Sk):
    q, k = torch.zeros(1, 2, Sq, 64), torch.zeros(1, 2, Sk, 64)
    dq, dk, dv = grad_ops.attn_bwd(q, q, k, k, q, torch.zeros(1, 2, Sq))
    assert dq.shape == q.shape and dk.shape == dv.shape == k.shape and not calls
    assert not dq.any() and not dk.any() and not dv.any()


def test_tangents_are_refused():
    t = torch.zeros(1, 2, 4, 64)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(t, torch.ones_like(t))
        bshd = forward_ad.make_dual(t.transpose(1, 2), torch.ones(1, 4, 2, 64))
        for call in (lambda: AB._mi355_attn_call(t, dual, t, 0.0, False), lambda: usp.attention(dual, t, t), lambda: ring.flash_attn_forward(bshd, bshd, bshd)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_which_calls_leave_a_graph():
    t = torch.zeros(1, 2, 4, 64)
    leaf = t.clone().requires_grad_()
    assert custom_ops.attn_grad_wanted(t, leaf) and custom_ops.attn_grad_wanted(None, leaf) and not custom_ops.attn_grad_wanted(t, t, None)
    assert not custom_ops.attn_grad_wanted(t.to(torch.float8_e4m3fn))
    with torch.no_grad():
        assert not custom_ops.attn_grad_wanted(leaf)


def test_rows_that_attention_reads_in_place():
    t = torch.zeros(2, 3, 10, 64, dtype=torch.bfloat16)
    for ok in (t, t.transpose(1, 2).contiguous().transpose(1, 2), t[..., :32], t[:, :, 2:]):
        assert custom_ops._attn_rows(ok) is ok
    for bad in (t.sum().expand(2, 3, 10, 64), t[:, :, :1].expand(2, 3, 10, 64), t[..., 1:33], t.transpose(2, 3), torch.zeros(4000, dtype=torch.bfloat16)[1:3841].view(2, 3, 10, 64)):
        copy = custom_ops._attn_rows(bad)
        assert copy is not bad and copy.is_contiguous() and copy.data_ptr() % 16 == 0 and torch.equal(copy, bad)


def test_lists_of_gradients(monkeypatch):
    """What a list is checked for, and that a tensor that moved is seen."""
    class OnGpu(torch.Tensor):
        is_cuda = True

    def gpu(*shape, dtype=torch.float32):
        return torch.zeros(*shape, dtype=dtype).as_subclass(OnGpu)

    a, b = gpu(6), gpu(4, 5)
    g = grad_ops.GradList([a, b])
    first = grad_ops._listed(g)
    assert first is grad_ops._listed(g) and first.sizes == [6, 20] and list(first.ptr) == [a.data_ptr(), b.data_ptr()]
    b.data = torch.zeros(30)
    second = grad_ops._listed(g)
    assert second is not first and second.sizes == [6, 30] and second.ptr[1] == b.data_ptr()
    whole = b.data
    b.data = whole[:20]   # at the same address
    third = grad_ops._listed(g)
    assert third is not second and third.sizes == [6, 20] and list(third.numel) == [6, 20]
    b.data = whole[:20].bfloat16()
    assert list(grad_ops._listed(g).dtype) == [2, 0]
    b.data = whole.view(5, 6).t()
    with pytest.raises(ValueError, match="contiguous"):
        grad_ops._listed(g)
    for kind, code in ((2, 2), (1, 1), (float("inf"), 0), (2.0, 2)):
        assert grad_ops._kind(kind) == code
    for kind in (0, 3, None, "two", float("nan"), -1):
        with pytest.raises(ValueError, match="norm_type"):
            grad_ops._kind(kind)
