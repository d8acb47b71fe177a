"""Host-side logic of the operators around the attention call on the CPU: no kernels run, device calls are stubbed."""
import contextlib

import pytest
import torch
from torch.autograd import forward_ad

from xdit_amd import block, block_ops, ops


@pytest.fixture
def calls(monkeypatch):
    """`block_ops` on CPU tensors -> a list of the workspace that each C call was given; `calls.capturing` is what the stream says."""
    class Calls(list):
        capturing = False

    seen = Calls()

    class Lib:
        def __getattr__(self, name):
            if name.endswith("workspace_bytes"):
                return lambda a: 4096

            def call(a):
                seen.append(getattr(a._obj, "workspace", None))
                return 0
            return call

    monkeypatch.setattr(block_ops, "_check", lambda *a: None)
    monkeypatch.setattr(block_ops, "_stream", lambda device: 7)
    monkeypatch.setattr(block_ops, "_on_device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(block_ops, "_capturing", lambda device, stream: seen.capturing, raising=False)
    monkeypatch.setattr(block_ops._lib, "lib", Lib)
    monkeypatch.setattr(block_ops, "_SCRATCH", {})
    for store in ("plans", "block_plans"):
        monkeypatch.setattr(ops._TLS, store, {}, raising=False)
    return seen


def norm_backward():
    h = torch.zeros(1, 4, 64)
    block_ops.gated_norm_backward(h, h, h, torch.zeros(1, 4, 4), scale=torch.zeros(1, 64))


def rope_backward():
    d = torch.zeros(1, 2, 4, 64)
    block_ops.axes_rope_backward(d, None, torch.zeros(4, 1), torch.zeros(32), (32,), q=d, norm=True, q_weight=torch.zeros(64))


def product():
    x = torch.zeros(4, 256).to(torch.float8_e4m3fn)
    block_ops.fp8_block_matmul(x, torch.zeros(4, 2), x, torch.zeros(1, 2))


@pytest.mark.parametrize("call", [norm_backward, rope_backward, product])
def test_a_captured_call_has_scratch_of_its_own(calls, call):
    """A graph keeps the scratch's address and may run beside other graphs and eager calls: it holds neither what the eager
    calls of its stream share nor, through that, what another graph holds."""
    calls.capturing = True
    call()
    assert calls[-1] and block_ops._SCRATCH == {}
    calls.capturing = False
    call()
    call()
    (buf,) = block_ops._SCRATCH.values()
    assert calls[-1] == calls[-2] == buf.data_ptr()
    calls.capturing = True
    call()
    assert calls[-1] != buf.data_ptr() and list(block_ops._SCRATCH.values())[0] is buf


@pytest.mark.parametrize("norm,C", [(None, 64), ("layer", 0)])
def test_statistics_of_a_call_without_a_launch(calls, norm, C):
    """Mean 0 and reciprocal deviation 1 for norms that are absent, also where nothing is left to compute."""
    poison = [torch.full((3, 5, 4), 7.0) for _ in range(50)]
    del poison
    x = torch.zeros(3, 5, C)
    h, n, stats = block_ops.gated_norm(x, norm=norm, return_stats=True)
    assert calls == [] and h is x and (n is None) == (norm is None)
    assert torch.equal(stats, torch.tensor([0.0, 1.0, 0.0, 1.0]).expand(3, 5, 4))


def test_tangents_are_refused():
    """A forward-mode dual tensor wants no reverse gradient, so the kernels would read its values and drop its tangent."""
    x, w, q = torch.randn(1, 4, 64), torch.ones(64), torch.randn(1, 2, 4, 64)
    freq, pairs = block.rope_frequencies((64,))
    linear = block.Fp8Linear.__new__(block.Fp8Linear)
    torch.nn.Module.__init__(linear)
    pos = torch.zeros(4, 1)
    with forward_ad.dual_level():
        d = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: block.gated_norm(d(x)), lambda: block.gated_norm(x, weight=d(w)), lambda: block.axes_rope(d(q), None, pos, freq, pairs),
                     lambda: block.axes_rope(q, q, pos, freq, pairs, norm=True, k_weight=d(w)), lambda: linear(d(x))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with pytest.raises(RuntimeError, match="no CPU path"):   # no tangent: as ever
            block.gated_norm(x)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: block.gated_norm(t)[1], (x,), (x,))


def test_a_gradient_that_starts_anywhere_is_copied():
    from xdit_amd import custom_ops
    flat = torch.arange(3 * 64 + 8, dtype=torch.bfloat16)
    for at in range(8):
        t = flat[at:at + 3 * 64].view(1, 3, 64)
        r = custom_ops._rows16(t)
        assert r.data_ptr() % 16 == 0 and r.is_contiguous() and torch.equal(r, t)
        assert (r is t) == (t.data_ptr() % 16 == 0)
    assert custom_ops._rows16(torch.ones(()).expand(1, 3, 64)).is_contiguous() and custom_ops._rows16(None) is None


def test_projection_takes_any_rows_without_gradients_too(calls):
    """What a call with gradients takes (the registered op copies rows that are not dense and aligned) one without them takes as well."""
    linear = block.Fp8Linear(torch.zeros(32, 64))
    seen = []
    plain, block_ops.fp8_block_quant = block_ops.fp8_block_quant, lambda x, *a: seen.append(x) or plain(x, *a)
    try:
        for x in (torch.zeros(2, 64, 6).transpose(1, 2), torch.zeros(2 * 64 + 1)[1:].view(2, 64), torch.zeros(4, 66)[:, :64], torch.zeros(4, 64)):
            assert linear(x).shape == (*x.shape[:-1], 32)
            assert seen[-1].stride(-1) == 1 and seen[-1].stride(-2) % 4 == 0 and seen[-1].data_ptr() % 16 == 0
        assert seen[-1] is x
    finally:
        block_ops.fp8_block_quant = plain


def test_attention_keeps_its_plans_beside_many_block_calls(calls, monkeypatch):
    """Blocks of many sequence lengths do not use up the store of attention's argument structs."""
    monkeypatch.setattr(ops, "_PLANS_MAX", 8)
    monkeypatch.setattr(block_ops, "_PLANS_MAX", 8)
    ops._TLS.plans["attention"] = "kept"
    for S in range(1, 30):
        block_ops.gated_norm(torch.zeros(1, S, 64))
    assert ops._TLS.plans["attention"] == "kept" and 0 < len(ops._TLS.block_plans) <= 8


def test_numbers_are_taken_by_value(calls, monkeypatch):
    """Scalars given as tensors that change in place: each call is made with what they hold then."""
    seen = []

    class Lib:
        def __getattr__(self, name):
            return (lambda a: 4096) if name.endswith("workspace_bytes") else lambda a: seen.append((round(getattr(a._obj, "eps", 0), 3), round(getattr(a._obj, "residual_scale", 0), 3))) or 0

    monkeypatch.setattr(block_ops._lib, "lib", Lib)
    x, q, pos, freq = torch.zeros(1, 4, 64), torch.zeros(1, 2, 4, 64), torch.zeros(4, 1), torch.zeros(32)
    eps, scale = torch.tensor(0.25), torch.tensor(0.5)
    for call, want in ((lambda: block_ops.gated_norm(x, y=x, eps=eps, residual_scale=scale), (1, 1)), (lambda: block_ops.gated_norm_backward(x, x, x, torch.zeros(1, 4, 4), y=x, residual_scale=scale), (0, 1)),
                       (lambda: block_ops.axes_rope(q, None, pos, freq, (32,), norm=True, eps=eps), (1, 0)), (lambda: block_ops.axes_rope_backward(q, None, pos, freq, (32,), q=q, norm=True, eps=eps), (1, 0))):
        for _ in range(2):
            call()
            eps += 1
            scale += 2
            call()
            assert seen[-1] == (want[0] * round(float(eps), 3), want[1] * round(float(scale), 3)) and (seen[-2] != seen[-1])


def test_gradients_to_positions_and_frequencies_are_refused():
    q, pos = torch.zeros(1, 2, 4, 64), torch.zeros(4, 1)
    freq, pairs = block.rope_frequencies((64,))
    for p, f in ((pos.clone().requires_grad_(), freq), (pos, freq.clone().requires_grad_())):
        for x in (q, q.clone().requires_grad_()):
            with pytest.raises(ValueError, match="no gradient"):
                block.axes_rope(x, None, p, f, pairs)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):   # nothing wants it: as ever
            block.axes_rope(q, None, p, f, pairs)


def test_tangents_of_positions_and_frequencies_are_refused():
    q, pos = torch.zeros(1, 2, 4, 64), torch.zeros(4, 1)
    freq, pairs = block.rope_frequencies((64,))
    with forward_ad.dual_level():
        for p, f in ((forward_ad.make_dual(pos, torch.ones_like(pos)), freq), (pos, forward_ad.make_dual(freq, torch.ones_like(freq)))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                block.axes_rope(q, None, p, f, pairs)


def test_projection_of_a_weight_that_starts_anywhere(calls):
    """A weight may be a part of a flat buffer: a contiguous one off a 16-byte boundary is copied, as one that is not dense is."""
    seen = []
    plain, block_ops.fp8_block_quant = block_ops.fp8_block_quant, lambda x, *a: seen.append(x) or plain(x, *a)
    try:
        flat = torch.arange(32 * 64 + 8, dtype=torch.float32)
        for w in (flat[:32 * 64].view(32, 64), flat[1:1 + 32 * 64].view(32, 64), flat[:32 * 64].view(64, 32).t(), torch.zeros(32, 66)[:, 1:65]):
            block.Fp8Linear(w)
            assert seen[-1].data_ptr() % 16 == 0 and seen[-1].stride(-1) == 1 and torch.equal(seen[-1], w)
    finally:
        block_ops.fp8_block_quant = plain


def test_projection_keeps_its_own_bias(calls):
    """Weight and bias are frozen as they were given, an fp32 bias as well as one that is converted; one that is not dense is laid out."""
    for b in (torch.ones(32), torch.ones(32, dtype=torch.bfloat16), torch.ones(64)[::2]):
        linear = block.Fp8Linear(torch.zeros(32, 64), b)
        b += 1
        assert torch.equal(linear.bias, torch.ones(32)) and linear.bias.is_contiguous()
