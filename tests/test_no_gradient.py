"""Calls without a backward pass, next to those that have one: a gradient that is asked for through them is an error, never left out.  On the CPU, with kernels that write
nothing but a number."""
import os
import subprocess
import sys

import pytest
import torch

from xdit_amd import attention_backend as AB
from xdit_amd import ops, prologue, ring, usp

B, H, S, D = 1, 2, 8, 64


@pytest.fixture
def kernels(monkeypatch):
    def quant(jobs, joined=()):
        out = []
        for i, (x, _, _, _, x2) in enumerate(jobs):
            y = [x.detach().to(torch.float8_e4m3fn)] + ([] if x2 is None else [x2.detach().to(torch.float8_e4m3fn)])
            if i in joined:
                y = [torch.cat(y, 2)]
            out.append((*y, torch.ones(x.shape[:2])))
        return out

    def fwd(q, k, v, out=None, out_dtype=None, **kw):
        out = torch.empty(q.shape, dtype=out_dtype or q.dtype) if out is None else out
        return out.detach().fill_(2.0), torch.full(q.shape[:3], 3.0)

    def merge(acc_out, acc_lse, block_out, block_lse, first=False, final_out=None):
        for t in (acc_out, acc_lse, final_out):
            if t is not None:
                t.detach().fill_(2.0)

    def qk_prologue(x, out=None, **kw):
        return out.detach().fill_(2.0)

    monkeypatch.setattr(ops, "fp8_quant_batch", quant)
    monkeypatch.setattr(ops, "attn_fwd", fwd)
    monkeypatch.setattr(ops, "attn_fwd_accumulate", lambda q, k, v, acc_out, acc_lse, final_out=None, **kw: final_out is not None and final_out.detach().fill_(2.0))
    monkeypatch.setattr(ops, "lse_merge", merge)
    monkeypatch.setattr(ops, "qk_prologue", qk_prologue)
    monkeypatch.setattr(ops, "launch_prologue_batch", lambda arr, n, device: None)
    monkeypatch.setattr(ops, "prologue_batch_args", _Jobs)


class _Jobs(list):
    """Argument structs of a batch, as far as `flux_joint_qkv` looks at them."""

    def __init__(self, jobs):
        class Job:
            def __init__(self, j):
                self.y, self.weight = j["out"].data_ptr(), j["weight"].data_ptr() if j.get("weight") is not None else None
                self.cos, self.sin = (t.data_ptr() for t in j["rotary_emb"]) if "rotary_emb" in j else (None, None)
                j["out"].detach().fill_(2.0)
        super().__init__(Job(j) for j in jobs)


def bhsd(S=S):
    return torch.zeros(B, H, S, D, dtype=torch.bfloat16)


def bshd():
    return torch.zeros(B, S, H, D, dtype=torch.bfloat16)


def fp8(**kw):
    return lambda q, k, v: AB._mi355_fp8_attn_call(q, k, v, 0.0, False, **kw)


def fp8_usp(**kw):
    return lambda *t: usp.USP(*t[:3], backend=AB.AttentionBackendType.MI355_FP8, **dict(zip(("joint_query", "joint_key", "joint_value"), t[3:])), **kw)


def merged(o, l):
    m = usp.SDPAMerger()
    m.step(bhsd(), torch.zeros(B, H, S))
    m.step(o, l, final_step=True)
    return m.results()


def update(block_out, block_lse):
    out, lse = ring.update_out_and_lse(None, None, bshd(), torch.zeros(B, H, S))
    out, lse = ring.update_out_and_lse(out, lse, block_out, block_lse)
    return ring.update_out_and_lse(out, lse, bshd(), torch.zeros(B, H, S))


def flux(*t):
    try:
        return prologue.flux_joint_qkv(*t[:6], H, *t[6:10], t[10:])
    finally:
        prologue._TLS.__dict__.pop("flux_plans", None)   # plans of the structs above


def hidden(n=S):
    return torch.zeros(B, n, H * D, dtype=torch.bfloat16)


def table(n=S):
    return torch.zeros(n, D)


def gain():
    return torch.zeros(D, dtype=torch.bfloat16)


def lse():
    return torch.zeros(B, H, S)


CALLS = {
    "fp8 attention": (fp8(), [bhsd] * 3),
    "fp8 attention by name": (lambda *t: usp.attention(*t, backend=AB.AttentionBackendType.MI355_FP8), [bhsd] * 3),
    "fp8 attention, joint": (fp8_usp(joint_strategy="rear"), [bhsd] * 6),
    "fp8 ring, joint": (fp8_usp(joint_strategy="front", ring_chunks=2), [bhsd] * 6),
    "ring on another function": (lambda *t: usp.ring_attn(lambda q, k, v, **kw: (q.detach().clone(), torch.zeros(q.shape[:3])), *t, ring_chunks=2), [bhsd] * 3),
    "merger": (merged, [bhsd, lse]),
    "accumulator": (update, [bshd, lse]),
    "apply_rotary_emb": (lambda x, c, s: prologue.apply_rotary_emb(x, (c, s)), [bhsd, table, table]),
    "apply_rotary_emb_wan": (prologue.apply_rotary_emb_wan, [bshd, table, table]),
    "norm_rope": (lambda x, w, c, s: prologue.norm_rope(x, w, freqs_cis=(c, s)), [bshd, gain, table, table]),
    "norm_rope into a tensor": (lambda x, w: prologue.norm_rope(x, w, out=bhsd(20), out_row0=3), [bshd, gain]),
    "flux_joint_qkv": (flux, [hidden] * 6 + [gain] * 4 + [lambda: table(2 * S)] * 2),
}


def floats(r):
    return [t for t in (r if isinstance(r, tuple) else (r,)) if isinstance(t, torch.Tensor)]


@pytest.mark.parametrize("name", CALLS)
def test_a_gradient_is_refused_and_not_dropped(kernels, name):
    call, given = CALLS[name]
    plain = floats(call(*(make() for make in given)))
    assert not any(t.requires_grad for t in plain)
    for i in range(len(given)):
        ts = [make() for make in given]
        ts[i].requires_grad_()
        got = floats(call(*ts))
        assert len(got) == len(plain) and all(torch.equal(a, b) and a.dtype == b.dtype for a, b in zip(got, plain))
        for t in got:
            with pytest.raises(RuntimeError, match="no gradient"):
                torch.autograd.grad(t.sum(), ts[i], retain_graph=True)
        with torch.no_grad():
            assert not any(t.requires_grad for t in floats(call(*ts)))


def test_gains_of_the_norm_module(kernels):
    m = prologue.RMSNorm(D, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no gradient"):
        m(bhsd()).sum().backward()
    with torch.no_grad():
        assert not m(bhsd()).requires_grad
    m.requires_grad_(False)
    assert not m(bhsd()).requires_grad


def test_results_in_a_given_tensor(kernels):
    out = bhsd(20)
    assert prologue.norm_rope(bshd(), gain(), out=out) is out
    with torch.no_grad():
        assert prologue.norm_rope(bshd().requires_grad_(), gain(), out=out) is out
    text = prologue.norm_rope(bshd().requires_grad_(), gain(), out=out)
    both = prologue.norm_rope(bshd().requires_grad_(), gain(), out=text, out_row0=S)
    assert both.data_ptr() == out.data_ptr() and both.requires_grad and not out.requires_grad


def test_the_compiler_is_not_imported_for_it():
    code = "import sys, torch, xdit_amd.attention_backend, xdit_amd.prologue, xdit_amd.ring, xdit_amd.usp; sys.exit('torch._dynamo' in sys.modules)"
    assert subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__)))).returncode == 0
