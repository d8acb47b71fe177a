"""Calls without a backward pass on the GPU: the bits that they have on detached tensors, and an error instead of a gradient that is left out."""
import pytest
import torch

from xdit_amd import attention_backend as AB
from xdit_amd import prologue, usp

pytestmark = pytest.mark.gpu
FP8 = AB.AttentionBackendType.MI355_FP8


def rand(gpu, seed, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator(device=gpu).manual_seed(seed), device=gpu).to(dtype)


def same_and_refused(call, tensors):
    plain = call(*tensors)
    plain = plain if isinstance(plain, tuple) else (plain,)
    for i in range(len(tensors)):
        ts = [t.clone().requires_grad_(j == i) for j, t in enumerate(tensors)]
        got = call(*ts)
        got = got if isinstance(got, tuple) else (got,)
        assert all(torch.equal(a, b) for a, b in zip(got, plain))
        with pytest.raises(RuntimeError, match="no gradient|no autograd"):
            torch.autograd.grad(sum(t.float().sum() for t in got), ts[i])


@pytest.mark.parametrize("chunks", [1, 2])
@pytest.mark.parametrize("strategy", [None, "rear", "front"])
def test_fp8_attention(gpu, chunks, strategy):
    ts = [rand(gpu, i, 1, 2, 128, 128) for i in range(3)]
    if strategy is None:
        same_and_refused(lambda q, k, v: usp.USP(q, k, v, backend=FP8, ring_chunks=chunks), ts)
    else:
        same_and_refused(lambda q, k, v, a, b, c: usp.USP(q, k, v, joint_query=a, joint_key=b, joint_value=c, joint_strategy=strategy, backend=FP8, ring_chunks=chunks),
                         ts + [rand(gpu, 3 + i, 1, 2, 32, 128) for i in range(3)])


def test_prologue(gpu):
    x, w = rand(gpu, 0, 2, 50, 3, 64), rand(gpu, 1, 64)
    c, s = rand(gpu, 2, 50, 64, dtype=torch.float32), rand(gpu, 3, 50, 64, dtype=torch.float32)
    same_and_refused(lambda x, w, c, s: prologue.norm_rope(x, w, freqs_cis=(c, s)), [x, w, c, s])
    same_and_refused(lambda x, c, s: prologue.apply_rotary_emb(x, (c, s), sequence_dim=1), [x, c, s])
    same_and_refused(lambda x, w, c, s: torch.ops.xdit_amd.norm_rope(x.transpose(1, 2), w, c, s, 1e-6, "head", "interleaved", 0, 50), [x, w, c, s])
    m = prologue.RMSNorm(64, device=gpu, dtype=torch.bfloat16)
    with torch.no_grad():
        plain = m(x)
    assert torch.equal(m(x), plain)
    with pytest.raises(RuntimeError, match="no gradient"):
        m(x).sum().backward()
    hidden = [rand(gpu, 10 + i, 1, n, 128) for i, n in enumerate((40, 40, 40, 8, 8, 8))]
    gains = [rand(gpu, 20 + i, 64) for i in range(4)]
    tables = [t[:48] for t in (c, s)]
    same_and_refused(lambda *t: prologue.flux_joint_qkv(*t[:6], 2, *t[6:10], t[10:]), hidden + gains + tables)


def test_a_training_step_behind_the_prologue(gpu):
    """The gradient of attention reaches the prologue and stops there with an error."""
    x, w = rand(gpu, 0, 1, 64, 2, 64).requires_grad_(), rand(gpu, 1, 64)
    q = prologue.norm_rope(x, w)
    o = usp.attention(q, q, q)
    with pytest.raises(RuntimeError, match="no gradient"):
        o.sum().backward()
    assert x.grad is None


def traced_calls(gpu):
    x, w = rand(gpu, 0, 1, 64, 2, 64), rand(gpu, 1, 64)
    c, s = rand(gpu, 2, 64, 64, dtype=torch.float32), rand(gpu, 3, 64, 64, dtype=torch.float32)
    m = prologue.RMSNorm(64, device=gpu, dtype=torch.bfloat16)
    return x, {
        "norm_rope": lambda x: prologue.norm_rope(2 * x, w, freqs_cis=(c, s)) + 1,
        "apply_rotary_emb": lambda x: prologue.apply_rotary_emb(2 * x, (c, s), sequence_dim=1) + 1,
        "apply_rotary_emb_wan": lambda x: prologue.apply_rotary_emb_wan(2 * x, c[None, :, None], s[None, :, None]) + 1,
        "RMSNorm": lambda x: m(2 * x) + 1,
        "flux_joint_qkv": lambda x: prologue.flux_joint_qkv(*[2 * x.flatten(2)] * 6, 2, w, w, w, w, (torch.cat((c, c)), torch.cat((s, s))))[0] + 1,
        "ring": lambda x: usp.ring_attn(lambda q, k, v, **kw: (2 * q, torch.zeros(q.shape[:3], device=q.device)), x, x, x, ring_chunks=2) + 1,
    }


@pytest.mark.parametrize("name", ["norm_rope", "apply_rotary_emb", "apply_rotary_emb_wan", "RMSNorm", "flux_joint_qkv", "ring"])
def test_traced_calls(gpu, name):
    x, calls = traced_calls(gpu)
    torch._dynamo.reset()
    call = torch.compile(calls[name], backend="aot_eager")
    with torch.no_grad():
        plain = calls[name](x)
        assert torch.equal(call(x), plain)
    leaf = x.clone().requires_grad_()
    got = call(leaf)
    assert torch.equal(got, plain)
    with pytest.raises(RuntimeError, match="no gradient"):
        got.float().sum().backward()
