"""The C entry points of a training step without a GPU: structs as the header declares them, refusals before anything is launched, and
sizes of workspaces."""
import ctypes
import os
import subprocess

import pytest
import torch

from xdit_amd import _lib, custom_ops, grad_ops  # noqa: F401

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BAD, UNSUP = _lib.XDIT_ERR_INVALID_ARG, _lib.XDIT_ERR_UNSUPPORTED
STRUCTS = {"xdit_attn_bwd_args": _lib.AttnBwdArgs, "xdit_grad_norm_args": _lib.GradNormArgs, "xdit_clip_grads_args": _lib.ClipGradsArgs}
P = 0x1000   # never dereferenced: a refusal comes first


def test_structs_match_the_header(tmp_path):
    fields = [(c, f[0]) for c, s in STRUCTS.items() for f in s._fields_]
    src = '#include "xdit_amd_attn.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(){'
    src += "".join('printf("%%zu\\n", sizeof(%s));' % c for c in STRUCTS)
    src += "".join('printf("%%zu\\n", offsetof(%s, %s));' % f for f in fields) + "}\n"
    (tmp_path / "s.c").write_text(src)
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")])
    got = [int(x) for x in subprocess.check_output([str(tmp_path / "s")]).split()]
    assert got == [ctypes.sizeof(s) for s in STRUCTS.values()] + [getattr(STRUCTS[c], f).offset for c, f in fields]


def bwd_args(**kw):
    a = _lib.AttnBwdArgs()
    B, H, Sq, Sk, Sk2, D = 2, 3, 100, 80, 20, 64
    values = dict(struct_size=ctypes.sizeof(a), dtype=_lib.DTYPE_BF16, B=B, H=H, D=D, Sq=Sq, Sk=Sk, Sk2=Sk2, softmax_scale=0.125, cu_count=256,
                  lse_stride=_lib.Strides(H * Sq, Sq, 1), workspace=P, workspace_bytes=1 << 40)
    for names, S in ((("q", "dout", "out", "dq"), Sq), (("k", "v", "dk", "dv"), Sk), (("k2", "v2", "dk2", "dv2"), Sk2)):
        for n in names:
            values[n], values[n + "_stride"] = P * (2 + len(values)), _lib.Strides(H * S * D, S * D, D)
    values["lse"] = P
    for k, v in {**values, **kw}.items():
        setattr(a, k, v)
    return a


def refused(fn, a, code, needle):
    assert fn(ctypes.byref(a)) == code
    assert needle in _lib.lib().xdit_attn_last_error().decode()


S = _lib.Strides


@pytest.mark.parametrize("kw,code,needle", [
    (dict(struct_size=8), BAD, "struct_size"), (dict(dtype=9), BAD, "dtype"), (dict(dtype=_lib.DTYPE_FP8_E4M3FN), UNSUP, "dtype"), (dict(B=0), BAD, "positive"),
    (dict(H=-1), BAD, "positive"), (dict(Sq=0), BAD, "Sq>0"), (dict(Sk=0), BAD, "Sk>0"), (dict(Sk2=-1), BAD, "Sk2>=0"), (dict(Sq=1 << 30), BAD, "2^29"),
    (dict(B=1 << 20, H=1 << 10), BAD, "too large"), (dict(softmax_scale=0.0), BAD, "softmax_scale"), (dict(softmax_scale=float("inf")), BAD, "softmax_scale"),
    (dict(D=60), UNSUP, "head_dim"), (dict(D=136), UNSUP, "head_dim"), (dict(cu_count=-1), BAD, "cu_count"), (dict(reserved0=1), BAD, "reserved0"),
    (dict(dq=None, dk=None, dv=None, dk2=None, dv2=None), BAD, "both NULL"), (dict(dv=None), BAD, "together"), (dict(dk2=None), BAD, "together"),
    (dict(dk=None), BAD, "together"),
] + [(dict([(n, None)]), BAD, n) for n in ("q", "k", "v", "k2", "v2", "out", "dout", "lse")]
  + [(dict([(n, P + 8)]), BAD, "aligned") for n in ("q", "k", "dout", "dq", "dv", "dk2")]
  + [(dict([(n + "_stride", S(0, 64, 60))]), BAD, n) for n in ("q", "v", "out", "dq", "dk")]
  + [(dict([(n + "_stride", S(6400, 0, 64))]), BAD, "overlap") for n in ("dq", "dk", "dv", "dk2", "dv2")]
  + [(dict(q_stride=S(0, 0, 1 << 23)), BAD, "too large"), (dict(k_stride=S(-8, 0, 64)), BAD, "negative"), (dict(lse=P + 2), BAD, "4-byte"),
     (dict(dq=P), BAD, "place of an input"), (dict(dk=P * 100, dv=P * 100), BAD, "one place"), (dict(dk2=P * 100, q=P * 100), BAD, "place of an input"),
     (dict(lse_stride=S(0, -1, 1)), BAD, "negative"), (dict(dlse=P, dlse_stride=S(0, 0, -1)), BAD, "negative"), (dict(workspace=None), BAD, "workspace"),
     (dict(workspace_bytes=16), BAD, "workspace"), (dict(workspace=P + 4), BAD, "workspace")])
def test_attention_backward_refusals(kw, code, needle):
    refused(_lib.lib().xdit_attn_bwd, bwd_args(**kw), code, needle)


def test_attention_backward_workspace():
    size = lambda **kw: _lib.lib().xdit_attn_bwd_workspace_bytes(ctypes.byref(bwd_args(**kw)))  # noqa: E731
    rows = 6 * 128 * 2 * 4                       # two fp32 of every query row, rounded up to whole tiles
    assert size(cu_count=1) == rows              # nothing to cut: no partial results
    assert size(cu_count=1, dtype=_lib.DTYPE_FP16) == rows + 256
    assert size(cu_count=4096, Sq=4096) > size(cu_count=1, Sq=4096)
    only = dict(dk=None, dv=None, dk2=None, dv2=None)
    assert size(cu_count=64, Sq=100, Sk=9000, **only) > size(cu_count=1, Sq=100, Sk=9000, **only)
    assert size(D=60) == UNSUP and size(Sq=0) == BAD
    assert _lib.lib().xdit_attn_bwd_workspace_bytes(None) == BAD and _lib.lib().xdit_attn_bwd(None) == BAD


class Table:
    """Host arrays of a list of gradients at made-up addresses."""

    def __init__(self, spans, dtype=_lib.DTYPE_FP32):
        n = len(spans)
        self.ptr = (ctypes.c_uint64 * n)(*(s[0] for s in spans))
        self.numel = (ctypes.c_int64 * n)(*(s[1] for s in spans))
        self.dtype = (ctypes.c_int32 * n)(*([dtype] * n if isinstance(dtype, int) else dtype))
        self.n = n


def norm_args(t, **kw):
    a = _lib.GradNormArgs()
    values = dict(struct_size=ctypes.sizeof(a), kind=_lib.GRADNORM_L2, count=t.n, data=ctypes.addressof(t.ptr), numel=ctypes.addressof(t.numel),
                  dtype=ctypes.addressof(t.dtype), norm=P, workspace=P, workspace_bytes=1 << 30)
    for k, v in {**values, **kw}.items():
        setattr(a, k, v)
    return a


def clip_args(s, d, **kw):
    a = _lib.ClipGradsArgs()
    values = dict(struct_size=ctypes.sizeof(a), max_norm=1.0, count=s.n, src=ctypes.addressof(s.ptr), dst=ctypes.addressof(d.ptr),
                  numel=ctypes.addressof(s.numel), src_dtype=ctypes.addressof(s.dtype), dst_dtype=ctypes.addressof(d.dtype), norm=P)
    for k, v in {**values, **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,needle", [(dict(struct_size=4), "struct_size"), (dict(kind=3), "unknown norm"), (dict(kind=-1), "unknown norm"), (dict(count=-1), "count"),
                                       (dict(count=1 << 25), "count"), (dict(data=None), "table"), (dict(numel=None), "table"), (dict(dtype=None), "table"),
                                       (dict(norm=None), "norm"), (dict(norm=P + 2), "norm"), (dict(workspace=None), "workspace"), (dict(workspace_bytes=8), "workspace"),
                                       (dict(workspace=P + 4), "workspace"), (dict(counter=P + 2), "counter")])
def test_norm_refusals(kw, needle):
    t = Table([(P, 5000), (0x9000, 10)])
    refused(_lib.lib().xdit_grad_norm, norm_args(t, **kw), BAD, needle)


@pytest.mark.parametrize("spans,dtype,needle", [([(0, 5)], 2, "NULL"), ([(P + 2, 5)], 2, "aligned"), ([(P + 1, 5)], 0, "aligned"), ([(P, -1)], 2, "elements"),
                                                ([(P, 1 << 41)], 2, "elements"), ([(P, 5)], 3, "dtype")])
def test_list_refusals(spans, dtype, needle):
    t = Table(spans, dtype)
    refused(_lib.lib().xdit_grad_norm, norm_args(t), BAD, needle)
    refused(_lib.lib().xdit_clip_grads, clip_args(t, t), BAD, needle)
    ok = Table([(P, max(1, spans[0][1]))])
    if spans[0][1] == 5:
        refused(_lib.lib().xdit_clip_grads, clip_args(ok, t, numel=ctypes.addressof(t.numel)), BAD, needle)


def test_norm_workspace():
    size = lambda spans: _lib.lib().xdit_grad_norm_workspace_bytes(ctypes.byref(norm_args(Table(spans))))  # noqa: E731
    assert size([(P, 1)]) == 8 and size([(P, 0)]) == 0
    assert size([(P, 2041)]) == 8 and size([(P, 2042)]) == 16   # up to seven elements before the first 16-byte group
    assert size([(P, 1 << 30)]) == 8 * ((1 << 14) + 1)
    assert _lib.lib().xdit_grad_norm_workspace_bytes(None) == BAD and _lib.lib().xdit_grad_norm(None) == BAD and _lib.lib().xdit_clip_grads(None) == BAD


@pytest.mark.parametrize("src,dst,dtypes", [
    ([(P, 10), (P, 10)], None, (2, 2)),                                  # the same tensor twice
    ([(P, 10), (P + 36, 10)], None, (2, 2)),                             # the last element of one is the first of the other
    ([(P, 10), (P + 400, 10)], [(P + 400, 10), (P, 10)], (2, 2)),        # each other's place
    ([(P, 10)], [(P + 4, 10)], (2, 2)),                                  # its own, shifted
    ([(P, 10)], [(P, 10)], (2, 0)),                                      # its own bytes in another type
    ([(P, 10), (0x9000, 4)], [(0x20000, 10), (P + 8, 4)], (2, 2)),       # a result inside another gradient
    ([(P, 100), (0x9000, 1), (0x9004, 1)], [(P, 100), (0x9004, 1), (0x30000, 1)], (2, 2)),
])
def test_results_that_overlap(src, dst, dtypes):
    s = Table(src, dtypes[0])
    d = s if dst is None else Table(dst, dtypes[1])
    refused(_lib.lib().xdit_clip_grads, clip_args(s, d), BAD, "overlaps")


@pytest.mark.parametrize("norm", [P, P + 36, 0x20000])
def test_a_norm_inside_a_result(norm):
    t = Table([(0x20000, 1), (P, 10)])
    refused(_lib.lib().xdit_clip_grads, clip_args(t, t, norm=norm), BAD, "norm")


@pytest.mark.parametrize("kw,needle", [(dict(struct_size=4), "struct_size"), (dict(count=-1), "count"), (dict(max_norm=-1.0), "max_norm"),
                                       (dict(max_norm=float("nan")), "max_norm"), (dict(max_norm=float("inf")), "max_norm"), (dict(norm=None), "norm"),
                                       (dict(norm=P + 2), "norm"), (dict(norm=None, norm_out=P + 2), "norm"), (dict(norm=None, norm_out=P, kind=3), "unknown norm"),
                                       (dict(norm=None, norm_out=P, kind=2), "workspace"), (dict(norm=None, norm_out=P, kind=2, workspace=P + 4, workspace_bytes=64), "workspace"),
                                       (dict(norm=None, norm_out=P, kind=2, workspace=P, workspace_bytes=4), "workspace"), (dict(src=None), "table"), (dict(dst=None), "table"), (dict(dst_dtype=None), "table")])
def test_clip_refusals(kw, needle):
    t = Table([(P, 10)])
    refused(_lib.lib().xdit_clip_grads, clip_args(t, t, **kw), BAD, needle)


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 1, 8, 64)
    lse = torch.zeros(1, 1, 8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        grad_ops.attn_bwd(q, q, q, q, q, lse)
    with pytest.raises(RuntimeError, match="no CPU path"):
        grad_ops.grad_norm([q])
    with pytest.raises(ValueError, match="4-D"):
        grad_ops.attn_bwd(q, q[0], q, q, q, lse)
    with pytest.raises(ValueError, match="simultaneously"):
        grad_ops.attn_bwd(q, q, q, q, q, lse, k2=q)
    with pytest.raises(ValueError, match="empty"):
        grad_ops.grad_norm([])
    with pytest.raises(ValueError, match="not one"):
        grad_ops.grad_norm(q)


def test_registered_backward_announces_its_gradients():
    with torch._subclasses.FakeTensorMode():
        q, k, k2 = (torch.empty(2, 3, n, 64, dtype=torch.bfloat16, device="cuda") for n in (10, 7, 4))
        lse = torch.empty(2, 3, 10, device="cuda")
        got = torch.ops.xdit_amd.attn_bwd(q, q, k, k, k2, k2, q, lse, None, 0.125, True, True)
        assert [tuple(t.shape) for t in got] == [(2, 3, n, 64) for n in (10, 7, 7, 4, 4)] and all(t.dtype == torch.bfloat16 for t in got)
        assert len(torch.ops.xdit_amd.attn_bwd(q, q, k, k, None, None, q, lse, None, 0.125, True, False)) == 1
        assert len(torch.ops.xdit_amd.attn_bwd(q, q, k, k, None, None, q, lse, None, 0.125, False, True)) == 2
