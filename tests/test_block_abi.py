"""The C entry points around the attention call without a GPU: structs as the header declares them, refusals before
anything is launched, sizes of workspaces, and the shapes that the registered ops announce."""
import ctypes
import os
import subprocess

import pytest
import torch

from xdit_amd import _lib, block, block_ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BAD, UNSUP = _lib.XDIT_ERR_INVALID_ARG, _lib.XDIT_ERR_UNSUPPORTED
NAN = float("nan")

STRUCTS = {"xdit_gated_norm_args": _lib.GatedNormArgs, "xdit_gated_norm_backward_args": _lib.GatedNormBackwardArgs,
           "xdit_axes_rope_tensor": _lib.AxesRopeTensor, "xdit_axes_rope_args": _lib.AxesRopeArgs,
           "xdit_block_quant_args": _lib.BlockQuantArgs, "xdit_block_matmul_args": _lib.BlockMatmulArgs}


def test_structs_match_the_header(tmp_path):
    fields = [(c, f[0]) for c, s in STRUCTS.items() for f in s._fields_]
    src = '#include "xdit_amd_attn.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(){'
    src += "".join('printf("%%zu\\n", sizeof(%s));' % c for c in STRUCTS)
    src += "".join('printf("%%zu\\n", offsetof(%s, %s));' % f for f in fields) + "}\n"
    (tmp_path / "s.c").write_text(src)
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")])
    got = [int(x) for x in subprocess.check_output([str(tmp_path / "s")]).split()]
    assert got == [ctypes.sizeof(s) for s in STRUCTS.values()] + [getattr(STRUCTS[c], f).offset for c, f in fields]


P = 0x1000   # never dereferenced: a refusal comes first


def fill(a, values, changes):
    a.struct_size = ctypes.sizeof(a)
    for k, v in {**values, **changes}.items():
        setattr(a, k, v)
    return a


def rows(C, S=5):
    return _lib.RowStrides(S * C, C)


def norm_args(**kw):
    return fill(_lib.GatedNormArgs(), dict(dtype=_lib.DTYPE_BF16, mod_dtype=_lib.DTYPE_FP32, weight_dtype=_lib.DTYPE_BF16, norm=2, B=2, S=5, C=64, eps=1e-6,
                                           residual_scale=1.0, x=P, y=P, h=P, n=P, gate=P, scale=P, **{t + "_stride": rows(64) for t in "xyhn"},
                                           gate_stride=_lib.RowStrides(64, 0), scale_stride=_lib.RowStrides(64, 0)), kw)


def refused(fn, a, code, needle):
    assert fn(ctypes.byref(a)) == code
    assert needle in _lib.lib().xdit_attn_last_error().decode()


@pytest.mark.parametrize("kw,code,needle", [
    (dict(struct_size=8), BAD, "struct_size"), (dict(dtype=9), BAD, "dtype"), (dict(mod_dtype=_lib.DTYPE_FP16), BAD, "mod_dtype"),
    (dict(weight_dtype=_lib.DTYPE_FP16), BAD, "weight_dtype"), (dict(norm=3), BAD, "norm"), (dict(y_norm=-1), BAD, "norm"),
    (dict(B=0), BAD, "positive"), (dict(S=0), BAD, "positive"), (dict(B=70000), BAD, "too many rows"), (dict(S=1 << 31), BAD, "too many rows"),
    (dict(C=60), UNSUP, "multiple of 8"), (dict(C=8200), UNSUP, "at most 8192"), (dict(residual_scale=NAN), BAD, "residual_scale"),
    (dict(eps=-1.0), BAD, "eps"), (dict(eps=NAN), BAD, "eps"), (dict(y_norm=1, y_eps=float("inf")), BAD, "eps"), (dict(x=None), BAD, "x is NULL"),
    (dict(n=None), BAD, "n is NULL"), (dict(y=None), BAD, "need y"), (dict(h=None, norm=0, scale=None), BAD, "h is NULL"),
    (dict(norm=0), BAD, "need a norm"), (dict(fp8=1), BAD, "n_scale"), (dict(x=P + 8), BAD, "aligned"), (dict(bias=P + 4), BAD, "aligned"),
    (dict(gate_stride=_lib.RowStrides(-64, 0)), BAD, "negative"), (dict(x_stride=_lib.RowStrides(320, 60)), BAD, "multiples of 8"),
    (dict(h_stride=_lib.RowStrides(320, 8)), BAD, "overlap"), (dict(n_stride=_lib.RowStrides(0, 64)), BAD, "overlap"),
])
def test_norm_refusals(kw, code, needle):
    refused(_lib.lib().xdit_gated_norm, norm_args(**kw), code, needle)


def norm_backward_args(**kw):
    return fill(_lib.GatedNormBackwardArgs(), dict(dtype=_lib.DTYPE_BF16, mod_dtype=_lib.DTYPE_BF16, weight_dtype=_lib.DTYPE_BF16, norm=2, B=2, S=5, C=64,
                                                   residual_scale=1.0, dh=P, dn=P, h=P, y=P, stats=P, gate=P, dx=P, dy=P, dgate=P,
                                                   **{t + "_stride": rows(64) for t in ("dh", "dn", "h", "y", "dx", "dy")}), kw)


@pytest.mark.parametrize("kw,code,needle", [
    (dict(struct_size=8), BAD, "struct_size"), (dict(C=12), UNSUP, "multiple of 8"), (dict(dh=None, dn=None), BAD, "both NULL"), (dict(stats=None), BAD, "stats"),
    (dict(norm=0), BAD, "dn needs a norm"), (dict(dn=None, dscale=P), BAD, "need dn"), (dict(y=None), BAD, "need y"), (dict(dx_stride=_lib.RowStrides(0, 64)), BAD, "overlap"),
    (dict(dgate=P + 8), BAD, "aligned"), (dict(), BAD, "workspace"), (dict(workspace=P, workspace_bytes=16), BAD, "workspace"), (dict(workspace=P + 8, workspace_bytes=1 << 30), BAD, "workspace"),
])
def test_norm_backward_refusals(kw, code, needle):
    refused(_lib.lib().xdit_gated_norm_backward, norm_backward_args(**kw), code, needle)


def rope_args(t=None, **kw):
    a = fill(_lib.AxesRopeArgs(), dict(dtype=_lib.DTYPE_BF16, weight_dtype=_lib.DTYPE_FP32, rope=_lib.ROPE_INTERLEAVED, norm=1, pos_bits=64, freq_bits=64, B=1, S=6, D=64,
                                       tensors=1, axes=2, eps=1e-6, positions=P, inv_freq=P, pos_stride_s=2), kw)
    if "pairs" not in kw:
        a.pairs[0], a.pairs[1] = 16, 16
    st = _lib.Strides(3 * 6 * 64, 6 * 64, 64)
    for k, v in {**dict(x=P, dy=P, y=P, weight=P, H=3, x_stride=st, dy_stride=st, y_stride=st), **(t or {})}.items():
        setattr(a.t[0], k, v)
    return a


PAIRS = ctypes.c_int32 * 4


@pytest.mark.parametrize("kw,code,needle", [
    (dict(struct_size=8), BAD, "struct_size"), (dict(dtype=_lib.DTYPE_FP8_E4M3FN), BAD, "dtype"), (dict(weight_dtype=_lib.DTYPE_FP16), BAD, "weight_dtype"), (dict(rope=3), BAD, "rope"),
    (dict(pos_bits=16), BAD, "pos_bits"), (dict(freq_bits=16), BAD, "freq_bits"), (dict(S=0), BAD, "positive"), (dict(S=1 << 31), BAD, "too many"),
    (dict(D=60), UNSUP, "head_dim"), (dict(D=520), UNSUP, "head_dim"), (dict(tensors=3), BAD, "tensors"), (dict(axes=0), BAD, "axes"), (dict(axes=5), BAD, "axes"),
    (dict(eps=NAN), BAD, "eps"), (dict(pairs=PAIRS(-4, 8)), BAD, "pairs"), (dict(pairs=PAIRS(32, 4)), BAD, "fit"), (dict(pairs=PAIRS(8, 6)), UNSUP, "multiple of 4"),
    (dict(positions=None), BAD, "positions"), (dict(positions=P + 4), BAD, "positions"), (dict(inv_freq=P + 4), BAD, "inv_freq"), (dict(pos_stride_s=-1), BAD, "negative"),
    (dict(norm=0), BAD, "weight needs the norm"), (dict(t=dict(H=0)), BAD, "H"), (dict(t=dict(x=None)), BAD, "x is NULL"), (dict(t=dict(y=P + 2)), BAD, "aligned"),
    (dict(t=dict(weight=P + 4)), BAD, "aligned"), (dict(t=dict(x_stride=_lib.Strides(64, 64, 60))), BAD, "multiples"), (dict(t=dict(y_stride=_lib.Strides(64, 0, 64))), BAD, "overlap"),
])
def test_rope_refusals(kw, code, needle):
    refused(_lib.lib().xdit_axes_rope, rope_args(**kw), code, needle)


def test_rope_backward_refusals():
    L = _lib.lib()
    refused(L.xdit_axes_rope_backward, rope_args(t=dict(dy=None)), BAD, "dy is NULL")
    refused(L.xdit_axes_rope_backward, rope_args(t=dict(weight=None, dweight=P)), BAD, "dweight needs weight")
    refused(L.xdit_axes_rope_backward, rope_args(t=dict(dweight=P)), BAD, "workspace")
    assert L.xdit_axes_rope_backward_workspace_bytes(ctypes.byref(rope_args())) == 0
    assert L.xdit_axes_rope_backward_workspace_bytes(ctypes.byref(rope_args(t=dict(dweight=P)))) >= 64 * 4


def quant_args(**kw):
    return fill(_lib.BlockQuantArgs(), dict(dtype=_lib.DTYPE_BF16, block_rows=1, B=1, S=6, K=136, x=P, y=P, scale=P, x_stride=rows(136, 6), y_stride=rows(136, 6)), kw)


@pytest.mark.parametrize("kw,code,needle", [
    (dict(struct_size=8), BAD, "struct_size"), (dict(dtype=_lib.DTYPE_FP8_E4M3FN), BAD, "dtype"), (dict(block_rows=64), BAD, "block_rows"), (dict(K=0), BAD, "positive"), (dict(K=132), UNSUP, "multiple of 8"),
    (dict(S=1 << 31), BAD, "too large"), (dict(block_rows=128, B=2), BAD, "B = 1"), (dict(x=None), BAD, "x is NULL"), (dict(scale=None), BAD, "scale"), (dict(y=P + 4), BAD, "aligned"),
    (dict(x_stride=_lib.RowStrides(0, 132)), BAD, "multiples"), (dict(y_stride=_lib.RowStrides(0, 128)), BAD, "overlap"),
])
def test_quant_refusals(kw, code, needle):
    refused(_lib.lib().xdit_fp8_block_quant, quant_args(**kw), code, needle)


def matmul_args(**kw):
    return fill(_lib.BlockMatmulArgs(), dict(out_dtype=_lib.DTYPE_BF16, bias_dtype=_lib.DTYPE_FP32, cu_count=256, M=5, N=200, K=400, x=P, x_scale=P, w=P, w_scale=P, out=P, x_stride=400,
                                             w_stride=400, out_stride=200, x_scale_stride_m=1, x_scale_stride_k=5, w_scale_stride_n=4, w_scale_stride_k=1), kw)


@pytest.mark.parametrize("kw,code,needle", [
    (dict(struct_size=8), BAD, "struct_size"), (dict(out_dtype=_lib.DTYPE_FP8_E4M3FN), BAD, "out_dtype"), (dict(bias_dtype=_lib.DTYPE_FP16), BAD, "bias_dtype"), (dict(M=0), BAD, "positive"),
    (dict(N=(1 << 24) + 1), BAD, "limited"), (dict(K=392), UNSUP, "multiple of 16"), (dict(cu_count=-1), BAD, "cu_count"), (dict(w=None), BAD, "NULL"), (dict(x=P + 8), BAD, "16-byte"),
    (dict(x_stride=384), BAD, "apart"), (dict(w_stride=408), BAD, "apart"), (dict(x_stride=1 << 24), BAD, "2^24"), (dict(out=P + 1), BAD, "out"), (dict(out_stride=100), BAD, "overlap"),
    (dict(w_scale_stride_k=-1), BAD, "negative"), (dict(bias=P + 2), BAD, "bias"), (dict(workspace=P + 4, workspace_bytes=64), BAD, "workspace"),
])
def test_matmul_refusals(kw, code, needle):
    refused(_lib.lib().xdit_fp8_block_matmul, matmul_args(**kw), code, needle)


def test_null_arguments():
    L = _lib.lib()
    for name in ("xdit_gated_norm", "xdit_gated_norm_backward", "xdit_axes_rope", "xdit_axes_rope_backward", "xdit_fp8_block_quant", "xdit_fp8_block_matmul",
                 "xdit_gated_norm_backward_workspace_bytes", "xdit_axes_rope_backward_workspace_bytes", "xdit_fp8_block_matmul_workspace_bytes"):
        assert getattr(L, name)(None) == BAD


def test_workspace_sizes():
    L = _lib.lib()
    one = L.xdit_gated_norm_backward_workspace_bytes
    assert one(ctypes.byref(norm_backward_args(dgate=None))) == 0
    assert one(ctypes.byref(norm_backward_args())) >= 2 * 64 * 4
    need = L.xdit_fp8_block_matmul_workspace_bytes
    few = need(ctypes.byref(matmul_args(M=1, K=8192, x_stride=8192, w_stride=8192)))
    assert few > 0 and few % (200 * 4) == 0   # K in parts: a row of fp32 sums each
    assert need(ctypes.byref(matmul_args(M=20000, N=4096, out_stride=4096))) == 0
    for exact in (0, 1):   # every plan is a number of parts that fits the chip
        for M in (1, 7, 64, 65, 300, 4000, 40000):
            for N in (1, 100, 2000, 30000):
                for K in (16, 400, 5120, 20000):
                    n = need(ctypes.byref(matmul_args(M=M, N=N, K=K, x_stride=K, w_stride=K, out_stride=N, exact_sums=exact)))
                    assert n >= 0 and n % 4 == 0 and n <= 16 * M * N * 4


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 4, 64)
    q = torch.zeros(1, 2, 4, 64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        block.gated_norm(x)
    with pytest.raises(RuntimeError, match="no CPU path"):
        block_ops.axes_rope(q, None, torch.zeros(4, 1), torch.zeros(32), (32,))
    with pytest.raises(RuntimeError, match="no CPU path"):
        block_ops.fp8_block_quant(x)
    with pytest.raises(ValueError, match="multiple of 16"):
        block.Fp8Linear(torch.zeros(32, 40))
    with pytest.raises(ValueError, match="multiple of 16"):
        block.Fp8Linear(torch.zeros(40, 32), backward=True)
    with pytest.raises(ValueError, match="out_features"):
        block.Fp8Linear(torch.zeros(32))


def test_rope_frequencies():
    f, pairs = block.rope_frequencies((16, 56, 56), theta=(100.0, 10000.0, 10000.0))
    assert pairs == (8, 28, 28) and f.dtype == torch.float64 and f.shape == (64,)
    for i, (axis, theta, dim) in {0: (0, 100.0, 16), 5: (5, 100.0, 16), 8: (0, 10000.0, 56), 40: (4, 10000.0, 56)}.items():
        assert abs(float(f[i]) - theta ** (-2 * axis / dim)) < 1e-15
    for bad in (dict(axes_dim=(3, 5)), dict(axes_dim=(-2,)), dict(axes_dim=(8, 8), theta=(1.0,))):
        with pytest.raises(ValueError):
            block.rope_frequencies(**bad)


def test_registered_ops_announce_shapes():
    o = torch.ops.xdit_amd
    m = lambda *s, **k: torch.empty(*s, device="meta", **k)  # noqa: E731
    x, c = m(2, 5, 200, dtype=torch.bfloat16), m(2, 1, 200)
    none = (None,) * 5
    h, n, st = o.gated_norm(x, x, c, *none, "layer", 1e-6, "none", 1e-6, 1.0)
    assert h.shape == n.shape == x.shape and n.dtype == x.dtype and st.shape == (2, 5, 4) and st.dtype == torch.float32
    assert o.gated_norm(x, None, None, *none, "none", 1e-6, "none", 1e-6, 1.0)[0].shape[1] == 0
    h, n, s = o.gated_norm_fp8(x, x, c, *none, "rms", 1e-6, "none", 1e-6, 1.0)
    assert n.dtype == torch.float8_e4m3fn and s.shape == (2, 5, 2) and s.stride() == (5, 1, 10)
    q, k = m(2, 4, 5, 64), m(2, 2, 5, 64)
    a, b = o.axes_rope(q, k, m(5, 1), m(32), [32], False, None, None, 1e-6, "interleaved")
    assert a.shape == q.shape and b.shape == k.shape
    y, s = o.fp8_block_quant(m(300, 136), 1)
    assert y.shape == (300, 136) and s.shape == (300, 2) and s.stride() == (1, 300)
    w, ws = o.fp8_block_quant(m(300, 136), 128)
    assert ws.shape == (3, 2)
    assert o.fp8_block_matmul(m(2, 5, 136, dtype=torch.float8_e4m3fn), m(2, 5, 2), w, ws, None, torch.float32, None).shape == (2, 5, 300)
    assert o.fp8_linear(x, w, ws, None, None, None).shape == (2, 5, 300)


def test_plans_with_rows_behind_whole_rounds():
    """The workspace tells the parts of K of the rows that are a product of their own: fewer rows than the whole product's."""
    need = _lib.lib().xdit_fp8_block_matmul_workspace_bytes
    for cus, M, N, K, exact, rows in ((3, 485, 206, 1456, 1, 101), (2, 578, 132, 2736, 0, 66)):
        n = need(ctypes.byref(matmul_args(cu_count=cus, M=M, N=N, K=K, exact_sums=exact, x_stride=K, w_stride=K, out_stride=N)))
        assert n > 0 and n % (rows * N * 4) == 0 and n < M * N * 4 * 2


def test_outputs_whose_rows_overlap_across_axes():
    """Strides that clear a row by themselves but meet between two axes: two rows at one place would be written in any order."""
    L, R, T = _lib.lib(), _lib.RowStrides, _lib.Strides
    for kw in (dict(h_stride=R(64, 64)), dict(n_stride=R(128, 64)), dict(h_stride=R(64 * 4, 64)), dict(h_stride=R(96, 64)), dict(h_stride=R(72, 64))):
        refused(L.xdit_gated_norm, norm_args(**kw), BAD, "overlap")
    refused(L.xdit_gated_norm_backward, norm_backward_args(dx_stride=R(64, 64)), BAD, "overlap")
    refused(L.xdit_fp8_block_quant, quant_args(B=2, y_stride=R(136, 136), x_stride=R(6 * 136, 136)), BAD, "overlap")
    for st in (T(18 * 64, 64, 64), T(18 * 64, 128, 64), T(64, 64, 64), T(18 * 64, 64, 128), T(18 * 64, 64 * 5, 64)):
        refused(L.xdit_axes_rope, rope_args(t=dict(y_stride=st)), BAD, "overlap")
    refused(L.xdit_axes_rope, rope_args(B=2, t=dict(y_stride=T(64, 6 * 64, 64))), BAD, "overlap")
    # what does not meet gets as far as the next refusal: any order of the axes, rows with space between them
    for st in (R(320, 64), R(64, 128), R(72, 144), R(1 << 60, 64), R(5 * 72, 72)):
        refused(L.xdit_gated_norm, norm_args(h_stride=st, weight=P + 4), BAD, "weight is not")
    for st in (T(0, 6 * 64, 64), T(0, 64, 3 * 64), T(0, 72, 72 * 3), T(0, 72 * 6, 72)):
        refused(L.xdit_axes_rope, rope_args(t=dict(y_stride=st, weight=P + 4)), BAD, "weight is not")


def test_the_row_stride_of_a_single_row_is_not_looked_at():
    L = _lib.lib()
    for stride in (1 << 24, 1 << 40, 5, -16, 0):
        for kw in (dict(M=1, x_stride=stride), dict(N=1, w_stride=stride)):
            refused(L.xdit_fp8_block_matmul, matmul_args(bias=P + 2, **kw), BAD, "bias")
    refused(L.xdit_fp8_block_matmul, matmul_args(x_stride=1 << 24), BAD, "2^24")
    refused(L.xdit_fp8_block_matmul, matmul_args(w_stride=1 << 24), BAD, "2^24")


def test_no_rotated_pairs_need_no_frequencies():
    L = _lib.lib()
    none = dict(pairs=PAIRS(0, 0), positions=None, inv_freq=None)
    refused(L.xdit_axes_rope_backward, rope_args(t=dict(dweight=P), **none), BAD, "workspace")   # past every check of what is read
    refused(L.xdit_axes_rope_backward, rope_args(t=dict(dweight=P), **{**none, "pairs": PAIRS(0, 4)}), BAD, "positions")


def test_scales_off_their_alignment():
    L = _lib.lib()
    refused(L.xdit_gated_norm, norm_args(fp8=1, n_scale=P + 2), BAD, "n_scale")
    for name in ("x_scale", "w_scale"):
        refused(L.xdit_fp8_block_matmul, matmul_args(**{name: P + 2, "bias": P + 2}), BAD, "x_scale and w_scale")
