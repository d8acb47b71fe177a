"""Where gradients may lie: apart from each other and from the inputs, whichever part of them it is.  On the CPU, by the C entries' own checks."""
import ctypes
import random

import pytest

from train_host import host
from xdit_amd import _lib

B, H, SQ, SK, SK2, D = 2, 3, 100, 80, 20, 64
INPUTS, GRADS = ("dout", "q", "k", "v", "k2", "v2", "out"), ("dq", "dk", "dv", "dk2", "dv2")
ROWS = {"dout": SQ, "q": SQ, "out": SQ, "dq": SQ, "k": SK, "v": SK, "dk": SK, "dv": SK, "k2": SK2, "v2": SK2, "dk2": SK2, "dv2": SK2}
FAR = 1 << 24


def args(**places):
    """A call whose tensors lie far apart, but for those in `places`: name -> (address, strides)."""
    a = _lib.AttnBwdArgs(struct_size=ctypes.sizeof(_lib.AttnBwdArgs), dtype=_lib.DTYPE_BF16, B=B, H=H, D=D, Sq=SQ, Sk=SK, Sk2=SK2, softmax_scale=0.125, cu_count=256,
                         workspace=FAR, workspace_bytes=FAR)
    for i, (name, S) in enumerate(ROWS.items()):
        at, st = places.get(name, ((i + 3) * FAR, (H * S * D, S * D, D)))
        setattr(a, name, at)
        setattr(a, name + "_stride", _lib.Strides(*st))
    for i, name in enumerate(("lse", "dlse")):
        at, st = places.get(name, ((i + 20) * FAR, (H * SQ, SQ, 1)))
        setattr(a, name, at)
        setattr(a, name + "_stride", _lib.Strides(*st))
    return a


def taken(**places):
    return host().xdit_attn_bwd(ctypes.byref(args(**places))) == 0


def refused(what, **places):
    assert host().xdit_attn_bwd(ctypes.byref(args(**places))) == _lib.XDIT_ERR_INVALID_ARG
    assert what in host().host_message().decode()


def dense(name):
    S = ROWS[name]
    return H * S * D, S * D, D


def test_tensors_apart():
    assert taken()


@pytest.mark.parametrize("grad", GRADS)
@pytest.mark.parametrize("other", INPUTS + ("lse", "dlse"))
@pytest.mark.parametrize("shift", ["row", "head", "last row", "before"])
def test_a_gradient_inside_an_input(grad, other, shift):
    at = args()
    S = ROWS.get(other, SQ)
    row = D * 2 if other in ROWS else 4   # bytes
    offset = {"row": row, "head": S * row, "last row": B * H * S * row - row, "before": -(B * H * ROWS[grad] - 1) * D * 2}[shift]
    refused("overlaps an input", **{grad: (getattr(at, other) + offset, dense(grad))})


@pytest.mark.parametrize("one,other", [(a, b) for i, a in enumerate(GRADS) for b in GRADS[:i]])
@pytest.mark.parametrize("rows", [1, 7, -1])
def test_gradients_across_each_other(one, other, rows):
    refused("gradients overlap", **{one: (getattr(args(), other) + rows * D * 2, dense(one))})


def test_views_of_one_buffer():
    """q, k, v as views of a projection's output, text behind the image's rows, and their gradients as views of its gradient."""
    st = (SQ * 3 * H * D, D, 3 * H * D)
    packed = {n: (FAR * 40 + i * H * D * 2, st) for i, n in enumerate(("q", "k", "v"))}
    assert taken(**packed, **{"d" + n: (FAR * 50 + i * H * D * 2, st) for i, n in enumerate(("q", "k", "v"))})
    refused("overlaps an input", **packed, dq=(FAR * 40 + 2, st))   # between the columns of q and k
    refused("gradients overlap", dq=(FAR * 50, st), dk=(FAR * 50 + (H * D - D // 2) * 2, st))
    # an input's gradient where the buffer has room for it
    assert taken(**packed, dq=(FAR * 50, st), dk=(FAR * 50 + H * D * 2, st), dv=(FAR * 50 + 2 * H * D * 2, st))
    wide = (SQ * 6 * H * D, D, 6 * H * D)
    six = {n: (FAR * 60 + i * H * D * 2, wide) for i, n in enumerate(("q", "k", "v", "dq", "dk", "dv"))}
    assert taken(**six)
    # image and text rows of one tensor, in either memory order
    for st in ((H * (SK + SK2) * D, (SK + SK2) * D, D), ((SK + SK2) * H * D, D, H * D)):
        assert taken(dk=(FAR * 40, st), dk2=(FAR * 40 + SK * st[2] * 2, st))
        refused("gradients overlap", dk=(FAR * 40, st), dk2=(FAR * 40 + (SK - 1) * st[2] * 2, st))


def test_inputs_may_lie_on_each_other():
    st = dense("q")
    assert taken(q=(FAR * 40, st), dout=(FAR * 40, st), out=(FAR * 40 + D * 2, st))
    one_head = (SK * D, 0, D)
    assert taken(k=(FAR * 40, one_head), v=(FAR * 40, one_head))
    refused("overlaps an input", k=(FAR * 40, one_head), dv=(FAR * 40 + D * 2, dense("dv")))


def bytes_of(x):
    at, width, *axes = x
    rows = [0]
    for n, stride in zip(axes[::2], axes[1::2]):
        rows = [r + i * stride for r in rows for i in range(n)]
    return {at + r + w for r in rows for w in range(width)}


@pytest.mark.parametrize("seed", range(4))
def test_shared_bytes_against_every_byte(seed):
    rng = random.Random(seed)
    pack = lambda v: (ctypes.c_int64 * 8)(*v)  # noqa: E731
    seen = [0, 0]
    for _ in range(1500):
        strides = [rng.choice([0, 4, 8, 12, 24, 48, 60, 96]) for _ in range(3)]

        def box():
            other = rng.random() < 0.4
            axes = [v for s in strides for v in (rng.randint(1, 5), rng.choice([4, 8, 16, 20, 36, 100]) if other and rng.random() < 0.5 else s)]
            return [1000 + rng.randint(0, 150), rng.choice([1, 4, 8]), *axes]

        x, y = box(), box()
        want = bool(bytes_of(x) & bytes_of(y))
        seen[want] += 1
        assert bool(host().host_share_bytes(pack(x), pack(y))) == want, (x, y)
    assert min(seen) > 200
