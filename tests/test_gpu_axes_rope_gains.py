"""The gains' gradients of the rotation, held to the roundings that their sum has, over few and many tokens.

A lane adds d x^ over its wavefront's tokens (at most a 4096th of them, and one more, as at most 1024 workgroups of four wavefronts go over
them) and over its share of the heads (heads / rows that a wavefront holds at once); then 64 / lanes of a row in at most 6 steps, four wavefronts
in 3, every 256th of the at most 1024 + (head groups) workgroups in at most 8, and the 256 runs in 2 + 6.  Each of those additions is off by at
most 2^-24 of the terms' sizes, a term by 32 units of it (the bar of an element), the result by its own rounding.  A bar of that length tells
a lost workgroup: the sums without the rows of four tokens in a row, which the oracle leaves out here, lie outside it.
"""
import pytest
import torch

from oracle import block_oracle as O
from test_gpu_axes_rope import F32, HALF, problem
from xdit_amd import block_ops

pytestmark = pytest.mark.gpu


def inside(got, ref, size, units):
    bound = HALF[got.dtype] * ref.abs() * 1.01 + units * 2.0 ** -24 * size
    return (got.double() - ref).abs() <= bound


@pytest.mark.parametrize("rope", ["interleaved", "split_half"])
@pytest.mark.parametrize("case", [(1, 1, 3, 3, 128, (16, 56, 56)), (2, 33, 5, 1, 64, (16, 24, 24)), (1, 70, 40, 10, 128, (44, 42, 42)), (2, 2600, 5, 3, 64, (16, 24, 24)),
                                  (1, 9001, 3, 1, 128, (44, 42, 42)), (3, 1501, 9, 9, 72, (0, 36, 36)), (1, 4200, 70, 2, 32, (32,)), (1, 1021, 7, 2, 512, (512,))])
def test_gains_gradients(gpu, rope, case):
    B, S, H, Hk, D, axes = case
    q, k, p, f, pairs, qw, kw = problem(gpu, B, S, H, Hk, D, axes, torch.float32, "bshd")
    g = torch.Generator(device=gpu).manual_seed(S)
    dq, dk = (torch.randn(t.shape, generator=g, device=gpu) for t in (q, k))
    got = block_ops.axes_rope_backward(dq, dk, p, f, pairs, q=q, k=k, norm=True, q_weight=qw, k_weight=kw, eps=1e-5, rope=rope)
    slots = 64 // max(1, 1 << (D // 8 - 1).bit_length())
    for x, w, d, dw in ((q, qw, dq, got[2]), (k, kw, dk, got[3])):
        units = 32 + (-(-B * S // 4096) + 1) * -(-x.shape[1] // slots) + 6 + 3 + 8 + 8
        assert units * 2.0 ** -24 >= F32
        _, ref, _, size = O.axes_rope_backward(d, x, w, p, f, pairs, True, 1e-5, rope)
        assert bool(inside(dw, ref, size, units).all()), ((dw.double() - ref).abs() / size).max().item() * 2 ** 24
        for at in {0, S // 2, max(0, S - 4)}:
            lost = d.clone()
            lost[0, :, at:at + 4] = 0
            part = O.axes_rope_backward(lost, x, w, p, f, pairs, True, 1e-5, rope)[1]
            assert not bool(inside(dw, part, size, units).all())
