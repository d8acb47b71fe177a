"""More tokens than wavefronts, with both tensors, gains and heads that do not fill a wavefront: the bars are those of few tokens."""
import pytest
import torch

from oracle import block_oracle as O
from test_gpu_axes_rope import F32, close, problem
from xdit_amd import block_ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rope", ["interleaved", "split_half"])
@pytest.mark.parametrize("case", [(2, 2600, 5, 3, 64, (16, 24, 24)), (1, 9001, 3, 1, 128, (44, 42, 42)), (3, 1501, 9, 9, 72, (0, 36, 36)), (1, 4200, 70, 2, 32, (32,))])
def test_many_tokens_against_oracle(gpu, dtype, rope, case):
    B, S, H, Hk, D, axes = case
    for layout, norm in (("bshd", True), ("bhsd", True), ("bhsd", False)):
        q, k, p, f, pairs, qw, kw = problem(gpu, B, S, H, Hk, D, axes, dtype, layout, "grid")
        if not norm:
            qw = kw = None
        opt = dict(norm=norm, q_weight=qw, k_weight=kw, eps=1e-5, rope=rope)
        yq, yk = block_ops.axes_rope(q, k, p, f, pairs, **opt)
        dq, dk = torch.randn_like(yq), torch.randn_like(yk)
        got = block_ops.axes_rope_backward(dq, dk, p, f, pairs, q=q, k=k, **opt)
        again = block_ops.axes_rope_backward(dq, dk, p, f, pairs, q=q, k=k, **opt)
        assert all(a is None or torch.equal(a, b) for a, b in zip(got, again))
        for x, w, y, d, dx, dw in ((q, qw, yq, dq, got[0], got[2]), (k, kw, yk, dk, got[1], got[3])):
            pre = O.axes_rope(x, w, p * 0, f, pairs, norm, 1e-5, rope)
            close(y, O.axes_rope(x, w, p, f, pairs, norm, 1e-5, rope), pre.abs().amax(-1, keepdim=True))
            rdx, rdw, sx, sw = O.axes_rope_backward(d, x, w, p, f, pairs, norm, 1e-5, rope)
            close(dx, rdx, sx)
            if dw is not None:
                close(dw, rdw, sw, F32 + (x.shape[1] * S * B / 4 + 40) * 2.0 ** -24)
