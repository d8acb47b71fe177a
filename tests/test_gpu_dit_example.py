"""The example's training step with attention in 32 bits: it runs, and its gradients are held as those of test_gpu_train_step.py are."""
import pytest
import torch

import test_gpu_train_step as base
from oracle import grad_oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,head_dim,mlp,grid", [(4, 64, 512, (1, 12, 11)), (4, 72, 640, (1, 9, 7))])
def test_attention_in_32_bits(gpu, heads, head_dim, mlp, grid):
    x, modulation, positions = base.dit.inputs(grid, heads, head_dim)
    m = base.dit.DiTBlock(heads, head_dim, mlp, train=True, fp32_attention=True)
    far = base.dit.check_gradients(m, x, modulation, positions)
    assert set(far) == {"x", "modulation", "q_gain", "k_gain"} and max(far.values()) <= 0.2, far
    r = torch.ones_like(x)
    grads, norm = base.dit.training_step(m, x, modulation.requires_grad_(), positions, r, max_norm=0.5)
    assert float(norm) > 0.5 and abs(O.grad_norm(grads) - 0.5) <= 2.0 ** -8 * 0.5
    m.fp32_attention = False
    other, _ = base.dit.training_step(m, x, modulation, positions, r, max_norm=0.5)
    assert not all(torch.equal(a, b) for a, b in zip(grads, other))   # attention's own roundings
