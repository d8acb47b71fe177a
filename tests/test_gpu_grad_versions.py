"""Clipping in place between a graph and its backward pass, on the GPU."""
import pytest
import torch

from xdit_amd import grad_ops

pytestmark = pytest.mark.gpu


def test_a_clipped_gradient_that_a_graph_has_saved(gpu):
    p = torch.ones(100, device=gpu, requires_grad=True)
    (g,) = torch.autograd.grad(p.pow(3).sum(), p, create_graph=True)
    second = (g * g).sum()   # saves g
    grad_ops.clip_grads([g], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        second.backward()
