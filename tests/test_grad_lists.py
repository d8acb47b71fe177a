"""Lists of gradients whose tensors change where they are, on the CPU: the tables that the kernels read follow, or the call is refused."""
import pytest
import torch

from xdit_amd import grad_ops


class OnGpu(torch.Tensor):
    is_cuda = True


def gpu(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnGpu)


def listed(g):
    t = grad_ops._listed(g)
    return list(t.ptr), list(t.numel), list(t.dtype)


BF16, FP16, FP32 = (grad_ops._code(t) for t in (torch.bfloat16, torch.float16, torch.float32))


def test_another_type_of_the_same_size():
    a, b = gpu(6), gpu(4, 5, dtype=torch.bfloat16)
    g = grad_ops.GradList([a, b])
    at, place = b.data_ptr(), b.data
    b.data = place.view(torch.float16)
    assert listed(g) == ([a.data_ptr(), at], [6, 20], [FP32, FP16])
    b.data = place
    assert listed(g)[2] == [FP32, BF16]


def test_as_many_bytes_in_another_type():
    a = gpu(10)
    g = grad_ops.GradList([a])
    at, place = a.data_ptr(), a.data
    a.data = place.view(torch.bfloat16)
    assert listed(g) == ([at], [20], [BF16])
    a.data = place
    assert listed(g) == ([at], [10], [FP32])


@pytest.mark.parametrize("change", [lambda t: t.t_(), lambda t: setattr(t, "data", t.data.t()), lambda t: t.as_strided_((5, 4), (0, 1))])
def test_another_order(change):
    a = gpu(4, 5)
    g = grad_ops.GradList([gpu(3), a])
    listed(g)
    change(a)
    with pytest.raises(ValueError, match="contiguous"):
        grad_ops._listed(g)


def test_a_type_that_no_kernel_has():
    a = gpu(10)
    g = grad_ops.GradList([a])
    a.data = a.data.view(torch.int32)
    with pytest.raises(ValueError, match="dtype"):
        grad_ops._listed(g)


def test_nothing_changed():
    g = grad_ops.GradList([gpu(3), gpu(4, 5)])
    assert grad_ops._listed(g) is grad_ops._listed(g)
