"""Where the norm of a clipping lies: one that the call writes is apart from the gradients, which other workgroups still read then."""
import ctypes

import pytest

from test_grad_abi import BAD, P, Table, clip_args, refused
from train_host import host
from xdit_amd import _lib

FAR = 1 << 20


def clip(norm_out=None, norm=None):
    s, d = Table([(FAR, 100), (4 * FAR, 10)]), Table([(2 * FAR, 100), (5 * FAR, 10)])
    return clip_args(s, d, norm=norm, norm_out=norm_out, kind=2, workspace=P, workspace_bytes=64), s, d


@pytest.mark.parametrize("at", [FAR, FAR + 200, FAR + 396, 4 * FAR + 36, 2 * FAR + 4, 5 * FAR])
def test_a_norm_that_is_written_inside_a_tensor(at):
    a, *keep = clip(norm_out=at)
    refused(_lib.lib().xdit_clip_grads, a, BAD, "norm")


@pytest.mark.parametrize("at", [FAR - 4, FAR + 400, 3 * FAR, 4 * FAR + 40])
def test_a_norm_beside_them(at):
    a, *keep = clip(norm_out=at)
    assert host().xdit_clip_grads(ctypes.byref(a)) == 0


def test_a_norm_that_is_read_may_be_a_gradient():
    a, *keep = clip(norm=FAR + 8)
    assert host().xdit_clip_grads(ctypes.byref(a)) == 0
