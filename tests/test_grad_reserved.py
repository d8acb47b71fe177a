"""Reserved fields of the training entries are zero."""
import ctypes

import pytest

from test_grad_abi import BAD, P, Table, bwd_args, clip_args, refused
from xdit_amd import _lib


@pytest.mark.parametrize("value", [1, -1, 1 << 30])
def test_reserved_fields(value):
    t = Table([(P, 10)])
    refused(_lib.lib().xdit_clip_grads, clip_args(t, t, reserved0=value, norm=P + 2), BAD, "reserved0")   # ahead of what else is wrong
    refused(_lib.lib().xdit_attn_bwd, bwd_args(reserved0=value), BAD, "reserved0")
    assert _lib.lib().xdit_attn_bwd_workspace_bytes(ctypes.byref(bwd_args(reserved0=value))) == BAD
