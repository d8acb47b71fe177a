"""How attention's backward pass is laid out, on the CPU: columns that are computed, launches that there can be."""
import ctypes

import pytest

from test_grad_abi import BAD, bwd_args, refused
from train_host import host
from xdit_amd import _lib


@pytest.mark.parametrize("D", range(8, 129, 8))
def test_fp32_computes_the_columns_that_there_are(D):
    """One rule for all head_dims: no column more above 32, none of them a case of its own."""
    assert host().host_f32_groups(D) * 8 == max(D, 32)


MANY = 1 << 23


@pytest.mark.parametrize("kw,fits", [
    (dict(B=MANY // 2, H=1, Sq=1, Sk=1), True), (dict(B=MANY, H=1, Sq=1, Sk=1), False),   # a workgroup for a tile of either role
    (dict(B=1, H=MANY, Sq=1, Sk=1, dq=None), True), (dict(B=2 * MANY, H=1, Sq=1, Sk=1, dq=None), False),
    (dict(B=MANY, H=1, Sq=1, Sk=1, dq=None, dtype=_lib.DTYPE_FP16), False),   # a block of the statistics for the queries and one for the values
    (dict(B=1, H=1, Sq=1 << 29, Sk=1 << 29), True), (dict(B=1, H=1, Sq=1 << 29, Sk=1, dtype=_lib.DTYPE_FP32), True)])
def test_launches_of_too_many_threads_are_refused(kw, fits):
    a = bwd_args(**{**dict(Sk2=0, dk2=None, dv2=None, D=8), **kw})
    L = _lib.lib()
    need = L.xdit_attn_bwd_workspace_bytes(ctypes.byref(a))
    assert need > 0 if fits else need == BAD and "too large" in L.xdit_attn_last_error().decode()
    if not fits:
        a.workspace_bytes = 1 << 60
        refused(L.xdit_attn_bwd, a, BAD, "too large")
