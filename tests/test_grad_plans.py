"""How attention's backward pass is laid out, on the CPU: columns that are computed, launches that there can be, tiles and their parts."""
import ctypes
import math
import random

import pytest

from test_grad_abi import BAD, bwd_args, refused
from train_host import CODES, KEYS_ONLY, host
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


FIELDS = ("tiles", "steps", "total", "per_xcd", "whole", "parts", "len", "units")


def plan(B=1, H=1, Sq=1, Sk=1, Sk2=0, D=64, dtype=_lib.DTYPE_BF16, cus=0, need_q=True, need_kv=True):
    """-> the arguments, and how the keys' and the queries' role are cut up."""
    a = _lib.AttnBwdArgs(struct_size=ctypes.sizeof(_lib.AttnBwdArgs), dtype=dtype, B=B, H=H, D=D, Sq=Sq, Sk=Sk, Sk2=Sk2, softmax_scale=1.0, cu_count=cus,
                         dq=16 if need_q else None, dk=16 if need_kv else None)
    out = (ctypes.c_int64 * 18)()
    host().host_plan(ctypes.byref(a), out)
    return a, dict(zip(FIELDS, out[:8])), dict(zip(FIELDS, out[8:16]))


def mixed(role):
    return 0 < role["whole"] < role["per_xcd"] and role["parts"] > 1


@pytest.mark.parametrize("dtype", [_lib.DTYPE_BF16, _lib.DTYPE_FP16, _lib.DTYPE_FP32])
def test_every_step_of_every_tile_is_done_once(dtype):
    """Random calls, real ones and ones planned for other chips: whole tiles, tiles in parts, both at once in either role."""
    rng = random.Random(dtype)
    size = lambda most: int(math.exp(rng.uniform(0, math.log(most))))  # noqa: E731
    seen = {"whole": 0, "cut": 0, "mixed keys": 0, "mixed queries": 0}
    for n in range(4000):
        wants = rng.choice([(True, True), (False, True), (True, False)])
        a, k, q = plan(rng.randint(1, 3), rng.randint(1, 8 if n % 2 else 40), size(8000), size(8000), size(600) if rng.random() < 0.3 else 0, 8 * rng.randint(1, 16), dtype,
                       rng.choice([0, 256, 8 * rng.randint(1, 32)]), *wants)
        assert host().host_walk(ctypes.byref(a)) == 0, {f: getattr(a, f) for f in ("B", "H", "Sq", "Sk", "Sk2", "D", "cu_count", "dq", "dk")}
        for name, role in (("keys", k), ("queries", q)):
            if role["total"]:
                seen["mixed " + name if mixed(role) else "cut" if role["parts"] > 1 else "whole"] += 1
    assert min(seen.values()) >= 20, seen


@pytest.mark.parametrize("kw", KEYS_ONLY)
def test_keys_in_whole_tiles_and_in_parts(kw):
    """The calls of test_gpu_attn_bwd_parts.py have both in the keys' role."""
    assert mixed(plan(need_q=False, **dict(kw, dtype=CODES[kw["dtype"]]))[1])
