"""`train_host.hip` as a library, compiled once a session."""
import atexit
import ctypes
import functools
import os
import shutil
import subprocess
import tempfile

from xdit_amd import _lib
from xdit_amd.build import _hipcc

HERE = os.path.dirname(os.path.abspath(__file__))


@functools.lru_cache(maxsize=None)
def host():
    folder = tempfile.mkdtemp()
    atexit.register(shutil.rmtree, folder, ignore_errors=True)
    path = os.path.join(folder, "libtrain_host.so")
    subprocess.check_call([_hipcc(), "-std=c++17", "-O1", "-fPIC", "-shared", "--offload-host-only", "-w", os.path.join(HERE, "train_host.hip"), "-o", path])
    L = ctypes.CDLL(path)
    L.host_message.restype = ctypes.c_char_p
    for name, args in (("xdit_attn_bwd", _lib.AttnBwdArgs), ("xdit_grad_norm", _lib.GradNormArgs), ("xdit_clip_grads", _lib.ClipGradsArgs)):
        getattr(L, name).argtypes = [ctypes.POINTER(args)]
    return L


CODES = {"bf16": _lib.DTYPE_BF16, "fp16": _lib.DTYPE_FP16, "fp32": _lib.DTYPE_FP32}

# Calls for the gradients of keys and values alone that have whole tiles and tiles in parts.
KEYS_ONLY = [dict(dtype=dtype, D=D, H=H, Sq=1003, Sk=Sk, Sk2=Sk2, cus=cus)
             for dtypes, cases in ((("bf16", "fp16"), ((64, 3, 1100, 0, 8), (128, 6, 300, 0, 8), (40, 7, 300, 60, 8), (128, 5, 300, 60, 8))),
                                   (("fp32",), ((64, 8, 300, 0, 8), (72, 6, 300, 60, 8), (128, 7, 300, 0, 24), (128, 5, 300, 60, 24))))
             for dtype in dtypes for D, H, Sk, Sk2, cus in cases]
