"""Tensor-level entry points of what a training step adds to the forward pass: attention's backward pass, the global norm of a
list of gradients and its clipping.

Attention's tensors are logical (B, H, S, D) as those of `ops.attn_fwd`; PyTorch is used for device memory and the current stream only.
"""
import collections.abc
import ctypes
import math

import torch
from torch.autograd.graph import increment_version

from . import _lib, ops
from .block_ops import _plan, _ptr, _scratch
from .ops import TUNING, _capturing, _code, _on_device, _sig, _stream, _stream_lock, _strides

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_GRADS = ("dq", "dk", "dv", "dk2", "dv2")


def attn_bwd(dout, q, k, v, out, lse, softmax_scale=None, k2=None, v2=None, dlse=None, dq=None, dk=None, dv=None, dk2=None, dv2=None,
             need_q=True, need_kv=True):
    """Gradients of `ops.attn_fwd` -> (dq, dk, dv), with a second key/value segment (dq, dk, dv, dk2, dv2):

        P = exp(scale q k^T - lse),  delta = rowsum(dout * out) - dlse,  dS = P * (dout v^T - delta)
        dv = P^T dout,  dk = scale dS^T q,  dq = scale dS k

    dout, out: (B, H, Sq, D) and lse: (B, H, Sq) fp32, of the forward call on the same q, k, v and scale; `dlse`, if given, is the
    gradient of lse.  bf16, fp16 or fp32, head_dim a multiple of 8 up to 128, rows as `attn_fwd` takes them.  `dq` .. `dv2` receive the results
    when given (any such rows, none of them shared with another tensor), new BHSD-contiguous tensors otherwise; `need_q` or `need_kv` False leaves out dq, or the gradients of
    keys and values (None in their places).  Sums are fp32 in a fixed order.

    With the out, lse and dout of attention over several chunks of keys, (k, v) one of them: that chunk's dk and dv, and its share of dq."""
    if not isinstance(q, torch.Tensor) or q.ndim != 4:
        raise ValueError("q must be a 4-D tensor (B, H, S, D)")
    if (k2 is None) != (v2 is None):
        raise ValueError("k2 and v2 should be None or not None simultaneously.")
    device, dtype = q.device, q.dtype
    scale = float(q.shape[-1]) ** -0.5 if softmax_scale is None else float(softmax_scale)
    key = ("attn_bwd", _sig(dout), _sig(q), _sig(k), _sig(v), _sig(out), _sig(lse), scale, _sig(k2), _sig(v2), _sig(dlse), _sig(dq), _sig(dk), _sig(dv),
           _sig(dk2), _sig(dv2), bool(need_q), bool(need_kv), TUNING["cu_count"])

    def build():
        if dtype not in _FLOATS:
            raise NotImplementedError("attention's backward pass takes bf16, fp16 or fp32, not %s" % dtype)
        B, H, Sq, D = q.shape
        a = _lib.AttnBwdArgs()
        a.struct_size = ctypes.sizeof(a)
        a.dtype, a.B, a.H, a.D, a.Sq = _code(dtype), B, H, D, Sq
        a.softmax_scale, a.cu_count = scale, int(TUNING["cu_count"])
        operands = [("q", q), ("dout", dout), ("out", out), ("k", k), ("v", v)] + ([] if k2 is None else [("k2", k2), ("v2", v2)])
        for name, t in operands:
            ops._check4(name, t, device)
            if t.dtype != dtype:
                raise ValueError("%s has dtype %s, q %s" % (name, t.dtype, dtype))
        a.Sk, a.Sk2 = k.shape[2], 0 if k2 is None else k2.shape[2]
        for name, t in operands:
            rows = Sq if name in ("q", "dout", "out") else a.Sk2 if name in ("k2", "v2") else a.Sk
            if tuple(t.shape) != (B, H, rows, D):
                raise ValueError("%s has shape %s, expected %s" % (name, tuple(t.shape), (B, H, rows, D)))
            setattr(a, name + "_stride", _strides(t))
        for name, t in (("lse", lse), ("dlse", dlse)):
            if t is None and name == "dlse":
                continue
            if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or tuple(t.shape) != (B, H, Sq) or t.device != device:
                raise ValueError("%s must be a (%d, %d, %d) fp32 tensor on %s" % (name, B, H, Sq, device))
        a.lse_stride = _strides(lse)
        if dlse is not None:
            a.dlse_stride = _strides(dlse)
        if not (need_q or need_kv):
            raise ValueError("need_q and need_kv are both False")
        wanted = []
        for name, t, of, need in (("dq", dq, q, need_q), ("dk", dk, k, need_kv), ("dv", dv, v, need_kv), ("dk2", dk2, k2, need_kv), ("dv2", dv2, v2, need_kv)):
            if of is None or not need:
                if t is not None:
                    raise ValueError("%s is given but not computed" % name)
                continue
            shape = tuple(of.shape)
            if t is None:
                setattr(a, name + "_stride", _lib.Strides(H * shape[2] * D, shape[2] * D, D))
            else:
                ops._check4(name, t, device)
                if tuple(t.shape) != shape or t.dtype != dtype:
                    raise ValueError("%s has the wrong shape or dtype" % name)
                setattr(a, name + "_stride", _strides(t))
            setattr(a, name, 16)   # any aligned address: the size of the workspace depends on which gradients there are
            wanted.append((name, shape))
        empty = B * H * Sq * D == 0 or a.Sk + a.Sk2 == 0
        with _on_device(device):
            need = 0 if empty else _lib.lib().xdit_attn_bwd_workspace_bytes(ctypes.byref(a))
        if need < 0:
            _lib.check(need)
        return a, wanted, 1 << (need - 1).bit_length(), empty   # a power of two: what calls of growing sizes leave allocated stays below the last one's

    a, wanted, need, empty = _plan(key, build)
    given = {"dq": dq, "dk": dk, "dv": dv, "dk2": dk2, "dv2": dv2}
    result = {name: q.new_empty(shape) if given[name] is None else given[name] for name, shape in wanted}
    if empty:
        for t in result.values():
            t.zero_()
    else:
        for name, t in result.items():
            setattr(a, name, t.data_ptr())
        a.dout, a.q, a.k, a.v, a.out, a.lse, a.dlse = dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), _ptr(dlse)
        a.k2, a.v2 = _ptr(k2), _ptr(v2)
        a.stream = stream = _stream(device)
        with _stream_lock(device, stream), _on_device(device):
            scratch = _scratch(device, stream, need)
            a.workspace, a.workspace_bytes = scratch.data_ptr(), need
            rc = _lib.lib().xdit_attn_bwd(ctypes.byref(a))
        if rc != 0:
            _lib.check(rc)
        increment_version([t for t in given.values() if t is not None])   # what autograd has saved of them is seen to have changed
    return tuple(result.get(name) for name in (_GRADS if k2 is not None else _GRADS[:3]))


_NORMS = {2.0: _lib.GRADNORM_L2, 1.0: _lib.GRADNORM_L1, math.inf: _lib.GRADNORM_MAX}


class _Tables:
    """What the C entry points read of a list of gradients."""
    __slots__ = ("tensors", "device", "seen", "sizes", "dtypes", "ptr", "numel", "dtype", "need", "count")

    def __init__(self, ts):
        if not ts:
            raise ValueError("the list of gradients is empty")
        for t in ts:
            if not isinstance(t, torch.Tensor):
                raise ValueError("gradients must be tensors, not %s" % type(t).__name__)
        self.tensors = ts
        self.device = ts[0].device
        for t in ts:
            if not t.is_cuda:
                raise RuntimeError("a gradient is not on a GPU: the kernels are HIP-only, there is no CPU path")
            if t.device != self.device:
                raise ValueError("a gradient is on %s, expected %s" % (t.device, self.device))
            if t.dtype not in _FLOATS:
                raise ValueError("a gradient has dtype %s, expected bf16, fp16 or fp32" % t.dtype)
            if not t.is_contiguous():
                raise ValueError("a gradient of shape %s is not contiguous" % (tuple(t.shape),))
        self.count = n = len(ts)
        self.seen = list(map(torch.Tensor.data_ptr, ts))
        self.sizes = list(map(torch.Tensor.numel, ts))
        self.ptr = (ctypes.c_uint64 * n)(*self.seen)
        self.numel = (ctypes.c_int64 * n)(*self.sizes)
        self.dtypes = [t.dtype for t in ts]
        self.dtype = (ctypes.c_int32 * n)(*map(_code, self.dtypes))
        self.need = None   # workspace bytes of their norm


class GradList(collections.abc.Sequence):
    """Gradients that stay where they are from step to step (views of a bucket, or kept by `zero_grad(set_to_none=False)`), with the
    tables that `grad_norm` and `clip_grads` pass on.  Those of 84 tensors take 40 us of host time to make and 14 us to look whether a tensor has
    another address, size, type or order than they say; they are made anew then."""

    def __init__(self, tensors):
        if isinstance(tensors, torch.Tensor):
            raise ValueError("expected a list of tensors, not one")
        self._tensors = list(tensors)
        self._tables = _Tables(self._tensors)

    def __len__(self):
        return len(self._tensors)

    def __getitem__(self, i):
        return self._tensors[i]


def _listed(grads):
    if not isinstance(grads, GradList):
        return GradList(grads)._tables
    tables, ts = grads._tables, grads._tensors
    if (list(map(torch.Tensor.data_ptr, ts)) != tables.seen or list(map(torch.Tensor.numel, ts)) != tables.sizes
            or [t.dtype for t in ts] != tables.dtypes or not all(map(torch.Tensor.is_contiguous, ts))):
        tables = grads._tables = _Tables(ts)
    return tables


def _kind(norm_type):
    try:
        return _NORMS[float(norm_type)]
    except (KeyError, TypeError, ValueError):
        raise ValueError("norm_type must be 2, 1 or inf") from None


def _norm_need(g):
    """Workspace bytes of the norm of a list."""
    if g.need is None:
        a = _lib.GradNormArgs()
        a.struct_size = ctypes.sizeof(a)
        a.kind, a.count = _lib.GRADNORM_L2, g.count
        a.data, a.numel, a.dtype = ctypes.addressof(g.ptr), ctypes.addressof(g.numel), ctypes.addressof(g.dtype)
        need = _lib.lib().xdit_grad_norm_workspace_bytes(ctypes.byref(a))
        if need < 0:
            _lib.check(need)
        g.need = need
    return g.need


_COUNTERS = {}


def _counter(device, stream):
    """The counter of a norm's workgroups, which every call leaves at zero: one per device and stream for eager calls; captured ones (whose graphs may run beside
    each other) do without."""
    if _capturing(device, stream):
        return None
    c = _COUNTERS.get((device, stream))
    if c is None:
        c = _COUNTERS[(device, stream)] = torch.zeros(1, dtype=torch.int32, device=device)
    return c.data_ptr()


def _launch(entry, a, device, need, counted=False):
    a.stream = stream = _stream(device)
    with _stream_lock(device, stream), _on_device(device):
        if need:
            scratch = _scratch(device, stream, need)
            a.workspace, a.workspace_bytes = scratch.data_ptr(), need
            if counted:
                a.counter = _counter(device, stream)
        rc = entry(ctypes.byref(a))
    if rc != 0:
        _lib.check(rc)


def grad_norm(grads, norm_type=2.0):
    """Norm of a list of gradients as if they were one vector -> fp32 tensor without dimensions, on their device.

    grads: contiguous bf16, fp16 or fp32 tensors (any mixture, any sizes) of one device, or a `GradList` of them.  norm_type: 2, 1 or inf.  Sums are in
    64 bits, in a fixed order.  Of gradients that are sharded over ranks the norms can be joined before `clip_grads`."""
    kind = _kind(norm_type)
    g = _listed(grads)
    norm = torch.empty((), dtype=torch.float32, device=g.device)
    a = _lib.GradNormArgs(ctypes.sizeof(_lib.GradNormArgs), kind, g.count, ctypes.addressof(g.ptr), ctypes.addressof(g.numel), ctypes.addressof(g.dtype),
                          norm.data_ptr())
    _launch(_lib.lib().xdit_grad_norm, a, g.device, _norm_need(g), counted=True)
    return norm


def clip_grads(grads, max_norm, norm=None, norm_type=2.0, out=None):
    """Scales gradients by min(1, max_norm / (norm + 1e-6)), in place or into the tensors of `out` -> their norm before that.

    `norm` (an fp32 tensor without dimensions or with one element, e.g. joined over ranks) is computed by `grad_norm` where it is not given.
    out: as many tensors of the same sizes, in any of the three dtypes (e.g. the fp32 gradients that an optimizer steps on); none may share memory with
    another, with `norm`, or with a gradient other than its own.  Products are fp32, rounded once; nothing waits for the GPU."""
    kind = _kind(norm_type)
    g = _listed(grads)
    o = g if out is None else _listed(out)
    if o is not g and (o.sizes != g.sizes or o.device != g.device):
        raise ValueError("out must be %d tensors of the gradients' sizes on %s" % (g.count, g.device))
    need = 0
    if norm is None:
        need, result = _norm_need(g), torch.empty((), dtype=torch.float32, device=g.device)
    elif not isinstance(norm, torch.Tensor) or norm.dtype != torch.float32 or norm.numel() != 1 or norm.device != g.device:
        raise ValueError("norm must be an fp32 tensor of one element on %s" % g.device)
    else:
        result = norm
    a = _lib.ClipGradsArgs(ctypes.sizeof(_lib.ClipGradsArgs), float(max_norm), g.count, ctypes.addressof(g.ptr), ctypes.addressof(o.ptr),
                           ctypes.addressof(g.numel), ctypes.addressof(g.dtype), ctypes.addressof(o.dtype), _ptr(norm), result.data_ptr(), kind)
    _launch(_lib.lib().xdit_clip_grads, a, g.device, need)
    increment_version(o.tensors)
    return result
