"""Tensor-level entry points of the operators around the attention call of a DiT block: the norms with
their modulation, gate and residual and the rotation of q and k by positions on several axes, forward and
backward, and the projections' fp8 product with a scale per block of 128 and its quantiser.

Hidden states are (B, S, C), q and k logical (B, H, S, D), with any outer strides (multiples of 16 bytes) and a
unit stride over the last dimension; PyTorch is used for device memory and the current stream only.  Argument structs are kept per call signature and thread,
as those of `ops.attn_fwd` are.
"""
import ctypes

import torch

from . import _lib
from .ops import TUNING, _PLANS_MAX, _RETIRED, _TLS, _capturing, _code, _on_device, _sig, _stream, _stream_lock

_ROWNORM = {None: _lib.ROWNORM_NONE, "rms": _lib.ROWNORM_RMS, "layer": _lib.ROWNORM_LAYER}
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_SCRATCH = {}


def _scratch(device, stream, nbytes):
    """Scratch of a call, to be held until it has launched; taken under the stream's lock.  The eager calls of one (device,
    stream) are ordered and share a buffer; one that a call has outgrown stays allocated.  A captured call has a buffer of
    its own from the graph's memory pool, which its later calls may take over in the graph's order."""
    if _capturing(device, stream):
        return torch.empty(int(nbytes), dtype=torch.uint8, device=device)
    buf = _SCRATCH.get((device, stream))
    if buf is None or buf.numel() < nbytes:
        if buf is not None:
            _RETIRED.append(buf)
        buf = _SCRATCH[(device, stream)] = torch.empty(int(nbytes), dtype=torch.uint8, device=device)
    return buf


def _plan(key, build):
    """The argument struct of a call signature on this thread, from a store of its own: a block makes ten signatures a sequence length, and
    attention's plans go all at once when theirs is full."""
    plans = _TLS.__dict__.setdefault("block_plans", {})
    plan = plans.get(key)
    if plan is None:
        plan = build()
        if len(plans) >= _PLANS_MAX:
            plans.clear()
        plans[key] = plan
    return plan


def _check(name, t, shape, dtypes, device):
    if not isinstance(t, torch.Tensor):
        raise ValueError("%s must be a tensor" % name)
    if t.device != device:
        raise ValueError("%s is on %s, expected %s" % (name, t.device, device))
    if not t.is_cuda:
        raise RuntimeError("%s is not on a GPU: the kernels are HIP-only, there is no CPU path" % name)
    if t.dtype not in dtypes:
        raise ValueError("%s has dtype %s, expected one of %s" % (name, t.dtype, ", ".join(str(d) for d in dtypes)))
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError("%s has shape %s, expected %s" % (name, tuple(t.shape), tuple(shape)))
    if t.ndim and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError("%s must have a unit stride over its last dimension" % name)


def _hidden(x):
    if not isinstance(x, torch.Tensor) or x.ndim != 3:
        raise ValueError("hidden states must be a 3-D tensor (B, S, C)")
    _check("hidden states", x, None, _FLOATS, x.device)
    return x.shape


def _rows(t):
    return _lib.RowStrides(t.stride(0), t.stride(1))


def _mod(name, t, B, S, C, dtype, device):
    """A modulation tensor (B or 1, S or 1, C) or (B or 1, C) -> (row strides, whether it has a row per token)."""
    _check(name, t, None, (dtype, torch.float32), device)
    s = t.shape
    if t.ndim not in (2, 3) or s[-1] != C or s[0] not in (B, 1) or (t.ndim == 3 and s[1] not in (S, 1)):
        raise ValueError("%s has shape %s, expected (%d or 1, [%d or 1,] %d)" % (name, tuple(s), B, S, C))
    per_token = t.ndim == 3 and s[1] == S and S > 1
    return _lib.RowStrides(t.stride(0) if s[0] > 1 else 0, t.stride(1) if per_token else 0), per_token


def _shared(name, tensors, dtype):
    """The one dtype of those of `tensors` that are given (`dtype` if none is)."""
    found = {t.dtype for t in tensors if t is not None}
    if len(found) > 1:
        raise ValueError("%s must share a dtype" % name)
    return found.pop() if found else dtype


def _norm_code(name, kind):
    try:
        return _ROWNORM[kind]
    except (KeyError, TypeError):
        raise ValueError("%s must be None, 'rms' or 'layer'" % name) from None


def _new_like(t):
    """A new contiguous tensor of t's shape, dtype and device."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _ptr(t):
    return None if t is None else t.data_ptr()


def gated_norm(x, y=None, gate=None, scale=None, shift=None, weight=None, bias=None, norm="layer", eps=1e-6, y_norm=None,
               y_weight=None, y_eps=1e-6, residual_scale=1.0, fp8=False, return_stats=False, out_h=None):
    """The residual addition behind a block and the modulated norm in front of the next one, in one pass -> (h, n):

        v = y, or its "rms" / "layer" norm times y_weight        (`y_norm`)
        h = x + residual_scale * gate * v                        (x itself where y is None)
        n = norm(h) * weight + bias, times (1 + scale), plus shift

    x, y: (B, S, C), bf16 / fp16 / fp32, C a multiple of 8 up to 8192.  gate, scale, shift: (B, C), (B, 1, C) or one row per
    token (B, S, C); weight, bias, y_weight: (C,); each in x's dtype or fp32, or None.  `norm` None leaves out n (returned as
    None).  All arithmetic is fp32, h and n are rounded once.  `fp8`: n is a pair (e4m3 tensor, scales (B, S, ceil(C / 128))
    fp32) quantised from the unrounded n, as by `fp8_block_quant` up to fp32 roundings of scale and quotient; `fp8_block_matmul` takes it where C is
    a multiple of 16.  `return_stats` appends the (B, S, 4) fp32 statistics that
    `gated_norm_backward` takes.  `out_h` receives h (it may be x: the residual stream is then updated in place)."""
    try:
        B, S, C = x.shape
    except (AttributeError, TypeError, ValueError):
        raise ValueError("hidden states must be a 3-D tensor (B, S, C)") from None
    device, dtype = x.device, x.dtype
    eps, y_eps, residual_scale = float(eps), float(y_eps), float(residual_scale)   # values: a tensor would be known by its identity
    key = ("gnorm", _sig(x), _sig(y), _sig(gate), _sig(scale), _sig(shift), _sig(weight), _sig(bias), _sig(y_weight), _sig(out_h), norm, y_norm, fp8,
           eps, y_eps, residual_scale)

    def build():
        _hidden(x)
        a = _lib.GatedNormArgs()
        a.struct_size = ctypes.sizeof(a)
        a.dtype = _code(dtype)
        a.mod_dtype = _code(_shared("gate, scale and shift", (gate, scale, shift), dtype))
        a.weight_dtype = _code(_shared("weight, bias and y_weight", (weight, bias, y_weight), dtype))
        a.norm, a.y_norm, a.fp8 = _norm_code("norm", norm), _norm_code("y_norm", y_norm), 1 if fp8 else 0
        a.B, a.S, a.C = B, S, C
        a.eps, a.y_eps, a.residual_scale = eps, y_eps, residual_scale
        a.x_stride = _rows(x)
        if y is not None:
            _check("y", y, x.shape, (dtype,), device)
            a.y_stride = _rows(y)
        elif gate is not None or y_weight is not None or y_norm is not None:
            raise ValueError("gate, y_weight and y_norm need y")
        if norm is None and (fp8 or any(t is not None for t in (scale, shift, weight, bias))):
            raise ValueError("fp8, scale, shift, weight and bias need a norm")
        for name, t in (("gate", gate), ("scale", scale), ("shift", shift)):
            if t is not None:
                setattr(a, name + "_stride", _mod(name, t, B, S, C, dtype, device)[0])
        for name, t in (("weight", weight), ("bias", bias), ("y_weight", y_weight)):
            if t is not None:
                _check(name, t, (C,), (dtype, torch.float32), device)
        if out_h is not None:
            _check("out_h", out_h, x.shape, (dtype,), device)
        a.h_stride = _lib.RowStrides(S * C, C) if out_h is None else _rows(out_h)
        a.n_stride = _lib.RowStrides(S * C, C)
        return a

    a = _plan(key, build)
    h = out_h
    if h is None:
        h = x if y is None else _new_like(x)
    n = n_scale = stats = None
    if fp8:
        n = x.new_empty((B, S, C), dtype=torch.float8_e4m3fn)
        n_scale = x.new_empty_strided((B, S, (C + 127) // 128), (S, 1, B * S), dtype=torch.float32)
    elif norm is not None:
        n = _new_like(x)
    if return_stats:
        stats = x.new_empty((B, S, 4), dtype=torch.float32)
    if B * S * C and (y is not None or norm is not None or out_h is not None):
        a.x, a.y, a.n = x.data_ptr(), _ptr(y), _ptr(n)
        a.h = h.data_ptr() if y is not None or out_h is not None else None
        a.n_scale, a.stats = _ptr(n_scale), _ptr(stats)
        a.gate, a.scale, a.shift, a.weight, a.bias, a.y_weight = _ptr(gate), _ptr(scale), _ptr(shift), _ptr(weight), _ptr(bias), _ptr(y_weight)
        a.stream = _stream(device)
        with _on_device(device):
            rc = _lib.lib().xdit_gated_norm(ctypes.byref(a))
        if rc != 0:
            _lib.check(rc)
    elif return_stats:   # nothing to compute: the statistics of norms that are absent
        stats.zero_()[..., 1::2] = 1
    if fp8:
        n = (n, n_scale)
    return (h, n, stats) if return_stats else (h, n)


def gated_norm_backward(dh, dn, h, stats, y=None, gate=None, scale=None, shift=None, weight=None, bias=None, norm="layer", y_norm=None,
                        y_weight=None, residual_scale=1.0):
    """Gradients of `gated_norm` from dh and dn (either may be None), its results h and stats, its y and its
    parameters -> a dict of dx and of those of dy, dgate, dscale, dshift, dweight, dbias and dy_weight whose operand was given.
    dgate, dscale and dshift have the shapes of gate, scale and shift (a batch dimension of 1 that was broadcast is refused:
    expand it); scale and shift must agree on having a row per token.  Sums over rows are fp32, in a fixed order."""
    B, S, C = _hidden(h)
    device, dtype = h.device, h.dtype
    residual_scale = float(residual_scale)
    key = ("gnorm_bwd", _sig(dh), _sig(dn), _sig(h), _sig(stats), _sig(y), _sig(gate), _sig(scale), _sig(shift), _sig(weight), _sig(bias), _sig(y_weight),
           norm, y_norm, residual_scale)

    def build():
        if dh is None and dn is None:
            raise ValueError("dh and dn are both None")
        a = _lib.GatedNormBackwardArgs()
        a.struct_size = ctypes.sizeof(a)
        a.dtype = _code(dtype)
        mod = _shared("gate, scale and shift", (gate, scale, shift), dtype)
        wt = _shared("weight, bias and y_weight", (weight, bias, y_weight), dtype)
        a.mod_dtype, a.weight_dtype = _code(mod), _code(wt)
        a.norm, a.y_norm = _norm_code("norm", norm), _norm_code("y_norm", y_norm)
        a.B, a.S, a.C = B, S, C
        a.residual_scale = residual_scale
        _check("stats", stats, (B, S, 4), (torch.float32,), device)
        if not stats.is_contiguous():
            raise ValueError("stats must be contiguous")
        for name, t in (("dh", dh), ("dn", dn), ("y", y)):
            if t is not None:
                _check(name, t, h.shape, (dtype,), device)
                setattr(a, name + "_stride", _rows(t))
        a.h_stride = _rows(h)
        if dn is not None and norm is None:
            raise ValueError("dn needs a norm")
        if y is None and (gate is not None or y_weight is not None or y_norm is not None):
            raise ValueError("gate, y_weight and y_norm need y")
        per = {}
        for name, t in (("gate", gate), ("scale", scale), ("shift", shift)):
            if t is not None:
                strides, per[name] = _mod(name, t, B, S, C, dtype, device)
                if t.shape[0] != B:
                    raise ValueError("%s is broadcast over the batch: expand it, its gradient has a row per batch entry" % name)
                if name != "shift":
                    setattr(a, name + "_stride", strides)
        if "scale" in per and "shift" in per and per["scale"] != per["shift"]:
            raise ValueError("scale and shift must both have a row per token or neither")
        a.gate_per_token = 1 if per.get("gate") else 0
        a.mod_per_token = 1 if per.get("scale") or per.get("shift") else 0
        for name, t in (("weight", weight), ("bias", bias), ("y_weight", y_weight)):
            if t is not None:
                _check(name, t, (C,), (dtype, torch.float32), device)
        a.dx_stride = a.dy_stride = _lib.RowStrides(S * C, C)
        outs = [("dx", (B, S, C), dtype)]
        if y is not None:
            outs.append(("dy", (B, S, C), dtype))
            outs += [("dgate", tuple(gate.shape), mod)] if gate is not None else []
            outs += [("dy_weight", (C,), wt)] if y_weight is not None else []
        if dn is not None:
            outs += [("d" + name, tuple(t.shape), mod) for name, t in (("scale", scale), ("shift", shift)) if t is not None]
            outs += [("d" + name, (C,), wt) for name, t in (("weight", weight), ("bias", bias)) if t is not None]
        for name, _, _ in outs:
            setattr(a, name, 16)   # any aligned address: the size of the workspace depends on which outputs there are
        with _on_device(device):
            need = _lib.lib().xdit_gated_norm_backward_workspace_bytes(ctypes.byref(a)) if B * S * C else 0
        if need < 0:
            _lib.check(need)
        return a, outs, need

    a, outs, need = _plan(key, build)
    result = {name: h.new_empty(shape, dtype=dt) for name, shape, dt in outs}
    if B * S * C == 0:
        for t in result.values():
            t.zero_()
        return result
    for name, t in result.items():
        setattr(a, name, t.data_ptr())
    a.dh, a.dn, a.h, a.y, a.stats = _ptr(dh), _ptr(dn), h.data_ptr(), _ptr(y), stats.data_ptr()
    a.gate, a.scale, a.weight, a.bias, a.y_weight = _ptr(gate), _ptr(scale), _ptr(weight), _ptr(bias), _ptr(y_weight)
    a.stream = stream = _stream(device)
    with _stream_lock(device, stream), _on_device(device):
        if need:
            scratch = _scratch(device, stream, need)
            a.workspace, a.workspace_bytes = scratch.data_ptr(), need
        rc = _lib.lib().xdit_gated_norm_backward(ctypes.byref(a))
    if rc != 0:
        _lib.check(rc)
    return result


def rope_frequencies(axes_dim, theta=10000.0, device=None):
    """Frequencies of a rotation in which every axis turns its own part of head_dim, `axes_dim[a]` columns of it ->
    (inv_freq fp64, pairs): theta ** (-2 i / axes_dim[a]) for the pairs i of axis a; `theta` may be one per axis."""
    thetas = theta if isinstance(theta, (tuple, list)) else (theta,) * len(axes_dim)
    if len(thetas) != len(axes_dim) or any(d % 2 or d < 0 for d in axes_dim):
        raise ValueError("axes_dim must be even numbers, with one theta or one per axis")
    parts = [t ** (-torch.arange(0, d, 2, dtype=torch.float64) / max(d, 1)) for d, t in zip(axes_dim, thetas)]
    return torch.cat(parts).to(device), tuple(d // 2 for d in axes_dim)


_ROPE = {"interleaved": _lib.ROPE_INTERLEAVED, "split_half": _lib.ROPE_SPLIT_HALF}
_POS_BITS = {torch.float32: -32, torch.int32: 32, torch.int64: 64}


def _bhsd(name, t, B, S, D, dtype, device):
    if not isinstance(t, torch.Tensor) or t.ndim != 4:
        raise ValueError("%s must be a 4-D tensor (B, H, S, D)" % name)
    _check(name, t, (B, t.shape[1], S, D), (dtype,), device)
    return _lib.Strides(t.stride(0), t.stride(1), t.stride(2))


def _rope_args(first, tensors, positions, inv_freq, pairs, norm, eps, rope):
    """The fields that forward and backward share.  `tensors`: (name, x, dy, y, weight) of q and, if it is there, k."""
    B, _, S, D = first.shape
    device, dtype = first.device, first.dtype
    if rope not in _ROPE:
        raise ValueError("rope must be one of %s" % (sorted(_ROPE),))
    if not 1 <= len(pairs) <= _lib.ROPE_MAX_AXES:
        raise ValueError("between 1 and %d axes are supported" % _lib.ROPE_MAX_AXES)
    a = _lib.AxesRopeArgs()
    a.struct_size = ctypes.sizeof(a)
    a.dtype, a.rope, a.norm, a.eps = _code(dtype), _ROPE[rope], 1 if norm else 0, eps
    a.weight_dtype = _code(_shared("q_weight and k_weight", [t[4] for t in tensors], dtype))
    _check("positions", positions, None, tuple(_POS_BITS), device)
    A = len(pairs)
    if positions.ndim not in (2, 3) or tuple(positions.shape[-2:]) != (S, A) or (positions.ndim == 3 and positions.shape[0] not in (B, 1)):
        raise ValueError("positions has shape %s, expected ([%d or 1,] %d, %d)" % (tuple(positions.shape), B, S, A))
    _check("inv_freq", inv_freq, (sum(pairs),), (torch.float32, torch.float64), device)
    a.pos_bits, a.freq_bits = _POS_BITS[positions.dtype], 64 if inv_freq.dtype == torch.float64 else 32
    a.pos_stride_s = positions.stride(-2)
    a.pos_stride_b = positions.stride(0) if positions.ndim == 3 and positions.shape[0] > 1 else 0
    a.B, a.S, a.D = B, S, D
    a.tensors, a.axes = len(tensors), A
    for i, n in enumerate(pairs):
        a.pairs[i] = n
    for i, (name, x, dy, y, weight) in enumerate(tensors):
        t = a.t[i]
        t.H = (x if x is not None else dy).shape[1]
        for kind, v in (("x", x), ("dy", dy), ("y", y)):
            if v is not None:
                strides = _bhsd(name if kind == "x" else "%s of %s" % (kind, name), v, B, S, D, dtype, device)
                if v.shape[1] != t.H:
                    raise ValueError("%s: the tensors have %d and %d heads" % (name, v.shape[1], t.H))
                setattr(t, kind + "_stride", strides)
        if y is None:
            t.y_stride = _lib.Strides(t.H * S * D, S * D, D)
        if weight is not None:
            if not norm:
                raise ValueError("%s has a weight but no norm" % name)
            _check(name + "_weight", weight, (D,), (dtype, torch.float32), device)
    return a


def axes_rope(q, k, positions, inv_freq, pairs, norm=False, q_weight=None, k_weight=None, eps=1e-6, rope="interleaved", out_q=None, out_k=None):
    """Rotates q and k (logical (B, H, S, D), any strides; k may be None or have other heads than q) by positions on up to
    four axes, after an RMSNorm over head_dim with gains `q_weight` / `k_weight` (D entries, q's dtype or fp32, or None) where
    `norm` is set -> (q, k), new BHSD-contiguous tensors or `out_q` / `out_k` (which may be q and k themselves).

    positions: (S, A) or (B, S, A), fp32, int32 or int64.  Pair p belongs to the axis whose part of `pairs` (pairs per axis) it
    lies in and turns by position * inv_freq[p] (`rope_frequencies` makes both; sum(pairs) a multiple of 4).  `rope`: a pair is
    the columns (2p, 2p + 1), "interleaved", or (p, p + sum(pairs)), "split_half"; columns from 2 sum(pairs) on are not rotated.
    Angles are reduced in fp64, the rest is fp32, the result is rounded once."""
    if not isinstance(q, torch.Tensor) or q.ndim != 4:
        raise ValueError("q must be a 4-D tensor (B, H, S, D)")
    device, dtype, pairs, eps = q.device, q.dtype, tuple(map(int, pairs)), float(eps)
    B, H, S, D = q.shape
    key = ("arope", _sig(q), _sig(k), _sig(positions), _sig(inv_freq), pairs, norm, _sig(q_weight), _sig(k_weight), eps, rope, _sig(out_q), _sig(out_k))

    def build():
        _check("q", q, None, _FLOATS, device)
        if k is None and (k_weight is not None or out_k is not None):
            raise ValueError("k_weight and out_k need k")
        if k is not None and not isinstance(k, torch.Tensor):
            raise ValueError("k must be a 4-D tensor (B, H, S, D)")
        return _rope_args(q, [("q", q, None, out_q, q_weight)] + ([("k", k, None, out_k, k_weight)] if k is not None else []),
                          positions, inv_freq, pairs, norm, eps, rope)

    a = _plan(key, build)
    oq = _new_like(q) if out_q is None else out_q
    ok = out_k
    if k is not None and ok is None:
        ok = _new_like(k)
    if B * S * D == 0:
        return oq, ok
    t = a.t[0]
    t.x, t.y, t.weight = q.data_ptr(), oq.data_ptr(), _ptr(q_weight)
    if k is not None:
        t = a.t[1]
        t.x, t.y, t.weight = k.data_ptr(), ok.data_ptr(), _ptr(k_weight)
    a.positions, a.inv_freq = positions.data_ptr(), inv_freq.data_ptr()
    a.stream = _stream(device)
    with _on_device(device):
        rc = _lib.lib().xdit_axes_rope(ctypes.byref(a))
    if rc != 0:
        _lib.check(rc)
    return oq, ok


def axes_rope_backward(dq, dk, positions, inv_freq, pairs, q=None, k=None, norm=False, q_weight=None, k_weight=None, eps=1e-6, rope="interleaved"):
    """Gradients of `axes_rope` from those of its results -> (dq, dk, dq_weight, dk_weight), new BHSD-contiguous tensors;
    None for what was not there (dk may be None).  With the norm q and k are the inputs of the forward call.  The gains'
    gradients are summed in fp32 in a fixed order."""
    if not isinstance(dq, torch.Tensor) or dq.ndim != 4:
        raise ValueError("dq must be a 4-D tensor (B, H, S, D)")
    device, dtype, pairs, eps = dq.device, dq.dtype, tuple(map(int, pairs)), float(eps)
    B, H, S, D = dq.shape
    if not norm:
        q = k = None
    key = ("arope_bwd", _sig(dq), _sig(dk), _sig(positions), _sig(inv_freq), pairs, _sig(q), _sig(k), norm, _sig(q_weight), _sig(k_weight), eps, rope)

    def build():
        _check("dq", dq, None, _FLOATS, device)
        if norm and (q is None or (dk is not None and k is None)):
            raise ValueError("the gradient of the norm needs q (and k)")
        if dk is None and (k is not None or k_weight is not None):
            raise ValueError("k and k_weight need dk")
        if dk is not None and not isinstance(dk, torch.Tensor):
            raise ValueError("dk must be a 4-D tensor (B, H, S, D)")
        a = _rope_args(dq, [("q", q, dq, None, q_weight)] + ([("k", k, dk, None, k_weight)] if dk is not None else []),
                       positions, inv_freq, pairs, norm, eps, rope)
        for i, w in enumerate((q_weight, k_weight)):
            a.t[i].dweight = None if w is None else 16   # any aligned address: only what is asked for decides the size
        with _on_device(device):
            need = _lib.lib().xdit_axes_rope_backward_workspace_bytes(ctypes.byref(a)) if B * S * D else 0
        if need < 0:
            _lib.check(need)
        return a, need

    a, need = _plan(key, build)
    outs, grads = [], []
    for d, w in ((dq, q_weight), (dk, k_weight)):
        outs.append(None if d is None else _new_like(d))
        grads.append(None if w is None else w.new_empty((D,)))
    if B * S * D == 0:
        for g in grads:
            if g is not None:
                g.zero_()
        return (*outs, *grads)
    for t, d, x, w, y, g in zip(a.t, (dq, dk), (q, k), (q_weight, k_weight), outs, grads):
        t.dy, t.x, t.weight, t.y, t.dweight = _ptr(d), _ptr(x), _ptr(w), _ptr(y), _ptr(g)
    a.positions, a.inv_freq = positions.data_ptr(), inv_freq.data_ptr()
    a.stream = stream = _stream(device)
    with _stream_lock(device, stream), _on_device(device):
        if need:
            scratch = _scratch(device, stream, need)
            a.workspace, a.workspace_bytes = scratch.data_ptr(), need
        rc = _lib.lib().xdit_axes_rope_backward(ctypes.byref(a))
    if rc != 0:
        _lib.check(rc)
    return (*outs, *grads)


def fp8_block_quant(x, block_rows=1):
    """fp8 (e4m3) values and fp32 scales of x, a scale per 1 x 128 block (`block_rows` 1: activations) or 128 x 128 block
    (128: weights) -> (y, scale), x about y * scale:  scale = absmax / 448 (1 for a block of zeros), y = e4m3(x / scale).

    x: (M, K), or (B, S, K) with `block_rows` 1, bf16 / fp16 / fp32, any row strides that are multiples of 16 bytes, K a multiple of 8;
    the last blocks are cut off by the tensor.  y is contiguous; scale is (M, ceil(K / 128)) or (B, S, ceil(K / 128)), the scales
    of one block of columns side by side in memory, or contiguous (ceil(M / 128), ceil(K / 128))."""
    if not isinstance(x, torch.Tensor) or x.ndim not in (2, 3) or (x.ndim == 3 and block_rows != 1):
        raise ValueError("x must be (M, K), or (B, S, K) with blocks of one row")
    device = x.device
    key = ("bquant", _sig(x), block_rows)
    B, S, K = x.shape if x.ndim == 3 else (1, *x.shape)
    kb = (K + 127) // 128

    def build():
        _check("x", x, None, _FLOATS, device)
        a = _lib.BlockQuantArgs()
        a.struct_size = ctypes.sizeof(a)
        a.dtype, a.block_rows = _code(x.dtype), int(block_rows)
        a.B, a.S, a.K = B, S, K
        a.x_stride = _lib.RowStrides(x.stride(0) if x.ndim == 3 else 0, x.stride(-2))
        a.y_stride = _lib.RowStrides(S * K, K)
        return a

    a = _plan(key, build)
    y = x.new_empty(x.shape, dtype=torch.float8_e4m3fn)
    if block_rows != 1:
        scale = x.new_empty(((S + 127) // 128, kb), dtype=torch.float32)
    elif x.ndim == 3:
        scale = x.new_empty_strided((B, S, kb), (S, 1, B * S), dtype=torch.float32)
    else:
        scale = x.new_empty_strided((S, kb), (1, S), dtype=torch.float32)
    if B * S * K:
        a.x, a.y, a.scale, a.stream = x.data_ptr(), y.data_ptr(), scale.data_ptr(), _stream(device)
        with _on_device(device):
            rc = _lib.lib().xdit_fp8_block_quant(ctypes.byref(a))
        if rc != 0:
            _lib.check(rc)
    return y, scale


def fp8_block_matmul(x, x_scale, w, w_scale, bias=None, out_dtype=torch.bfloat16, out=None, exact_sums=None):
    """x w^T + bias of block-scaled fp8 matrices -> (M, N) (or (B, S, N)) in `out_dtype`:

        out[m, n] = sum over blocks kb of  x_scale[m, kb] * w_scale[n // 128, kb] * (x[m, kb] . w[n, kb])  + bias[n]

    x: (M, K) or (B, S, K) e4m3 with scales (M, ceil(K / 128)) or (B, S, ceil(K / 128)); w: (N, K) with scales (ceil(N / 128),
    ceil(K / 128)) (`fp8_block_quant` of both; scales may have any strides); K a multiple of 16; bias (N,) in out_dtype or fp32.
    The blocks' sums are held in fp32 and the result is rounded once; the same call gives the same bits.  `exact_sums` True:
    products are exact and summed in fp32; False: the fp8 matrix instructions, twice as fast, which add eight consecutive k at a
    time with every product cut at 2^-13 of the largest one's binade (1.4e-5 to 3.3e-5 of the result's size: nothing beside a rounding to bf16, 0.2 to
    1.2 % more error beside one to fp16); None: exact for fp32 results, where that shows."""
    for name, t in (("x", x), ("x_scale", x_scale), ("w", w), ("w_scale", w_scale)):
        if not isinstance(t, torch.Tensor):
            raise ValueError("%s must be a tensor" % name)
    device, shape = x.device, x.shape
    if x.ndim == 3:
        if x_scale.ndim != 3 or x_scale.shape[:2] != shape[:2]:
            raise ValueError("x_scale has shape %s, expected (%d, %d, ceil(K / 128))" % (tuple(x_scale.shape), shape[0], shape[1]))
        x, x_scale = x.flatten(0, 1), x_scale.flatten(0, 1)
    key = ("bmm", _sig(x), _sig(x_scale), _sig(w), _sig(w_scale), _sig(bias), out_dtype, _sig(out), exact_sums, TUNING["cu_count"])
    if x.ndim != 2 or w.ndim != 2:
        raise ValueError("x must be (M, K) or (B, S, K), w (N, K)")
    (M, K), N = x.shape, w.shape[0]

    def build():
        kb = (K + 127) // 128
        _check("x", x, None, (torch.float8_e4m3fn,), device)
        _check("w", w, (N, K), (torch.float8_e4m3fn,), device)
        for name, t, rows in (("x_scale", x_scale, M), ("w_scale", w_scale, (N + 127) // 128)):
            if t.device != device or t.dtype != torch.float32 or tuple(t.shape) != (rows, kb):
                raise ValueError("%s must be a (%d, %d) fp32 tensor on %s" % (name, rows, kb, device))
        if out_dtype not in _FLOATS:
            raise ValueError("out_dtype must be bf16, fp16 or fp32")
        if bias is not None:
            _check("bias", bias, (N,), (out_dtype, torch.float32), device)
        a = _lib.BlockMatmulArgs()
        a.struct_size = ctypes.sizeof(a)
        a.out_dtype, a.bias_dtype = _code(out_dtype), _code(out_dtype if bias is None else bias.dtype)
        a.cu_count = int(TUNING["cu_count"])
        a.exact_sums = int(out_dtype == torch.float32 if exact_sums is None else bool(exact_sums))
        a.M, a.N, a.K = M, N, K
        a.x_stride, a.w_stride, a.out_stride = x.stride(0), w.stride(0), N
        if out is not None:
            _check("out", out, (*shape[:-1], N), (out_dtype,), device)
            flat = out.view(-1, N) if out.ndim == 3 else out
            a.out_stride = flat.stride(0)
        a.x_scale_stride_m, a.x_scale_stride_k = x_scale.stride()
        a.w_scale_stride_n, a.w_scale_stride_k = w_scale.stride()
        with _on_device(device):
            need = _lib.lib().xdit_fp8_block_matmul_workspace_bytes(ctypes.byref(a)) if M * N * K else 0
        if need < 0:
            _lib.check(need)
        return a, need

    a, need = _plan(key, build)
    y = x.new_empty((*shape[:-1], N), dtype=out_dtype) if out is None else out
    if M * N == 0:
        return y
    if K == 0:
        return y.zero_() if bias is None else y.copy_(bias)
    a.x, a.x_scale, a.w, a.w_scale, a.bias, a.out = x.data_ptr(), x_scale.data_ptr(), w.data_ptr(), w_scale.data_ptr(), _ptr(bias), y.data_ptr()
    a.stream = stream = _stream(device)
    with _stream_lock(device, stream), _on_device(device):
        if need:
            scratch = _scratch(device, stream, need)
            a.workspace, a.workspace_bytes = scratch.data_ptr(), need
        rc = _lib.lib().xdit_fp8_block_matmul(ctypes.byref(a))
    if rc != 0:
        _lib.check(rc)
    return y
