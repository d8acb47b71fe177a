"""`torch.library` custom ops over the HIP entry points, so `torch.compile` can trace through them.

The reference wraps a vendor kernel the same way (xfuser/core/distributed/attention_backend.py:383-399:
`@custom_op("xfuser::flydsl_attn_kernel", mutates_args=())` plus a `register_fake` that returns
`torch.empty_like(query)`).  Here every op has a device implementation that calls the C ABI
(`xdit_amd.ops`) and a fake implementation that only describes the outputs:

    xdit_amd::attn_fwd        (q, k, v, softmax_scale)                      -> (out, lse)
    xdit_amd::attn_fwd_joint  (q, k, v, k2, v2, softmax_scale)              -> (out, lse)
    xdit_amd::attn_fwd_fp8    (q, k, v, q_descale, k_descale, v_descale,
                               softmax_scale, out_fp16)                     -> (out, lse)
    xdit_amd::lse_merge       (acc_out, acc_lse, block_out, block_lse, first)   in place
    xdit_amd::lse_merge_final (acc_out, acc_lse, block_out, block_lse, final_out)  in place
    xdit_amd::attn_fwd_fp8_joint (q, k, v, k2, v2, q_descale, k_descale, v_descale,
                               softmax_scale, out_fp16)                     -> (out, lse)
    xdit_amd::attn_fwd_accumulate (q, k, v, k2?, v2?, acc_out, acc_lse, final_out?, first,
                               discard_acc_out, softmax_scale)              in place (one ring step)
    xdit_amd::fp8_quant       (x, per_tensor, hadamard_block)               -> (y, descale)
    xdit_amd::fp8_quant_ex    (x, x2?, scale?, per_tensor, hadamard_block)  -> (y, y2, descale)
    xdit_amd::norm_rope       (x, weight, cos, sin, eps, norm, rope,
                               rope_row0, rope_rows)                        -> y (BHSD-contiguous)

    xdit_amd::attn_bwd        (dout, q, k, v, k2?, v2?, out, lse, dlse?, softmax_scale, need_q,
                               need_kv)             -> list of gradients of attn_fwd or attn_fwd_joint
    xdit_amd::attn_result     (out, lse, q, k, v, k2?, v2?, softmax_scale)    -> (out, lse), differentiable in q .. v2

and the operators around the attention call (`xdit_amd.block_ops`), with their gradients:

    xdit_amd::gated_norm      (x, y?, gate?, scale?, shift?, weight?, bias?, y_weight?, norm, eps,
                               y_norm, y_eps, residual_scale)          -> (h, n, stats)
    xdit_amd::gated_norm_fp8  (the same)                               -> (h, n, n_scale)
    xdit_amd::gated_norm_backward (dh?, dn?, h, stats, y?, gate?, scale?, shift?, weight?, bias?,
                               y_weight?, norm, y_norm, residual_scale) -> list of gradients
    xdit_amd::axes_rope       (q, k?, positions, inv_freq, pairs, norm, q_weight?, k_weight?, eps,
                               rope)                                   -> (q, k)
    xdit_amd::axes_rope_backward (dq, dk?, positions, inv_freq, pairs, q?, k?, norm, q_weight?,
                               k_weight?, eps, rope)                   -> list of gradients
    xdit_amd::fp8_block_quant (x, block_rows)                          -> (y, scale)
    xdit_amd::fp8_block_matmul (x, x_scale, w, w_scale, bias?, out_dtype, exact_sums?) -> y
    xdit_amd::fp8_linear      (x, w, w_scale, w_t?, w_t_scale?, bias?) -> y

Attention's tensors are logical BHSD (any B/H/S strides); outputs are BHSD-contiguous, lse is (B,H,Sq)
fp32.  The ops are registered for GPU tensors only: there is no CPU implementation.
"""
from typing import List, Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.library import custom_op, register_autograd, register_fake

from . import block_ops, grad_ops, ops

Tensor = torch.Tensor


def _fake_out_lse(query: Tensor, out_dtype) -> Tuple[Tensor, Tensor]:
    B, H, Sq, D = query.shape
    return (query.new_empty((B, H, Sq, D), dtype=out_dtype),
            query.new_empty((B, H, Sq), dtype=torch.float32))


@custom_op("xdit_amd::attn_fwd", mutates_args=(), device_types="cuda")
def attn_fwd(query: Tensor, key: Tensor, value: Tensor, softmax_scale: float) -> Tuple[Tensor, Tensor]:
    return ops.attn_fwd(query, key, value, softmax_scale=softmax_scale)


@register_fake("xdit_amd::attn_fwd")
def _attn_fwd_fake(query, key, value, softmax_scale):
    return _fake_out_lse(query, query.dtype)


@custom_op("xdit_amd::attn_fwd_joint", mutates_args=(), device_types="cuda")
def attn_fwd_joint(query: Tensor, key: Tensor, value: Tensor, key2: Tensor, value2: Tensor,
                   softmax_scale: float) -> Tuple[Tensor, Tensor]:
    return ops.attn_fwd(query, key, value, softmax_scale=softmax_scale, k2=key2, v2=value2)


@register_fake("xdit_amd::attn_fwd_joint")
def _attn_fwd_joint_fake(query, key, value, key2, value2, softmax_scale):
    return _fake_out_lse(query, query.dtype)


def _attn_rows(t):
    """A tensor whose rows attention's kernels read in place; a copy of any other (autograd may pass an expanded or transposed gradient)."""
    es, (sb, sh, ss, sd) = t.element_size(), t.stride()
    if (sd == 1 and ss >= t.shape[3] and ss * es < 1 << 24 and sb * es % 16 == 0 and sh * es % 16 == 0 and ss * es % 16 == 0
            and t.data_ptr() % 16 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


@custom_op("xdit_amd::attn_bwd", mutates_args=(), device_types="cuda")
def attn_bwd(dout: Tensor, query: Tensor, key: Tensor, value: Tensor, key2: Optional[Tensor], value2: Optional[Tensor], out: Tensor, lse: Tensor,
             dlse: Optional[Tensor], softmax_scale: float, need_q: bool, need_kv: bool) -> List[Tensor]:
    """`grad_ops.attn_bwd`: those of dq, dk, dv, dk2 and dv2 that there are."""
    r = grad_ops.attn_bwd(_attn_rows(dout), query, key, value, _attn_rows(out), lse, softmax_scale, key2, value2, dlse, need_q=need_q, need_kv=need_kv)
    return [t for t in r if t is not None]


@register_fake("xdit_amd::attn_bwd")
def _attn_bwd_fake(dout, query, key, value, key2, value2, out, lse, dlse, softmax_scale, need_q, need_kv):
    return [t.new_empty(t.shape) for t, need in ((query, need_q), (key, need_kv), (value, need_kv), (key2, need_kv), (value2, need_kv))
            if t is not None and need]


def _attn_grads(needs, dout, dlse, query, key, value, key2, value2, out, lse, softmax_scale):
    """Gradients of query, key, value, key2 and value2 as far as `needs` (one truth value each) asks; None for the others."""
    need_q, need_kv = bool(needs[0]), any(needs[1:])
    if (dout is None and dlse is None) or not (need_q or need_kv):
        return (None,) * 5
    if dout is None:
        dout = torch.zeros_like(out)
    r = iter(torch.ops.xdit_amd.attn_bwd(dout, query, key, value, key2, value2, out, lse, dlse, softmax_scale, need_q, need_kv))
    there = (need_q, need_kv, need_kv, need_kv and key2 is not None, need_kv and key2 is not None)
    return tuple(next(r) if t else None for t in there)


def _attn_fwd_setup(ctx, inputs, output):
    *tensors, ctx.scale = inputs
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(*tensors, *output)


def _attn_fwd_grad(ctx, dout, dlse):
    q, k, v, out, lse = ctx.saved_tensors
    return (*_attn_grads(ctx.needs_input_grad[:3], dout, dlse, q, k, v, None, None, out, lse, ctx.scale)[:3], None)


def _attn_fwd_joint_grad(ctx, dout, dlse):
    return (*_attn_grads(ctx.needs_input_grad[:5], dout, dlse, *ctx.saved_tensors, ctx.scale), None)


register_autograd("xdit_amd::attn_fwd", _attn_fwd_grad, setup_context=_attn_fwd_setup)
register_autograd("xdit_amd::attn_fwd_joint", _attn_fwd_joint_grad, setup_context=_attn_fwd_setup)


def attn_grad_wanted(*tensors):
    """Whether an attention call on these tensors has to leave a graph behind (of the types that have a backward pass; fp8 has none).  Gradients are those
    of reverse mode: tangents of forward-mode differentiation are refused."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("forward-mode differentiation is not supported: the tangent would be lost")
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad and t.dtype in (torch.bfloat16, torch.float16, torch.float32) for t in tensors)


class _NoGradient(torch.autograd.Function):
    @staticmethod
    def forward(ctx, what, call, *tensors):
        ctx.what = what
        return call()

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("%s has no gradient: call it on detached tensors, or under torch.no_grad()" % ctx.what)


@torch._disable_dynamo   # (torch.compiler.disable would import the compiler here, a second)
def _untraced(what, call, *tensors):
    return _NoGradient.apply(what, call, *tensors)


def without_gradient(what, call, *tensors, traced=False):
    """`call()`, new tensors made of `tensors` by kernels without a backward pass.  Where one of them asks for a gradient, the result's backward pass raises: it would
    be left out in silence.  In traced code the call is left to Python then, unless it is one of registered operators (`traced`), which raise by themselves."""
    compiling = torch.compiler.is_compiling()
    if (compiling and traced) or not attn_grad_wanted(*tensors):
        return call()
    return (_untraced if compiling else _NoGradient.apply)(what, call, *tensors)


class RingAttention(torch.autograd.Function):
    """Attention over all of key, value [, key2, value2] that `call()` computes in its own steps -> (out, lse); the gradient is one backward
    call over the whole key range, from the merged output and log-sum-exp.  `bshd`: query, key, value and out are BSHD, lse is (B, H, Sq) either way."""

    @staticmethod
    def forward(ctx, call, scale, bshd, query, key, value, key2, value2):
        out, lse = call()
        ctx.scale, ctx.bshd = scale, bshd
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(query, key, value, key2, value2, out, lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dlse):
        def t(x):
            return x.transpose(1, 2) if ctx.bshd and x is not None else x

        q, k, v, k2, v2, out, lse = ctx.saved_tensors
        grads = _attn_grads(ctx.needs_input_grad[3:], t(dout), dlse, t(q), t(k), t(v), t(k2), t(v2), t(out), lse, ctx.scale)
        return (None, None, None, *map(t, grads))


@custom_op("xdit_amd::attn_result", mutates_args=(), device_types="cuda")
def attn_result(out: Tensor, lse: Tensor, query: Tensor, key: Tensor, value: Tensor, key2: Optional[Tensor], value2: Optional[Tensor],
                softmax_scale: float) -> Tuple[Tensor, Tensor]:
    """Copies of the out and lse that several calls made of attention over all of key, value [, key2, value2]: with its gradient, in a traced graph."""
    return out.clone(), lse.clone()


@register_fake("xdit_amd::attn_result")
def _attn_result_fake(out, lse, query, key, value, key2, value2, softmax_scale):
    return torch.empty_like(out), torch.empty_like(lse)


def _attn_result_setup(ctx, inputs, output):
    _attn_fwd_setup(ctx, inputs[2:], output)


def _attn_result_grad(ctx, dout, dlse):
    return (None, None, *_attn_grads(ctx.needs_input_grad[2:7], dout, dlse, *ctx.saved_tensors, ctx.scale), None)


register_autograd("xdit_amd::attn_result", _attn_result_grad, setup_context=_attn_result_setup)


def attn_in_steps(call, scale, bshd, *tensors):
    """`RingAttention` of query, key, value, key2, value2, in traced code by the registered operator."""
    if not torch.compiler.is_compiling():
        return RingAttention.apply(call, scale, bshd, *tensors)
    with torch.no_grad():
        out, lse = call()
    if not bshd:
        return torch.ops.xdit_amd.attn_result(out, lse, *tensors, scale)
    out, lse = torch.ops.xdit_amd.attn_result(out.transpose(1, 2), lse, *(None if t is None else t.transpose(1, 2) for t in tensors), scale)
    return out.transpose(1, 2), lse


@custom_op("xdit_amd::attn_fwd_fp8", mutates_args=(), device_types="cuda")
def attn_fwd_fp8(query: Tensor, key: Tensor, value: Tensor, q_descale: Tensor, k_descale: Tensor,
                 v_descale: Tensor, softmax_scale: float, out_fp16: bool) -> Tuple[Tensor, Tensor]:
    return ops.attn_fwd(query, key, value, softmax_scale=softmax_scale, q_descale=q_descale,
                        k_descale=k_descale, v_descale=v_descale,
                        out_dtype=torch.float16 if out_fp16 else torch.bfloat16)


@register_fake("xdit_amd::attn_fwd_fp8")
def _attn_fwd_fp8_fake(query, key, value, q_descale, k_descale, v_descale, softmax_scale, out_fp16):
    return _fake_out_lse(query, torch.float16 if out_fp16 else torch.bfloat16)


@custom_op("xdit_amd::attn_fwd_fp8_joint", mutates_args=(), device_types="cuda")
def attn_fwd_fp8_joint(query: Tensor, key: Tensor, value: Tensor, key2: Tensor, value2: Tensor, q_descale: Tensor,
                       k_descale: Tensor, v_descale: Tensor, softmax_scale: float, out_fp16: bool) -> Tuple[Tensor, Tensor]:
    return ops.attn_fwd(query, key, value, softmax_scale=softmax_scale, k2=key2, v2=value2, q_descale=q_descale,
                        k_descale=k_descale, v_descale=v_descale,
                        out_dtype=torch.float16 if out_fp16 else torch.bfloat16)


@register_fake("xdit_amd::attn_fwd_fp8_joint")
def _attn_fwd_fp8_joint_fake(query, key, value, key2, value2, q_descale, k_descale, v_descale, softmax_scale, out_fp16):
    return _fake_out_lse(query, torch.float16 if out_fp16 else torch.bfloat16)


@custom_op("xdit_amd::attn_fwd_accumulate", mutates_args=("acc_out", "acc_lse", "final_out"), device_types="cuda")
def attn_fwd_accumulate(query: Tensor, key: Tensor, value: Tensor, key2: Optional[Tensor], value2: Optional[Tensor],
                        acc_out: Tensor, acc_lse: Tensor, final_out: Optional[Tensor], first: bool,
                        discard_acc_out: bool, softmax_scale: float) -> None:
    """One ring step (`ops.attn_fwd_accumulate`): the block of (key, value) [+ (key2, value2)] folded
    into the fp32 accumulator in the attention kernel's epilogue; `final_out` also receives the
    merged rows in the query's dtype."""
    ops.attn_fwd_accumulate(query, key, value, acc_out, acc_lse, first=first, final_out=final_out,
                            discard_acc_out=discard_acc_out, softmax_scale=softmax_scale, k2=key2, v2=value2)


@register_fake("xdit_amd::attn_fwd_accumulate")
def _attn_fwd_accumulate_fake(query, key, value, key2, value2, acc_out, acc_lse, final_out, first, discard_acc_out, softmax_scale):
    return None


@custom_op("xdit_amd::lse_merge", mutates_args=("acc_out", "acc_lse"), device_types="cuda")
def lse_merge(acc_out: Tensor, acc_lse: Tensor, block_out: Tensor, block_lse: Tensor, first: bool) -> None:
    ops.lse_merge(acc_out, acc_lse, block_out, block_lse, first=first)


@register_fake("xdit_amd::lse_merge")
def _lse_merge_fake(acc_out, acc_lse, block_out, block_lse, first):
    return None


@custom_op("xdit_amd::lse_merge_final", mutates_args=("acc_out", "acc_lse", "final_out"), device_types="cuda")
def lse_merge_final(acc_out: Tensor, acc_lse: Tensor, block_out: Tensor, block_lse: Tensor, final_out: Tensor) -> None:
    ops.lse_merge(acc_out, acc_lse, block_out, block_lse, first=False, final_out=final_out)


@register_fake("xdit_amd::lse_merge_final")
def _lse_merge_final_fake(acc_out, acc_lse, block_out, block_lse, final_out):
    return None


@custom_op("xdit_amd::fp8_quant", mutates_args=(), device_types="cuda")
def fp8_quant(x: Tensor, per_tensor: bool, hadamard_block: int) -> Tuple[Tensor, Tensor]:
    return ops.fp8_quant(x, per_tensor=per_tensor, hadamard_block=hadamard_block)


@register_fake("xdit_amd::fp8_quant")
def _fp8_quant_fake(x, per_tensor, hadamard_block):
    B, H, S, D = x.shape
    return (x.new_empty((B, H, S, D), dtype=torch.float8_e4m3fn),
            x.new_empty((B, H), dtype=torch.float32))


@custom_op("xdit_amd::fp8_quant_ex", mutates_args=(), device_types="cuda")
def fp8_quant_ex(x: Tensor, x2: Optional[Tensor], scale: Optional[Tensor], per_tensor: bool,
                 hadamard_block: int) -> Tuple[Tensor, Tensor, Tensor]:
    """`ops.fp8_quant` with its optional second tensor (quantised with the scales of the first) and
    its optional static scale (a one-element fp32 tensor).  Without `x2` the second result has no rows."""
    out = ops.fp8_quant(x, per_tensor=per_tensor, scale=scale, hadamard_block=hadamard_block, x2=x2)
    if x2 is None:
        B, H, _, D = x.shape
        return out[0], x.new_empty((B, H, 0, D), dtype=torch.float8_e4m3fn), out[1]
    return out


@register_fake("xdit_amd::fp8_quant_ex")
def _fp8_quant_ex_fake(x, x2, scale, per_tensor, hadamard_block):
    B, H, S, D = x.shape
    S2 = 0 if x2 is None else x2.shape[2]
    return (x.new_empty((B, H, S, D), dtype=torch.float8_e4m3fn),
            x.new_empty((B, H, S2, D), dtype=torch.float8_e4m3fn),
            x.new_empty((B, H), dtype=torch.float32))


@custom_op("xdit_amd::norm_rope", mutates_args=(), device_types="cuda")
def norm_rope(x: Tensor, weight: Tensor, cos: Tensor, sin: Tensor, eps: float, norm: str, rope: str,
              rope_row0: int, rope_rows: int) -> Tensor:
    """Fused RMSNorm + rotary embedding + re-layout of a logical BHSD tensor (`ops.qk_prologue`).
    `norm` is "none", "head" or "token" (`weight` is ignored for "none": pass any tensor);
    `rope` is "none", "interleaved", "split_half" or "wan" (`cos`/`sin` ignored for "none")."""
    return ops.qk_prologue(x, weight=None if norm == "none" else weight, eps=eps, norm=None if norm == "none" else norm,
                           rotary_emb=None if rope == "none" else (cos, sin), rope="interleaved" if rope == "none" else rope,
                           rope_row0=rope_row0, rope_rows=rope_rows if rope != "none" else None)


@register_fake("xdit_amd::norm_rope")
def _norm_rope_fake(x, weight, cos, sin, eps, norm, rope, rope_row0, rope_rows):
    return x.new_empty(tuple(x.shape))


# ---------------------------------------------------------------------------- around the attention call
def _or_none(kind: str):
    return None if kind == "none" else kind


def _rows16(t):
    """A tensor as the kernels take it: autograd may pass a gradient that was expanded from a scalar, or a part of a larger
    one that starts anywhere (a copy: `contiguous` would return the part itself)."""
    if t is None or (t.data_ptr() % 16 == 0 and (t.is_contiguous() or (t.stride(-1) == 1 and all(s * t.element_size() % 16 == 0 for s in t.stride()[:-1])))):
        return t
    return t.clone(memory_format=torch.contiguous_format)


@custom_op("xdit_amd::gated_norm", mutates_args=(), device_types="cuda")
def gated_norm(x: Tensor, y: Optional[Tensor], gate: Optional[Tensor], scale: Optional[Tensor], shift: Optional[Tensor],
               weight: Optional[Tensor], bias: Optional[Tensor], y_weight: Optional[Tensor], norm: str, eps: float, y_norm: str,
               y_eps: float, residual_scale: float) -> Tuple[Tensor, Tensor, Tensor]:
    """`block_ops.gated_norm` with its statistics; `norm` and `y_norm` are "none", "rms" or "layer".  Without `y` the first
    result has no rows (it would be x itself), with norm "none" the second has none."""
    h, n, stats = block_ops.gated_norm(x, y, gate, scale, shift, weight, bias, _or_none(norm), eps, _or_none(y_norm), y_weight, y_eps,
                                       residual_scale, return_stats=True)
    B, S, C = x.shape
    return x.new_empty((B, 0, C)) if y is None else h, x.new_empty((B, 0, C)) if n is None else n, stats


@register_fake("xdit_amd::gated_norm")
def _gated_norm_fake(x, y, gate, scale, shift, weight, bias, y_weight, norm, eps, y_norm, y_eps, residual_scale):
    B, S, C = x.shape
    return (x.new_empty((B, 0 if y is None else S, C)), x.new_empty((B, 0 if norm == "none" else S, C)),
            x.new_empty((B, S, 4), dtype=torch.float32))


@custom_op("xdit_amd::gated_norm_fp8", mutates_args=(), device_types="cuda")
def gated_norm_fp8(x: Tensor, y: Optional[Tensor], gate: Optional[Tensor], scale: Optional[Tensor], shift: Optional[Tensor],
                   weight: Optional[Tensor], bias: Optional[Tensor], y_weight: Optional[Tensor], norm: str, eps: float, y_norm: str,
                   y_eps: float, residual_scale: float) -> Tuple[Tensor, Tensor, Tensor]:
    """The same with n as fp8 values and scales, and no gradient."""
    h, (n, n_scale) = block_ops.gated_norm(x, y, gate, scale, shift, weight, bias, norm, eps, _or_none(y_norm), y_weight, y_eps,
                                           residual_scale, fp8=True)
    return x.new_empty((x.shape[0], 0, x.shape[2])) if y is None else h, n, n_scale


@register_fake("xdit_amd::gated_norm_fp8")
def _gated_norm_fp8_fake(x, y, gate, scale, shift, weight, bias, y_weight, norm, eps, y_norm, y_eps, residual_scale):
    B, S, C = x.shape
    return (x.new_empty((B, 0 if y is None else S, C)), x.new_empty((B, S, C), dtype=torch.float8_e4m3fn),
            x.new_empty(((C + 127) // 128, B, S), dtype=torch.float32).permute(1, 2, 0))


_NORM_GRADS = ("dx", "dy", "dgate", "dscale", "dshift", "dweight", "dbias", "dy_weight")


def _norm_grad_shapes(dn, h, y, gate, scale, shift, weight, bias, y_weight):
    """The operand whose shape and dtype each gradient has, None where there is none (as `block_ops.gated_norm_backward`)."""
    def seen(t):
        return t if dn is not None else None
    return (h, y, gate, seen(scale), seen(shift), seen(weight), seen(bias), y_weight)


@custom_op("xdit_amd::gated_norm_backward", mutates_args=(), device_types="cuda")
def gated_norm_backward(dh: Optional[Tensor], dn: Optional[Tensor], h: Tensor, stats: Tensor, y: Optional[Tensor], gate: Optional[Tensor],
                        scale: Optional[Tensor], shift: Optional[Tensor], weight: Optional[Tensor], bias: Optional[Tensor],
                        y_weight: Optional[Tensor], norm: str, y_norm: str, residual_scale: float) -> List[Tensor]:
    """`block_ops.gated_norm_backward`: those of dx, dy, dgate, dscale, dshift, dweight, dbias and dy_weight that there are."""
    r = block_ops.gated_norm_backward(_rows16(dh), _rows16(dn), h, stats, y, gate, scale, shift, weight, bias, _or_none(norm),
                                      _or_none(y_norm), y_weight, residual_scale)
    return [r[name] for name in _NORM_GRADS if name in r]


@register_fake("xdit_amd::gated_norm_backward")
def _gated_norm_backward_fake(dh, dn, h, stats, y, gate, scale, shift, weight, bias, y_weight, norm, y_norm, residual_scale):
    return [t.new_empty(t.shape) for t in _norm_grad_shapes(dn, h, y, gate, scale, shift, weight, bias, y_weight) if t is not None]


def _gated_norm_setup(ctx, inputs, output):
    x, y, gate, scale, shift, weight, bias, y_weight, norm, _, y_norm, _, residual_scale = inputs
    h, _, stats = output
    ctx.save_for_backward(x if y is None else h, stats, y, gate, scale, shift, weight, bias, y_weight)
    ctx.kinds = (norm, y_norm, residual_scale)


def _gated_norm_grad(ctx, dh, dn, dstats):
    h, stats, y, gate, scale, shift, weight, bias, y_weight = ctx.saved_tensors
    norm, y_norm, residual_scale = ctx.kinds
    dh = None if y is None else dh
    dn = None if norm == "none" else dn
    if dh is None and dn is None:
        return (None,) * 13
    out = iter(torch.ops.xdit_amd.gated_norm_backward(dh, dn, h, stats, y, gate, scale, shift, weight, bias, y_weight, norm, y_norm, residual_scale))
    of = _norm_grad_shapes(dn, h, y, gate, scale, shift, weight, bias, y_weight)
    return (*(None if t is None else next(out) for t in of), None, None, None, None, None)


register_autograd("xdit_amd::gated_norm", _gated_norm_grad, setup_context=_gated_norm_setup)


@custom_op("xdit_amd::axes_rope", mutates_args=(), device_types="cuda")
def axes_rope(q: Tensor, k: Optional[Tensor], positions: Tensor, inv_freq: Tensor, pairs: List[int], norm: bool, q_weight: Optional[Tensor],
              k_weight: Optional[Tensor], eps: float, rope: str) -> Tuple[Tensor, Tensor]:
    """`block_ops.axes_rope`; without `k` the second result has no heads."""
    oq, ok = block_ops.axes_rope(q, k, positions, inv_freq, pairs, norm, q_weight, k_weight, eps, rope)
    return oq, q.new_empty((q.shape[0], 0, *q.shape[2:])) if k is None else ok


@register_fake("xdit_amd::axes_rope")
def _axes_rope_fake(q, k, positions, inv_freq, pairs, norm, q_weight, k_weight, eps, rope):
    return q.new_empty(q.shape), q.new_empty((q.shape[0], 0 if k is None else k.shape[1], *q.shape[2:]))


@custom_op("xdit_amd::axes_rope_backward", mutates_args=(), device_types="cuda")
def axes_rope_backward(dq: Tensor, dk: Optional[Tensor], positions: Tensor, inv_freq: Tensor, pairs: List[int], q: Optional[Tensor],
                       k: Optional[Tensor], norm: bool, q_weight: Optional[Tensor], k_weight: Optional[Tensor], eps: float,
                       rope: str) -> List[Tensor]:
    """`block_ops.axes_rope_backward`: those of dq, dk, dq_weight and dk_weight that there are."""
    r = block_ops.axes_rope_backward(_rows16(dq), _rows16(dk), positions, inv_freq, pairs, q, k, norm, q_weight, k_weight, eps, rope)
    return [t for t in r if t is not None]


@register_fake("xdit_amd::axes_rope_backward")
def _axes_rope_backward_fake(dq, dk, positions, inv_freq, pairs, q, k, norm, q_weight, k_weight, eps, rope):
    return [t.new_empty(t.shape) for t in (dq, dk, q_weight, k_weight) if t is not None]


def _axes_rope_setup(ctx, inputs, output):
    q, k, positions, inv_freq, pairs, norm, q_weight, k_weight, eps, rope = inputs
    ctx.save_for_backward(*((q, k) if norm else (None, None)), positions, inv_freq, q_weight, k_weight)
    ctx.kinds = (list(pairs), norm, eps, rope, k is not None)


def _axes_rope_grad(ctx, dq, dk):
    q, k, positions, inv_freq, q_weight, k_weight = ctx.saved_tensors
    pairs, norm, eps, rope, has_k = ctx.kinds
    dk = dk if has_k else None
    out = iter(torch.ops.xdit_amd.axes_rope_backward(dq, dk, positions, inv_freq, pairs, q, k, norm, q_weight, k_weight, eps, rope))
    gq, gk, gqw, gkw = (None if t is None else next(out) for t in (dq, dk, q_weight, k_weight))
    return gq, gk, None, None, None, None, gqw, gkw, None, None


register_autograd("xdit_amd::axes_rope", _axes_rope_grad, setup_context=_axes_rope_setup)


@custom_op("xdit_amd::fp8_block_quant", mutates_args=(), device_types="cuda")
def fp8_block_quant(x: Tensor, block_rows: int) -> Tuple[Tensor, Tensor]:
    return block_ops.fp8_block_quant(x, block_rows)


@register_fake("xdit_amd::fp8_block_quant")
def _fp8_block_quant_fake(x, block_rows):
    y = x.new_empty(x.shape, dtype=torch.float8_e4m3fn)
    M, kb = x.shape[-2], (x.shape[-1] + 127) // 128
    if block_rows != 1:
        return y, x.new_empty(((M + 127) // 128, kb), dtype=torch.float32)
    if x.ndim == 3:
        return y, x.new_empty((kb, x.shape[0], M), dtype=torch.float32).permute(1, 2, 0)
    return y, x.new_empty((kb, M), dtype=torch.float32).t()


@custom_op("xdit_amd::fp8_block_matmul", mutates_args=(), device_types="cuda")
def fp8_block_matmul(x: Tensor, x_scale: Tensor, w: Tensor, w_scale: Tensor, bias: Optional[Tensor], out_dtype: torch.dtype,
                     exact_sums: Optional[bool]) -> Tensor:
    return block_ops.fp8_block_matmul(x, x_scale, w, w_scale, bias, out_dtype, exact_sums=exact_sums)


@register_fake("xdit_amd::fp8_block_matmul")
def _fp8_block_matmul_fake(x, x_scale, w, w_scale, bias, out_dtype, exact_sums):
    return x.new_empty((*x.shape[:-1], w.shape[0]), dtype=out_dtype)


@custom_op("xdit_amd::fp8_linear", mutates_args=(), device_types="cuda")
def fp8_linear(x: Tensor, w: Tensor, w_scale: Tensor, w_t: Optional[Tensor], w_t_scale: Optional[Tensor], bias: Optional[Tensor]) -> Tensor:
    """x w^T + bias of a 16- or 32-bit x, quantised here, and a frozen block-scaled weight; the gradient to x is the
    same product of dy with the transposed weight (w_t, w_t_scale)."""
    x8, xs = block_ops.fp8_block_quant(_rows16(x))
    return block_ops.fp8_block_matmul(x8, xs, w, w_scale, bias, x.dtype)


@register_fake("xdit_amd::fp8_linear")
def _fp8_linear_fake(x, w, w_scale, w_t, w_t_scale, bias):
    return x.new_empty((*x.shape[:-1], w.shape[0]))


def _fp8_linear_setup(ctx, inputs, output):
    ctx.save_for_backward(inputs[3], inputs[4])


def _fp8_linear_grad(ctx, dy):
    w_t, w_t_scale = ctx.saved_tensors
    if w_t is None:
        raise RuntimeError("the gradient of an fp8 projection needs its transposed weight")
    return torch.ops.xdit_amd.fp8_linear(dy, w_t, w_t_scale, None, None, None), None, None, None, None, None


register_autograd("xdit_amd::fp8_linear", _fp8_linear_grad, setup_context=_fp8_linear_setup)
