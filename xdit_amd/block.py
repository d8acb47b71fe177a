"""Module-level forms of the operators around the attention call of a DiT block, differentiable and traceable.

The functions take what `xdit_amd.block_ops` takes.  Where a gradient is wanted, or under `torch.compile`, they go through the
registered ops of `xdit_amd.custom_ops`; otherwise straight to the kernels.  Gradients are those of reverse mode: tangents of
forward-mode differentiation are refused.
"""
import torch
from torch.autograd import forward_ad

from . import block_ops
from . import custom_ops  # registers torch.ops.xdit_amd.*

rope_frequencies = block_ops.rope_frequencies


def _registered(*tensors):
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("forward-mode differentiation is not supported: the tangent would be lost")
    return torch.compiler.is_compiling() or (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors))


def _with_batch(t, B):
    """A modulation tensor with a row per batch entry, what its gradient has; autograd adds them up again."""
    return t if t is None or t.shape[0] == B else t.expand(B, *t.shape[1:])


def gated_norm(x, y=None, gate=None, scale=None, shift=None, weight=None, bias=None, norm="layer", eps=1e-6, y_norm=None, y_weight=None,
               y_eps=1e-6, residual_scale=1.0, fp8=False):
    """`block_ops.gated_norm` -> (h, n), differentiable in every tensor.  `fp8` gives n as the (values, scales) pair that
    `Fp8Linear` takes; it has no gradient and is refused where one is wanted."""
    given = (x, y, gate, scale, shift, weight, bias, y_weight)
    if not _registered(*given):
        return block_ops.gated_norm(x, y, gate, scale, shift, weight, bias, norm, eps, y_norm, y_weight, y_eps, residual_scale, fp8)
    if fp8 and torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in given):
        raise ValueError("an fp8 result has no gradient: take n in 16 or 32 bits, Fp8Linear quantises it")
    if fp8 and norm is None:
        raise ValueError("fp8, scale, shift, weight and bias need a norm")
    gate, scale, shift = (_with_batch(t, x.shape[0]) for t in (gate, scale, shift))
    if scale is not None and shift is not None and scale.ndim != shift.ndim:   # (B, C) beside (B, 1 or S, C)
        scale, shift = (t.unsqueeze(1) if t.ndim == 2 else t for t in (scale, shift))
    if scale is not None and shift is not None and scale.shape != shift.shape:   # one of them has a row per token: so has the other's gradient then
        scale, shift = (t.expand(x.shape) for t in (scale, shift))
    op = torch.ops.xdit_amd.gated_norm_fp8 if fp8 else torch.ops.xdit_amd.gated_norm
    h, n, last = op(x, y, gate, scale, shift, weight, bias, y_weight, norm or "none", eps, y_norm or "none", y_eps, residual_scale)
    return x if y is None else h, (n, last) if fp8 else (None if norm is None else n)


def axes_rope(q, k, positions, inv_freq, pairs, norm=False, q_weight=None, k_weight=None, eps=1e-6, rope="interleaved"):
    """`block_ops.axes_rope` -> (q, k), differentiable in q, k and the gains; positions and frequencies that want a gradient are refused."""
    registered = _registered(q, k, positions, inv_freq, q_weight, k_weight)
    if (positions.requires_grad or inv_freq.requires_grad) and torch.is_grad_enabled():
        raise ValueError("positions and inv_freq have no gradient here: detach them")
    if not registered:
        return block_ops.axes_rope(q, k, positions, inv_freq, pairs, norm, q_weight, k_weight, eps, rope)
    oq, ok = torch.ops.xdit_amd.axes_rope(q, k, positions, inv_freq, list(pairs), norm, q_weight, k_weight, eps, rope)
    return oq, None if k is None else ok


class Fp8Linear(torch.nn.Module):
    """A projection with a frozen weight in fp8 and a scale per 128 x 128 block.

    forward(x): x (M, K) or (B, S, K) in 16 or 32 bits (copied first where its rows are not 16-byte aligned and dense), or the (values, scales) pair of `fp8_block_quant` or of `gated_norm(fp8=True)`
    -> x w^T + bias in x's dtype (for a pair in that of the weight it was made from).  `backward=True` also lays out the transposed
    weight, whose blocks keep their bytes, for the gradient to x; in_features has to be a multiple of 16, out_features too then."""

    def __init__(self, weight, bias=None, backward=False):
        super().__init__()
        if weight.ndim != 2:
            raise ValueError("weight must be (out_features, in_features)")
        self.out_features, self.in_features = weight.shape
        if self.in_features % 16 or (backward and self.out_features % 16):
            raise ValueError("in_features (for the gradient out_features too) must be a multiple of 16")
        self.dtype = weight.dtype
        w, scale = block_ops.fp8_block_quant(custom_ops._rows16(weight.detach()), 128)
        self.register_buffer("weight", w)
        self.register_buffer("weight_scale", scale)
        self.register_buffer("weight_t", w.t().contiguous() if backward else None)
        self.register_buffer("weight_t_scale", scale.t().contiguous() if backward else None)
        self.register_buffer("bias", None if bias is None else bias.detach().to(torch.float32, copy=True).contiguous())   # its own, and any result's dtype takes it

    @classmethod
    def from_linear(cls, linear, backward=False):
        return cls(linear.weight, linear.bias, backward)

    def _apply(self, fn, recurse=True):
        # moves between devices, and keeps the types: .to(dtype) of a model is not meant for fp8 bytes and their scales
        for name, b in self._buffers.items():
            if b is not None:
                moved = fn(b)
                self._buffers[name] = moved if moved.dtype == b.dtype else b.to(moved.device)
        return self

    def forward(self, x):
        if isinstance(x, tuple):
            x8, scale = x
            if torch.compiler.is_compiling():
                return torch.ops.xdit_amd.fp8_block_matmul(x8, scale, self.weight, self.weight_scale, self.bias, self.dtype, None)
            return block_ops.fp8_block_matmul(x8, scale, self.weight, self.weight_scale, self.bias, self.dtype)
        if _registered(x):
            return torch.ops.xdit_amd.fp8_linear(x, self.weight, self.weight_scale, self.weight_t, self.weight_t_scale, self.bias)
        x8, scale = block_ops.fp8_block_quant(custom_ops._rows16(x))
        return block_ops.fp8_block_matmul(x8, scale, self.weight, self.weight_scale, self.bias, x.dtype)
