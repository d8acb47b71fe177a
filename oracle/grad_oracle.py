"""Float64 restatement of what a training step adds: attention's backward pass, norm and clipping of gradients.

Every function takes tensors of any floating dtype and returns float64 results; `attn_bwd` also the sizes that a kernel's rounding errors
scale with.
"""
import math

import torch

GAMMA = 2.0 ** -17


def attn_fwd(q, k, v, scale):
    """-> out, lse of softmax(scale q k^T) v."""
    s = scale * (q.double() @ k.double().transpose(-1, -2))
    lse = torch.logsumexp(s, -1)
    return torch.exp(s - lse.unsqueeze(-1)) @ v.double(), lse


def attn_bwd(dout, q, k, v, out, lse, scale, dlse=None, half_step=0.0):
    """-> (dq, dk, dv), and for each how far a kernel's result may lie from it, element by element: P and dS rounded by
    `half_step` relative to their size, the result by as much, and every fp32 sum by GAMMA of the sizes it adds.

    GAMMA: sums of up to 128 products are off by at most 128 * 2^-24 = 2^-17 of the sum of their sizes; those of n rows of either sign by about
    sqrt(n) 2^-24 of theirs, 2^-17 at 16384 rows.  An exponent is off by GAMMA of the sizes that it adds, plus two roundings of its own."""
    dout, q, k, v, out, lse = (t.double() for t in (dout, q, k, v, out, lse))
    tr = lambda t: t.transpose(-1, -2)  # noqa: E731
    none = (lse == -math.inf).unsqueeze(-1)
    p = torch.where(none, torch.zeros((), dtype=torch.float64, device=q.device), torch.exp(scale * (q @ tr(k)) - lse.unsqueeze(-1)))
    delta = (dout * out).sum(-1) - (0 if dlse is None else dlse.double())
    ds = p * (dout @ tr(v) - delta.unsqueeze(-1))
    dq, dk, dv = scale * (ds @ k), scale * (tr(ds) @ q), tr(p) @ dout
    a = GAMMA * (1 + scale * (q.abs() @ tr(k.abs())) + torch.where(none, 0.0, lse.abs().unsqueeze(-1)))   # relative error of P
    size = dout.abs() @ tr(v.abs()) + (dout * out).abs().sum(-1, keepdim=True) + (0 if dlse is None else dlse.double().abs().unsqueeze(-1))
    e_ds = (half_step + a + GAMMA) * ds.abs() + GAMMA * p * size
    e_p = (half_step + a + GAMMA) * p
    far = (scale * (e_ds @ k.abs()), scale * (tr(e_ds) @ q.abs()), tr(e_p) @ dout.abs())
    return (dq, dk, dv), tuple(f + (half_step + 2.0 ** -22) * g.abs() for f, g in zip(far, (dq, dk, dv)))


def grad_norm(grads, kind=2.0):
    parts = [t.double().abs().flatten() for t in grads]
    flat = torch.cat(parts) if parts else torch.zeros(1, dtype=torch.float64)
    if flat.numel() == 0:
        return 0.0
    if kind == math.inf:
        return float(flat.max())
    return float(flat.sum()) if kind == 1 else math.sqrt(float(flat.square().sum()))


def clip(grads, norm, max_norm):
    factor = max_norm / (norm + 1e-6)
    factor = min(1.0, factor) if factor == factor else factor
    return [t.double() * factor for t in grads]
