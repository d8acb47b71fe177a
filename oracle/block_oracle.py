"""Float64 restatement of the operators around the attention call of a DiT block, from their formulas.

Every function takes tensors of any floating dtype and returns float64 results (unrounded: what a kernel
rounds once at its end), together with the magnitudes that its rounding errors scale with where a test needs them.
"""
import torch


def _d(t):
    return None if t is None else t.double()


def _tokens(m):
    """(B, C) modulation -> (B, 1, C)."""
    return None if m is None else (m.double()[:, None] if m.ndim == 2 else m.double())


def row_norm(x, kind, eps):
    """-> normed x, mean (zero for "rms"), 1 / deviation, over the last dimension."""
    mean = x.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(x[..., :1])
    r = 1.0 / torch.sqrt((x - mean).pow(2).mean(-1, keepdim=True) + eps)
    return (x - mean) * r, mean, r


def gated_norm(x, y=None, gate=None, scale=None, shift=None, weight=None, bias=None, norm="layer", eps=1e-6, y_norm=None,
               y_weight=None, y_eps=1e-6, residual_scale=1.0):
    """-> h, n, stats (B,S,4), and a row-wise size of the terms n is made of."""
    x, y = _d(x), _d(y)
    ym, yr = torch.zeros_like(x[..., :1]), torch.ones_like(x[..., :1])
    h, terms = x, x.abs()
    if y is not None:
        v = y
        if y_norm is not None:
            v, ym, yr = row_norm(y, y_norm, y_eps)
        if y_weight is not None:
            v = v * _d(y_weight)
        if gate is not None:
            v = v * _tokens(gate)
        h = x + residual_scale * v
        terms = terms + abs(residual_scale) * v.abs()
    if norm is None:
        return h, None, torch.cat([torch.zeros_like(ym), torch.ones_like(yr), ym, yr], -1), terms
    n, m, r = row_norm(h, norm, eps)
    size = terms.amax(-1, keepdim=True) * r
    if weight is not None:
        n, size = n * _d(weight), size * _d(weight).abs()
    if bias is not None:
        n, size = n + _d(bias), size + _d(bias).abs()
    if scale is not None:
        n, size = n * (1 + _tokens(scale)), size * (1 + _tokens(scale).abs())
    if shift is not None:
        n, size = n + _tokens(shift), size + _tokens(shift).abs()
    return h, n, torch.cat([m, r, ym, yr], -1), size


def gated_norm_backward(dh, dn, h, stats, y=None, gate=None, scale=None, shift=None, weight=None, bias=None, norm="layer", y_norm=None,
                        y_weight=None, residual_scale=1.0):
    """-> gradients, and for each the size of the terms it is the sum of."""
    h = _d(h)
    B, S, C = h.shape
    m, r, ym, yr = stats.double().split(1, -1)
    t = torch.zeros_like(h) if dh is None else _d(dh)
    size = t.abs()
    g, big = {}, {}

    def put(name, like, terms, elementwise):
        """Sums `terms` over the rows that share an entry of `like`."""
        if like is None:
            return
        if elementwise:
            g[name], big[name] = terms, terms.abs()
            return
        dims = (0, 1) if like.ndim == 1 else (1,)
        g[name], big[name] = terms.sum(dims).view(like.shape), terms.abs().sum(dims).view(like.shape)

    def per_token(m):
        return m is not None and m.ndim == 3 and m.shape[1] == S and S > 1

    if dn is not None:
        dn = _d(dn)
        u = (h - m) * r
        us = (h.abs() + m.abs()) * r
        w = 1.0 if weight is None else _d(weight)
        b = 0.0 if bias is None else _d(bias)
        one = 1.0 if scale is None else 1 + _tokens(scale)
        put("dshift", shift, dn, per_token(shift))
        put("dscale", scale, dn * (u * w + b), per_token(scale))
        if scale is not None:   # the sum is formed as w * sum(dn u) + b * sum(dn)
            s2 = dn.abs() * (us * abs(w) + abs(b))
            big["dscale"] = s2 if per_token(scale) else s2.sum(1).view(scale.shape)
        put("dweight", weight, dn * one * u, False)
        if weight is not None:
            big["dweight"] = (dn * one * us).abs().sum((0, 1))
        put("dbias", bias, dn * one + torch.zeros_like(h), False)
        du = dn * one * w
        dot = (du * u).mean(-1, keepdim=True)
        flat = du.mean(-1, keepdim=True) if norm == "layer" else 0.0
        t = t + r * (du - flat - u * dot)
        size = size + r * (du.abs() + du.abs().mean(-1, keepdim=True) + us * (du.abs() * us).mean(-1, keepdim=True))
    g["dx"], big["dx"] = t, size
    if y is not None:
        z = (_d(y) - ym) * yr
        zs = (_d(y).abs() + ym.abs()) * yr
        yw = 1.0 if y_weight is None else _d(y_weight)
        ga = 1.0 if gate is None else _tokens(gate)
        put("dgate", gate, residual_scale * t * z * yw, per_token(gate))
        if gate is not None:
            s2 = (residual_scale * size * zs * yw).abs()
            big["dgate"] = s2 if per_token(gate) else s2.sum(1).view(gate.shape)
        e = residual_scale * ga * t
        put("dy_weight", y_weight, e * z, False)
        if y_weight is not None:
            big["dy_weight"] = (residual_scale * ga * size * zs).abs().sum((0, 1))
        e = e * yw
        es = (residual_scale * ga * yw * size).abs() if isinstance(ga, torch.Tensor) or isinstance(yw, torch.Tensor) else abs(residual_scale) * size
        if y_norm is not None:
            dot = (e * z).mean(-1, keepdim=True)
            flat = e.mean(-1, keepdim=True) if y_norm == "layer" else 0.0
            e = yr * (e - flat - z * dot)
            es = yr * (es + es.mean(-1, keepdim=True) + zs * (es * zs).mean(-1, keepdim=True))
        g["dy"], big["dy"] = e, es
    return g, big


def block_scales(x, rows):
    """Exact scale of every rows x 128 block of (M, K)."""
    M, K = x.shape
    mb, kb = -(-M // rows), -(-K // 128)
    p = torch.zeros(mb * rows, kb * 128, dtype=torch.float64, device=x.device)
    p[:M, :K] = x.double().abs()
    top = p.view(mb, rows, kb, 128).amax((1, 3))
    return torch.where(top > 0, (top / 448.0).clamp(min=2.0 ** -126), torch.ones_like(top))


def spread(scale, rows, M, K):
    """Block scales -> one per element of (M, K)."""
    return scale.repeat_interleave(rows, 0)[:M].repeat_interleave(128, 1)[:, :K]


def turn(x, positions, inv_freq, pairs, rope, sign=1):
    """Every pair of (B,H,S,D) columns as a complex number times exp(i sign phi)."""
    B, H, S, D = x.shape
    axis = torch.tensor([a for a, n in enumerate(pairs) for _ in range(n)], dtype=torch.long, device=x.device)
    phi = sign * positions.double()[..., axis] * inv_freq.double()            # ([B,] S, P)
    phi = phi[:, None] if phi.ndim == 3 else phi
    P = axis.numel()
    a, b = (x[..., 0:2 * P:2], x[..., 1:2 * P:2]) if rope == "interleaved" else (x[..., :P], x[..., P:2 * P])
    z = torch.complex(a.contiguous(), b.contiguous()) * torch.complex(torch.cos(phi), torch.sin(phi))
    y = x.clone()
    if rope == "interleaved":
        y[..., 0:2 * P:2], y[..., 1:2 * P:2] = z.real, z.imag
    else:
        y[..., :P], y[..., P:2 * P] = z.real, z.imag
    return y


def axes_rope(x, weight, positions, inv_freq, pairs, norm, eps, rope):
    x = _d(x)
    if norm:
        x = row_norm(x, "rms", eps)[0]
        x = x if weight is None else x * _d(weight)
    return turn(x, positions, inv_freq, pairs, rope)


def axes_rope_backward(dy, x, weight, positions, inv_freq, pairs, norm, eps, rope):
    """-> dx, dweight, and the sizes of the terms of both."""
    d = turn(_d(dy), positions, inv_freq, pairs, rope, -1)
    size = _d(dy).abs().amax(-1, keepdim=True) * 1.5
    if not norm:
        return d, None, size, None
    u, _, r = row_norm(_d(x), "rms", eps)
    w = 1.0 if weight is None else _d(weight)
    g = d * w
    dx = r * (g - u * (g * u).mean(-1, keepdim=True))
    top = size * (1.0 if weight is None else w.abs())
    return dx, (d * u).sum((0, 1, 2)), r * (top + u.abs() * (top * u.abs()).mean(-1, keepdim=True)), (size * u.abs()).sum((0, 1, 2))


def block_matmul(x, x_scale, w, w_scale, bias=None):
    """-> (M, N) product of the values the operands stand for, and the sum of its terms' sizes."""
    M, K = x.shape
    N = w.shape[0]
    a = x.double() * spread(x_scale.double(), 1, M, K)
    b = w.double() * spread(w_scale.double(), 128, N, K)
    y, size = a @ b.t(), a.abs() @ b.t().abs()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y, size


def largest_of_eights(x, x_scale, w, w_scale):
    """Sum over the groups of eight consecutive k of the largest |x w| of the group."""
    a = x.float() * spread(x_scale.float(), 1, *x.shape)
    b = w.float() * spread(w_scale.float(), 128, *w.shape)
    total = torch.zeros(x.shape[0], w.shape[0], device=x.device)
    for k in range(0, x.shape[1], 8):
        top = torch.zeros_like(total)
        for j in range(k, k + 8):
            top = torch.maximum(top, torch.outer(a[:, j].abs(), b[:, j].abs()))
        total += top
    return total.double()
