"""What the operators around the attention call of a DiT block are timed on: the norm with its
modulation, gate and residual, the rotation by positions on several axes, the block-wise fp8
quantiser and the block-scaled fp8 product that the projections run on.

A case is a dict of plain values; `op` says which entry point it goes through:

  norm        block_ops.gated_norm: residual stream + gated block output, then the modulated norm of
              the next block; `fp8`: the norm leaves as e4m3 with a scale per 1 x 128 block
  norm_bwd    block_ops.gated_norm_backward from the saved stream, statistics and block output
  rope        block_ops.axes_rope on q and k: RMSNorm over head_dim (`qk_norm`) and rotation
  rope_bwd    block_ops.axes_rope_backward
  quant       block_ops.fp8_block_quant with blocks of 1 x 128 (`rows` 1) or 128 x 128 (`rows` 128)
  product     block_ops.fp8_block_matmul

`run` computes them in 32 bits by elementary torch operations where `own` is false, and calls the
package's entry points where it is true.  Sizes are those of the shapes that the benchmark and the
tests of this repository use (hidden sizes of 16 x 72, 24 x 64, 30 x 64 and 40 x 128, image models at
512 and 1024 pixels, video at 480p) and, in `draw`, the ranges between and around them.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_BLOCK = 128
_F8_MAX = 448.0


def _norm(op, B, S, C, dtype="bf16", mods="fp32", per_token=False, y=True, norm="layer", y_norm="none", affine=False, fp8=False, name=None):
    c = {"op": op, "B": B, "S": S, "C": C, "dtype": dtype, "mods": mods, "per_token": per_token, "y": y, "norm": norm,
         "y_norm": y_norm, "affine": affine, "fp8": fp8}
    return c if name is None else dict(c, name=name)


def _rope(op, B, S, H, Hk, D, axes, dtype="bf16", qk_norm=True, pairing="interleaved", layout="bshd", text=0, name=None):
    c = {"op": op, "B": B, "S": S, "H": H, "Hk": Hk, "D": D, "axis_t": axes[0], "axis_h": axes[1], "axis_w": axes[2], "dtype": dtype,
         "qk_norm": qk_norm, "pairing": pairing, "layout": layout, "text": text}
    return c if name is None else dict(c, name=name)


def _quant(M, K, dtype="bf16", rows=1, name=None):
    c = {"op": "quant", "M": M, "K": K, "dtype": dtype, "rows": rows}
    return c if name is None else dict(c, name=name)


def _product(M, N, K, out="bf16", bias=True, name=None):
    c = {"op": "product", "M": M, "N": N, "K": K, "out": out, "bias": bias}
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # text stream of a 1024-pixel DiT under classifier-free guidance, 120 tokens: the smallest call, latency
        _norm("norm", 2, 120, 1152, mods="same", name="norm_text120"),
        # 480p video: gated residual, layer norm and modulation (fp32 vectors), e4m3 blocks for the next projection
        _norm("norm", 1, 32760, 5120, fp8=True, name="norm_video480p_fp8"),
        # gradients of a sandwich block (RMS norms with gains before and after), image + text under guidance
        _norm("norm_bwd", 2, 4250, 1536, dtype="fp16", norm="rms", y_norm="rms", affine=True, name="norm_image_backward"),
        # a Ulysses-8 rank's 3 heads of a 512-pixel MMDiT block: 512 text tokens at position 0, a 32 x 32 image grid
        _rope("rope", 1, 1536, 3, 3, 128, (16, 56, 56), text=512, name="rope_image512_3heads"),
        # 480p video, all heads: time, height and width axes
        _rope("rope", 1, 32760, 40, 40, 128, (44, 42, 42), name="rope_video480p"),
        # gradients of a head_dim-64 image model under guidance, BHSD memory, half-split pairs
        _rope("rope_bwd", 2, 4250, 24, 24, 64, (16, 24, 24), dtype="fp16", pairing="split_half", layout="bhsd", text=154, name="rope_image_backward"),
        # activations of a 1024-pixel image + text sequence, ragged last block
        _quant(4250, 1480, name="quant_image_rows"),
        # the weight of a video block's feed-forward, laid out once
        _quant(13824, 5120, rows=128, name="quant_weight"),
        # the timestep embedding to six modulation vectors: one token, weight bandwidth
        _product(1, 30720, 5120, out="fp32", name="product_one_token"),
        # text tokens, 226 of them, odd width
        _product(226, 1925, 1920, out="fp16", name="product_text226"),
        # attention output projection of a 1024-pixel image + text sequence
        _product(4250, 5120, 5120, name="product_image1024"),
        # first product of a 480p video block's feed-forward: the largest
        _product(32760, 13824, 5120, name="product_video480p"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HIDDEN = (640, 1152, 1280, 1536, 1920, 2560, 5120, 7680, 10240, 13824)
_TOKENS = (1, 2, 16, 120, 226, 512, 1024, 4096, 4250, 4608, 9450, 17776, 32760)


def _size(rng, known, unit, lo, hi):
    """One of the known sizes within the range, or an odd number of units."""
    fit = [n for n in known if lo <= n <= hi]
    if fit and rng.random() < 0.4:
        return rng.choice(fit)
    return unit * (2 * _log_int(rng, max(0.5, lo / unit / 2), max(0.5, (hi / unit - 1) / 2)) + 1) if hi > 2 * unit else unit


def _width(rng, unit, lo, hi):
    return _size(rng, _HIDDEN, unit, lo, hi)


def _tokens(rng, hi):
    return _size(rng, _TOKENS, 1, 1, min(32760, int(hi)))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_bwd", "rope", "rope", "rope_bwd", "quant", "product", "product", "product"])
    if op in ("norm", "norm_bwd"):
        B, C = rng.choice([1, 1, 2, 3]), _width(rng, 8, 320, 5120)
        S = _tokens(rng, 160e6 / (B * C))
        fp8 = op == "norm" and rng.random() < 0.4
        return _norm(op, B, S, C, rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.choice(["fp32", "same"]), rng.random() < 0.2 and B * S * C < 6e7,
                     rng.random() < 0.85, rng.choice(["layer", "rms"]), rng.choice(["none", "none", "rms", "layer"]), rng.random() < 0.4, fp8)
    if op in ("rope", "rope_bwd"):
        B, H = rng.choice([1, 1, 2]), rng.randint(1, 40)
        D, axes = rng.choice([(128, (16, 56, 56)), (128, (44, 42, 42)), (64, (16, 24, 24)), (72, (0, 36, 36)), (96, (32, 32, 24)), (128, (16, 24, 24))])
        S = _tokens(rng, 160e6 / (B * H * D))
        Hk = rng.choice([H, H, H, max(1, H // 4)])
        return _rope(op, B, S, H, Hk, D, axes, rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.random() < 0.7, rng.choice(["interleaved", "split_half"]),
                     rng.choice(["bshd", "bhsd"]), rng.choice([0, 0, min(S, 154)]))
    if op == "quant":
        K = _width(rng, 16, 320, 13824)
        return _quant(_tokens(rng, 160e6 / K), K, rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.choice([1, 1, 128]))
    N, K = _width(rng, 1, 64, 16000), _width(rng, 16, 320, 13824)
    M = _tokens(rng, 2e12 / (N * K))
    return _product(M, N, K, rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.random() < 0.6)


# ---- inputs --------------------------------------------------------------------------------


class _State:
    pass


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _channels(g, C):
    """Per-channel sizes of activations: most near 1, a few of them many times that."""
    return torch.exp(0.4 * _randn(g, C)) * (1 + 12 * (torch.rand(C, generator=g, device="cuda") < 0.01))


def _prepare_norm(s, case, g):
    B, S, C, dt = case["B"], case["S"], case["C"], _DTYPES[case["dtype"]]
    md = torch.float32 if case["mods"] == "fp32" else dt
    ms = (B, S, C) if case["per_token"] else (B, 1, C)
    size = _channels(g, C)
    s.x = (_randn(g, B, S, C) * size + 0.2).to(dt)
    s.y = (_randn(g, B, S, C) * size.flip(0)).to(dt) if case["y"] else None
    s.gate = (0.5 * _randn(g, *ms)).to(md) if case["y"] else None
    s.scale, s.shift = (0.3 * _randn(g, *ms)).to(md), (0.3 * _randn(g, *ms)).to(md)
    s.weight = (1 + 0.2 * _randn(g, C)).to(dt) if case["affine"] else None
    s.bias = (0.2 * _randn(g, C)).to(dt) if case["affine"] and case["norm"] == "layer" else None
    s.y_norm = None if case["y_norm"] == "none" or not case["y"] else case["y_norm"]
    s.y_weight = (1 + 0.2 * _randn(g, C)).to(dt) if s.y_norm and case["affine"] else None
    s.alpha, s.eps = 0.7, 1e-6
    if case["op"] == "norm_bwd":  # what the forward pass has left behind
        h, _, stats = _norm_plain(s, case)
        s.h, s.stats = h.to(dt), stats.float()
        s.dh, s.dn = _randn(g, B, S, C).to(dt), _randn(g, B, S, C).to(dt)
        s.x = None


def _prepare_rope(s, case, g):
    B, S, H, Hk, D, dt = case["B"], case["S"], case["H"], case["Hk"], case["D"], _DTYPES[case["dtype"]]

    def tensor(heads):
        if case["layout"] == "bshd":
            return _randn(g, B, S, heads, D).to(dt).transpose(1, 2)
        return _randn(g, B, heads, S, D).to(dt)

    s.q, s.k = tensor(H), tensor(Hk)
    s.q_weight = (1 + 0.2 * _randn(g, D)).to(dt) if case["qk_norm"] else None
    s.k_weight = (1 + 0.2 * _randn(g, D)).to(dt) if case["qk_norm"] else None
    axes = (case["axis_t"], case["axis_h"], case["axis_w"])
    s.pairs = tuple(d // 2 for d in axes)
    s.inv_freq = torch.cat([10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / max(d, 1)) for d in axes])
    # text tokens first, all at the origin, then the grid, centred in height and width
    n = S - case["text"]
    wide = max(1, int(math.sqrt(max(n, 1))) if case["axis_t"] < 20 else 52)
    tall = max(1, -(-n // wide) if case["axis_t"] < 20 else 30)
    i = torch.arange(max(n, 0), device="cuda")
    grid = torch.stack([i // (wide * tall), (i // wide) % tall - tall // 2, i % wide - wide // 2], 1)
    s.positions = torch.cat([torch.zeros(S - n, 3, dtype=grid.dtype, device="cuda"), grid]).float()
    if case["op"] == "rope_bwd":
        s.dq, s.dk = tensor(H), tensor(Hk)


def _quant_plain(x, rows):
    """x (M, K) fp32 -> (e4m3 values, scales (M or M / 128, K / 128))."""
    M, K = x.shape
    kb, mb = -(-K // _BLOCK), -(-M // rows)
    p = torch.nn.functional.pad(x, (0, kb * _BLOCK - K, 0, mb * rows - M)).view(mb, rows, kb, _BLOCK)
    amax = p.abs().amax((1, 3))
    scale = torch.where(amax == 0, torch.ones_like(amax), torch.clamp(amax / _F8_MAX, min=2.0 ** -126))
    y = (p / scale[:, None, :, None]).clamp(-_F8_MAX, _F8_MAX)
    return y.view(mb * rows, kb * _BLOCK)[:M, :K].to(torch.float8_e4m3fn), scale


def _prepare_product(s, case, g):
    M, N, K = case["M"], case["N"], case["K"]
    s.x8, xs = _quant_plain(_randn(g, M, K) * _channels(g, K), 1)
    s.xs = xs.t().contiguous().t()   # as the quantiser leaves it: the scales of a block of columns side by side
    s.w8, s.ws = _quant_plain(_randn(g, N, K) * K ** -0.5, _BLOCK)
    s.x8, s.w8 = s.x8.contiguous(), s.w8.contiguous()
    s.bias = 0.1 * _randn(g, N) if case["bias"] else None
    s.dtype = _DTYPES[case["out"]]


def prepare(case, seed):
    s, g = _State(), _gen(seed)
    s.case = case
    if case["op"] in ("norm", "norm_bwd"):
        _prepare_norm(s, case, g)
    elif case["op"] in ("rope", "rope_bwd"):
        _prepare_rope(s, case, g)
    elif case["op"] == "quant":
        s.x = (_randn(g, case["M"], case["K"]) * (_channels(g, case["K"]) if case["rows"] == 1 else 0.02)).to(_DTYPES[case["dtype"]])
    else:
        _prepare_product(s, case, g)
    return s


# ---- plain forms ---------------------------------------------------------------------------


def _f(t):
    return None if t is None else t.float()


def _stat(x, kind, eps):
    """(mean, reciprocal deviation) of a norm over the last dimension; the RMS norm's mean is zero."""
    mean = x.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(x[..., :1])
    return mean, torch.rsqrt((x - mean).square().mean(-1, keepdim=True) + eps)


def _norm_plain(s, case):
    x, y, w, b, yw = _f(s.x), _f(s.y), _f(s.weight), _f(s.bias), _f(s.y_weight)
    ym, yr = torch.zeros_like(x[..., :1]), torch.ones_like(x[..., :1])
    h = x
    if y is not None:
        if s.y_norm:
            ym, yr = _stat(y, s.y_norm, s.eps)
            y = (y - ym) * yr
            y = y if yw is None else y * yw
        h = x + s.alpha * s.gate.float() * y
    m, r = _stat(h, case["norm"], s.eps)
    n = (h - m) * r
    n = n if w is None else n * w
    n = n if b is None else n + b
    n = n * (1 + s.scale.float()) + s.shift.float()
    return h, n, torch.cat([m, r, ym, yr], -1)


def _norm_bwd_plain(s, case):
    over = (1,) if not case["per_token"] else ()
    cols = (0, 1)
    dh, dn, h, y = _f(s.dh), _f(s.dn), _f(s.h), _f(s.y)
    w, b, yw = _f(s.weight), _f(s.bias), _f(s.y_weight)
    m, r, ym, yr = s.stats.split(1, -1)
    col = lambda t: t.sum(over, keepdim=True) if over else t  # noqa: E731
    u = (h - m) * r
    a = dn * (1 + s.scale.float())
    out = {"dshift": col(dn), "dscale": col(dn * ((u if w is None else u * w) + (0 if b is None else b)))}
    if w is not None:
        out["dweight"] = (a * u).sum(cols)
    if b is not None:
        out["dbias"] = a.sum(cols)
    du = a if w is None else a * w
    t = du - u * (du * u).mean(-1, keepdim=True)
    if case["norm"] == "layer":
        t = t - du.mean(-1, keepdim=True)
    t = dh + r * t
    out["dx"] = t
    if y is not None:
        z = (y - ym) * yr
        out["dgate"] = col(s.alpha * t * (z if yw is None else z * yw))
        e = s.alpha * s.gate.float() * t
        if yw is not None:
            out["dy_weight"] = (e * z).sum(cols)
            e = e * yw
        if s.y_norm:
            d = e - z * (e * z).mean(-1, keepdim=True)
            if s.y_norm == "layer":
                d = d - e.mean(-1, keepdim=True)
            e = yr * d
        out["dy"] = e
    types = {"dx": s.h, "dy": s.y, "dgate": s.gate, "dscale": s.scale, "dshift": s.shift, "dweight": s.weight, "dbias": s.bias, "dy_weight": s.y_weight}
    return {k: v.to(types[k].dtype) for k, v in out.items()}


def _angles(s):
    """(S, rotated pairs): the position of a pair's axis times its frequency."""
    axis = torch.cat([torch.full((n,), a, dtype=torch.long, device="cuda") for a, n in enumerate(s.pairs)])
    phi = s.positions[:, axis] * s.inv_freq.float()
    return torch.cos(phi), torch.sin(phi)


def _rotate(x, cos, sin, pairing):
    R = 2 * cos.shape[-1]
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if pairing == "interleaved" else (x[..., :R // 2], x[..., R // 2:R])
    a, b = a * cos - b * sin, a * sin + b * cos
    r = torch.stack([a, b], -1).flatten(-2) if pairing == "interleaved" else torch.cat([a, b], -1)
    return torch.cat([r, x[..., R:]], -1)


def _rope_plain(s, case):
    cos, sin = _angles(s)

    def one(x, w):
        x = x.float()
        if case["qk_norm"]:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()
        return _rotate(x, cos, sin, case["pairing"])

    dt = s.q.dtype
    return one(s.q, s.q_weight).to(dt), one(s.k, s.k_weight).to(dt)


def _rope_bwd_plain(s, case):
    cos, sin = _angles(s)

    def one(d, x, w):
        d = _rotate(d.float(), cos, -sin, case["pairing"])
        if not case["qk_norm"]:
            return d.to(x.dtype), None
        r = torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6)
        u = x.float() * r
        g = d * w.float()
        return (r * (g - u * (g * u).mean(-1, keepdim=True))).to(x.dtype), (d * u).sum((0, 1, 2)).to(w.dtype)

    (dq, dqw), (dk, dkw) = one(s.dq, s.q, s.q_weight), one(s.dk, s.k, s.k_weight)
    return dq, dk, dqw, dkw


def _spread(scale, rows, M, K):
    return scale.repeat_interleave(_BLOCK, 1)[:, :K].repeat_interleave(rows, 0)[:M]


def _product_plain(s, case):
    x = s.x8.float() * _spread(s.xs, 1, case["M"], case["K"])
    w = s.w8.float() * _spread(s.ws, _BLOCK, case["N"], case["K"])
    y = x @ w.t()
    return (y if s.bias is None else y + s.bias).to(s.dtype)


def _run_plain(s):
    case = s.case
    if case["op"] == "norm":
        h, n, _ = _norm_plain(s, case)
        h = h.to(s.x.dtype)
        if not case["fp8"]:
            return h, n.to(s.x.dtype)
        n8, scale = _quant_plain(n.view(-1, case["C"]), 1)
        return h, n8.view(n.shape), scale.view(n.shape[0], n.shape[1], -1)
    if case["op"] == "norm_bwd":
        return _norm_bwd_plain(s, case)
    if case["op"] == "rope":
        return _rope_plain(s, case)
    if case["op"] == "rope_bwd":
        return _rope_bwd_plain(s, case)
    if case["op"] == "quant":
        return _quant_plain(s.x.float(), case["rows"])
    return _product_plain(s, case)


# ---- the package's entry points --------------------------------------------------------------


def _run_own(s):
    from xdit_amd import block_ops
    case = s.case
    if case["op"] == "norm":
        h, n = block_ops.gated_norm(s.x, y=s.y, gate=s.gate, scale=s.scale, shift=s.shift, weight=s.weight, bias=s.bias, norm=case["norm"], eps=s.eps,
                                    y_norm=s.y_norm, y_weight=s.y_weight, residual_scale=s.alpha, fp8=case["fp8"])
        return (h, n[0], n[1]) if case["fp8"] else (h, n)
    if case["op"] == "norm_bwd":
        return block_ops.gated_norm_backward(s.dh, s.dn, s.h, s.stats, y=s.y, gate=s.gate, scale=s.scale, shift=s.shift, weight=s.weight, bias=s.bias,
                                             norm=case["norm"], y_norm=s.y_norm, y_weight=s.y_weight, residual_scale=s.alpha)
    if case["op"] == "rope":
        return block_ops.axes_rope(s.q, s.k, s.positions, s.inv_freq, s.pairs, norm=case["qk_norm"], q_weight=s.q_weight, k_weight=s.k_weight,
                                   eps=1e-6, rope=case["pairing"])
    if case["op"] == "rope_bwd":
        return block_ops.axes_rope_backward(s.dq, s.dk, s.positions, s.inv_freq, s.pairs, q=s.q, k=s.k, norm=case["qk_norm"], q_weight=s.q_weight,
                                            k_weight=s.k_weight, eps=1e-6, rope=case["pairing"])
    if case["op"] == "quant":
        return block_ops.fp8_block_quant(s.x, block_rows=case["rows"])
    return block_ops.fp8_block_matmul(s.x8, s.xs, s.w8, s.ws, bias=s.bias, out_dtype=s.dtype)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- from the definitions, in 64 bits --------------------------------------------------------


def _d(t):
    return None if t is None else t.double()


def _exact_quant(x, rows):
    M, K = x.shape
    mb, kb = -(-M // rows), -(-K // _BLOCK)
    top = torch.zeros(mb * rows, kb * _BLOCK, dtype=torch.float64, device=x.device)
    top[:M, :K] = x.abs()
    top = top.view(mb, rows, kb, _BLOCK).amax(3).amax(1)
    scale = torch.where(top > 0, (top / _F8_MAX).clamp(min=2.0 ** -126), 1.0)
    return x / scale.repeat_interleave(rows, 0)[:M].repeat_interleave(_BLOCK, 1)[:, :K], scale


def _exact_unit(x, kind, eps):
    """A vector over its last dimension brought to mean 0 (layer) and mean square 1."""
    c = x - x.sum(-1, keepdim=True) / x.shape[-1] if kind == "layer" else x
    return c / torch.sqrt(c.pow(2).sum(-1, keepdim=True) / x.shape[-1] + eps)


def _exact_norm(s, case):
    h = _d(s.x)
    if s.y is not None:
        v = _exact_unit(_d(s.y), s.y_norm, s.eps) if s.y_norm else _d(s.y)
        if s.y_weight is not None:
            v = v * _d(s.y_weight)
        h = h + s.alpha * (_d(s.gate) * v)
    n = _exact_unit(h, case["norm"], s.eps)
    if s.weight is not None:
        n = n * _d(s.weight)
    if s.bias is not None:
        n = n + _d(s.bias)
    n = n + n * _d(s.scale) + _d(s.shift)
    if not case["fp8"]:
        return h, n
    q, scale = _exact_quant(n.view(-1, case["C"]), 1)
    return h, q.view(n.shape), scale.view(n.shape[0], n.shape[1], -1)


def _exact_norm_bwd(s, case):
    """Chain rule through n = N(h) . w . (1 + scale) + ... and h = x + alpha gate v, element by element."""
    st = _d(s.stats)
    C = case["C"]
    h_mean, h_r, y_mean, y_r = (st[..., i:i + 1] for i in range(4))
    hat = (_d(s.h) - h_mean) * h_r
    w = torch.ones(C, dtype=torch.float64, device="cuda") if s.weight is None else _d(s.weight)
    b = torch.zeros(C, dtype=torch.float64, device="cuda") if s.bias is None else _d(s.bias)
    up = _d(s.dn)
    one = 1 + _d(s.scale)
    keep = case["per_token"]
    fold = (lambda t: t) if keep else (lambda t: torch.sum(t, 1, keepdim=True))
    g = {"dshift": fold(up), "dscale": fold(up * (hat * w + b))}
    if s.weight is not None:
        g["dweight"] = torch.sum(up * one * hat, (0, 1))
    if s.bias is not None:
        g["dbias"] = torch.sum(up * one, (0, 1))
    back = up * one * w
    inner = torch.sum(back * hat, -1, keepdim=True) / C
    flat = torch.sum(back, -1, keepdim=True) / C if case["norm"] == "layer" else 0.0
    total = _d(s.dh) + (back - flat - hat * inner) * h_r
    g["dx"] = total
    if s.y is not None:
        yw = torch.ones(C, dtype=torch.float64, device="cuda") if s.y_weight is None else _d(s.y_weight)
        hat = (_d(s.y) - y_mean) * y_r
        g["dgate"] = fold(total * hat * yw) * s.alpha
        e = total * _d(s.gate) * s.alpha
        if s.y_weight is not None:
            g["dy_weight"] = torch.sum(e * hat, (0, 1))
        e = e * yw
        if s.y_norm:
            inner = torch.sum(e * hat, -1, keepdim=True) / C
            flat = torch.sum(e, -1, keepdim=True) / C if s.y_norm == "layer" else 0.0
            e = (e - flat - hat * inner) * y_r
        g["dy"] = e
    return g


def _exact_turn(x, s, case, sign):
    """Every pair as a complex number times exp(i sign phi)."""
    axis = [a for a, n in enumerate(s.pairs) for _ in range(n)]
    phi = sign * s.positions.double()[:, axis] * s.inv_freq
    R = 2 * len(axis)
    z = x[..., :R].unflatten(-1, (R // 2, 2)) if case["pairing"] == "interleaved" else x[..., :R].unflatten(-1, (2, R // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * torch.polar(torch.ones_like(phi), phi))
    r = z.flatten(-2) if case["pairing"] == "interleaved" else z.transpose(-1, -2).flatten(-2)
    return torch.cat([r, x[..., R:]], -1)


def _exact_rope(s, case):
    def one(x, w):
        x = _exact_unit(_d(x), "rms", 1e-6) * _d(w) if case["qk_norm"] else _d(x)
        return _exact_turn(x, s, case, 1)

    return one(s.q, s.q_weight), one(s.k, s.k_weight)


def _exact_rope_bwd(s, case):
    def one(d, x, w):
        d = _exact_turn(_d(d), s, case, -1)
        if not case["qk_norm"]:
            return d, None
        x = _d(x)
        size = torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6)
        hat = x / size
        g = d * _d(w)
        return (g - hat * (torch.sum(g * hat, -1, keepdim=True) / x.shape[-1])) / size, torch.sum(d * hat, (0, 1, 2))

    (dq, dqw), (dk, dkw) = one(s.dq, s.q, s.q_weight), one(s.dk, s.k, s.k_weight)
    return dq, dk, dqw, dkw


def _exact_product(s, case):
    M, N, K = case["M"], case["N"], case["K"]
    x, w = s.x8.double(), s.w8.double()
    y = torch.zeros(M, N, dtype=torch.float64, device="cuda")
    for kb in range(-(-K // _BLOCK)):
        at = slice(kb * _BLOCK, min(K, (kb + 1) * _BLOCK))
        y.addmm_(x[:, at] * s.xs[:, kb:kb + 1].double(), (w[:, at] * s.ws[:, kb].double().repeat_interleave(_BLOCK)[:N, None]).t())
    return y if s.bias is None else y + s.bias.double()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s, case)
    if case["op"] == "norm_bwd":
        return _exact_norm_bwd(s, case)
    if case["op"] == "rope":
        return _exact_rope(s, case)
    if case["op"] == "rope_bwd":
        return _exact_rope_bwd(s, case)
    if case["op"] == "quant":
        return _exact_quant(s.x.double(), case["rows"])
    return _exact_product(s, case)


# ---- what a pass cannot do without -----------------------------------------------------------


def work(case):
    if case["op"] in ("norm", "norm_bwd"):
        n, e = case["B"] * case["S"] * case["C"], _BYTES[case["dtype"]]
        me = 4 if case["mods"] == "fp32" else e
        mods = (n if case["per_token"] else case["B"] * case["C"]) * me
        has_y = 1 if case["y"] else 0
        if case["op"] == "norm":
            out = n + 4 * case["B"] * case["S"] * -(-case["C"] // _BLOCK) if case["fp8"] else n * e
            return {"bytes": n * e * (1 + 2 * has_y) + out + mods * (2 + has_y), "flops": 14.0 * n}
        return {"bytes": n * e * (4 + 2 * has_y) + mods * (3 + 2 * has_y), "flops": 30.0 * n}
    if case["op"] in ("rope", "rope_bwd"):
        n, e = case["B"] * case["S"] * (case["H"] + case["Hk"]) * case["D"], _BYTES[case["dtype"]]
        reads = 1 if case["op"] == "rope" or not case["qk_norm"] else 2
        return {"bytes": n * e * (reads + 1) + 12 * case["S"], "flops": 10.0 * n}
    if case["op"] == "quant":
        n = case["M"] * case["K"]
        return {"bytes": n * (_BYTES[case["dtype"]] + 1) + 4 * -(-case["M"] // case["rows"]) * -(-case["K"] // _BLOCK), "flops": 3.0 * n}
    M, N, K = case["M"], case["N"], case["K"]
    kb = -(-K // _BLOCK)
    return {"bytes": M * K + N * K + 4 * (M + -(-N // _BLOCK)) * kb + M * N * _BYTES[case["out"]] + (4 * N if case["bias"] else 0), "flops": 2.0 * M * N * K}
