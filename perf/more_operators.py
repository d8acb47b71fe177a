"""What the operators that a training step adds to the forward pass are timed on: attention's backward pass, and the global norm of
a model's gradients with their clipping.

A case is a dict of plain values; `op` says which entry point it goes through:

  attn_bwd    grad_ops.attn_bwd: gradients of q, k, v (and of the joint text keys and values) from those of the
              output, with what the forward pass has left behind (output and log-sum-exp)
  grad_norm   grad_ops.grad_norm of a list of gradients
  clip        grad_ops.clip_grads into a second list (the optimizer's own gradients)

`run` computes them in 32 bits by elementary torch operations where `own` is false, and calls the package's entry points where it is
true.  Sizes are those of the shapes that the benchmark, the tests and the example of this repository use (image models at 512 and
1024 pixels, video at 480p, blocks of 16 x 72, 16 x 128 and 40 x 128) and, in `draw`, the ranges between and around them.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _attn(B, H, Sq, Sk, D, Sk2=0, dtype="bf16", layout="bshd", name=None):
    c = {"op": "attn_bwd", "B": B, "H": H, "Sq": Sq, "Sk": Sk, "Sk2": Sk2, "D": D, "dtype": dtype, "layout": layout}
    return c if name is None else dict(c, name=name)


def _grads(op, blocks, C, mlp, D, dtype="bf16", out="same", frozen=False, name=None):
    """Gradients of `blocks` blocks of hidden size C; `frozen`: of their gains and modulation tables alone."""
    c = {"op": op, "blocks": blocks, "C": C, "mlp": mlp, "D": D, "dtype": dtype, "out": dtype if out == "same" else out, "frozen": frozen}
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # a Ulysses-8 rank's 3 heads of a 512-pixel joint block: 1024 image and 512 text tokens; the smallest
        _attn(1, 3, 1536, 1024, 128, 512, name="attn_image512_3heads"),
        # image model at 512 pixels trained in fp32
        _attn(1, 16, 1024, 1024, 72, dtype="fp32", name="attn_image512_fp32"),
        # 1024-pixel joint block: 4096 image and 512 text tokens
        _attn(1, 24, 4608, 4096, 128, 512, name="attn_image1024_joint"),
        # head_dim-64 image model with two captions a step, BHSD memory
        _attn(2, 24, 4250, 4250, 64, dtype="fp16", layout="bhsd", name="attn_image1024_head64"),
        # cross-attention of 480p video tokens on 512 text tokens
        _attn(1, 40, 32760, 512, 128, name="attn_video480p_cross"),
        # the rank's 5 heads of 480p video self-attention
        _attn(1, 5, 32760, 32760, 128, name="attn_video480p_5heads"),
        # gains and modulation tables of a 28-block model whose weights are frozen: many small tensors, latency
        _grads("grad_norm", 28, 1152, 4608, 72, "fp32", frozen=True, name="norm_gains"),
        # the whole 28-block model
        _grads("grad_norm", 28, 1152, 4608, 72, name="norm_28blocks"),
        # the gains again, clipped
        _grads("clip", 28, 1152, 4608, 72, "fp32", frozen=True, name="clip_gains"),
        # 8 blocks of 16 x 128: bf16 gradients clipped into the fp32 ones that the optimizer steps on
        _grads("clip", 8, 2048, 8192, 128, "bf16", "fp32", name="clip_8blocks_bf16"),
        # two video blocks of 40 x 128, gradients in fp32
        _grads("clip", 2, 5120, 13824, 128, "fp32", name="clip_video_blocks_fp32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn_bwd", "attn_bwd", "attn_bwd", "attn_bwd", "grad_norm", "clip"])
    if op == "attn_bwd":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        D = rng.choice([40, 64, 64, 72, 80, 88, 96, 128, 128, 128])
        B, H = rng.choice([1, 1, 2, 3]), rng.randint(1, 40)
        most = 8e11 if dtype == "fp32" else 5e12   # operations
        Sq = _log_int(rng, 1, min(32760, math.sqrt(most / (10 * B * H * D)) * rng.choice([1, 1, 4])))
        room = max(2.0, most / (10 * B * H * D * Sq))   # over one key the gradients of queries and keys are zeros
        kind = rng.choice(["self", "joint", "cross"])
        if kind == "cross":
            return _attn(B, H, Sq, _log_int(rng, 2, min(1024, room)), D, 0, dtype, rng.choice(["bshd", "bhsd"]))
        keys = max(2, min(Sq, int(room)))
        text = min(keys - 1, _log_int(rng, 16, 512)) if kind == "joint" else 0
        return _attn(B, H, Sq, keys - text, D, text, dtype, rng.choice(["bshd", "bhsd"]))
    D = rng.choice([40, 64, 72, 128])
    C = D * _log_int(rng, 2, 40)
    mlp = 8 * _log_int(rng, C / 8, 4 * C / 8)
    frozen = rng.random() < 0.3
    size = 2 * D + 6 * C if frozen else 4 * C * C + 2 * C * mlp
    blocks = _log_int(rng, 1, max(1, min(40, 4.5e8 / size)))
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    return _grads(op, blocks, C, mlp, D, dtype, rng.choice(["same", "fp32"]), frozen)


# ---- inputs --------------------------------------------------------------------------------


class _State:
    pass


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _shapes(case):
    """Shapes of a model's gradients: projections with their biases, gains and modulation table of every block."""
    C, mlp, D = case["C"], case["mlp"], case["D"]
    gains = [(D,), (D,), (6, C)]
    block = gains if case["frozen"] else [(3 * C, C), (3 * C,), (C, C), (C,), (mlp, C), (mlp,), (C, mlp), (C,)] + gains
    return block * case["blocks"]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = _State()
    s.op, dt = case["op"], _DTYPES[case["dtype"]]
    if s.op == "attn_bwd":
        B, H, D, Sq, Sk, Sk2 = (case[n] for n in ("B", "H", "D", "Sq", "Sk", "Sk2"))

        def tensor(S):
            if case["layout"] == "bshd":
                return _randn(g, B, S, H, D).transpose(1, 2)
            return _randn(g, B, H, S, D)

        # queries and keys as a norm over head_dim with gains leaves them: logits with a deviation of 2
        s.q, s.k, s.v, s.dout = (2 * tensor(Sq)).to(dt), tensor(Sk).to(dt), tensor(Sk).to(dt), tensor(Sq).to(dt)
        s.k2, s.v2 = (tensor(Sk2).to(dt), tensor(Sk2).to(dt)) if Sk2 else (None, None)
        s.scale = D ** -0.5
        # what the forward pass has left behind, head by head
        s.out, s.lse = torch.empty_like(s.q), torch.empty(B, H, Sq, device="cuda")
        for h in range(H):
            keys, values = (torch.cat((a[:, h], b[:, h]), 1) if Sk2 else a[:, h] for a, b in ((s.k, s.k2), (s.v, s.v2)))
            logits = torch.matmul(s.q[:, h].float(), keys.float().transpose(1, 2)) * s.scale
            s.lse[:, h] = torch.logsumexp(logits, -1)
            s.out[:, h] = torch.matmul(torch.exp(logits - s.lse[:, h, :, None]), values.float()).to(dt)
        return s
    # gradients as a backward pass with buckets leaves them: views of one buffer, each of its own size
    shapes = _shapes(case)
    pad = 16 // _BYTES[case["dtype"]]
    sizes = [math.prod(x) for x in shapes]
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + -(-n // pad) * pad)
    s.flat = torch.zeros(starts[-1], dtype=dt, device="cuda")
    s.grads = [s.flat[a:a + n].view(shape) for a, n, shape in zip(starts, sizes, shapes)]
    for t, size in zip(s.grads, torch.exp(torch.randn(len(sizes), generator=torch.Generator().manual_seed(seed))).tolist()):
        t.copy_(_randn(g, *t.shape) * (0.01 * size))
    s.max_norm = 1.0
    if s.op == "clip":
        s.main = torch.zeros(starts[-1], dtype=_DTYPES[case["out"]], device="cuda")
        s.out = [s.main[a:a + n].view(shape) for a, n, shape in zip(starts, sizes, shapes)]
    if own:   # the tensors stay from step to step: a training program lists them once
        from xdit_amd import grad_ops
        s.grads = grad_ops.GradList(s.grads)
        s.out = grad_ops.GradList(s.out) if s.op == "clip" else None
    return s


# ---- plain form ----------------------------------------------------------------------------


def _attn_bwd_plain(s):
    """P = exp(scale q k^T - lse), dV = P^T dO, dS = P (dO V^T - rowsum(dO O)), dQ = scale dS K, dK = scale dS^T Q."""
    dt = s.q.dtype
    q, dout = s.q.float(), s.dout.float()
    k, v = (torch.cat((a, b), 2).float() if b is not None else a.float() for a, b in ((s.k, s.k2), (s.v, s.v2)))
    p = torch.matmul(q, k.transpose(2, 3)).mul_(s.scale).sub_(s.lse.unsqueeze(-1)).exp_()
    dv = torch.matmul(p.transpose(2, 3), dout)
    delta = (dout * s.out.float()).sum(-1, keepdim=True)
    p.mul_(torch.matmul(dout, v.transpose(2, 3)).sub_(delta))
    dq = torch.matmul(p, k).mul_(s.scale).to(dt)
    dk = torch.matmul(p.transpose(2, 3), q).mul_(s.scale).to(dt)
    dv = dv.to(dt)
    n = s.k.shape[2]
    return (dq, dk, dv) if s.k2 is None else (dq, dk[:, :, :n], dv[:, :, :n], dk[:, :, n:], dv[:, :, n:])


def _norm_plain(s):
    """The gradients lie in one buffer, with zeros between them; squares in 32 bits, their long sum in 64."""
    return torch.sqrt(torch.sum(s.flat.float().square(), dtype=torch.float64)).float()


def _clip_plain(s):
    norm = _norm_plain(s)
    factor = torch.clamp(s.max_norm / (norm + 1e-6), max=1.0)
    s.main.copy_(s.flat.float() * factor)
    return norm, s.main


def run(s):
    if own:
        from xdit_amd import grad_ops
        if s.op == "attn_bwd":
            return grad_ops.attn_bwd(s.dout, s.q, s.k, s.v, s.out, s.lse, softmax_scale=s.scale, k2=s.k2, v2=s.v2)
        if s.op == "grad_norm":
            return grad_ops.grad_norm(s.grads)
        return grad_ops.clip_grads(s.grads, s.max_norm, out=s.out), s.main
    if s.op == "attn_bwd":
        return _attn_bwd_plain(s)
    return _norm_plain(s) if s.op == "grad_norm" else _clip_plain(s)


def work(case):
    if case["op"] == "attn_bwd":
        B, H, D, Sq, Sk = case["B"], case["H"], case["D"], case["Sq"], case["Sk"] + case["Sk2"]
        # q, out and dout in, dq out; k and v in, their gradients out; lse.  Five products of Sq x Sk x D.
        return {"bytes": B * H * (4 * D * (Sq + Sk) * _BYTES[case["dtype"]] + 4 * Sq), "flops": 10 * B * H * Sq * Sk * D}
    n = sum(math.prod(x) for x in _shapes(case))
    if case["op"] == "grad_norm":
        return {"bytes": n * _BYTES[case["dtype"]] + 4, "flops": 2 * n}
    return {"bytes": n * (_BYTES[case["dtype"]] + _BYTES[case["out"]]) + 4, "flops": 3 * n}


# ---- 64 bits -------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if s.op == "attn_bwd":
        B, H, D, Sq, Sk = case["B"], case["H"], case["D"], case["Sq"], case["Sk"]
        grads = [torch.empty(B, H, n, D, dtype=torch.float64, device="cuda") for n in (Sq, Sk, Sk, case["Sk2"], case["Sk2"])]
        for b in range(B):
            for h in range(H):
                q, o, do = (t[b, h].double() for t in (s.q, s.out, s.dout))
                parts = [(s.k, s.v, 1, 2)] + ([(s.k2, s.v2, 3, 4)] if s.k2 is not None else [])
                dq = torch.zeros_like(q)
                centre = torch.einsum("id,id->i", do, o)
                for keys, values, at_k, at_v in parts:   # a row's probabilities under its given log-sum-exp
                    k, v = keys[b, h].double(), values[b, h].double()
                    w = torch.exp(torch.einsum("id,jd->ij", q, k) * s.scale - s.lse[b, h].double()[:, None])
                    grads[at_v][b, h] = w.t() @ do
                    w *= (do @ v.t() - centre[:, None]) * s.scale
                    grads[at_k][b, h] = w.t() @ q
                    dq += w @ k
                grads[0][b, h] = dq
        return tuple(grads if s.k2 is not None else grads[:3])
    total = math.sqrt(sum(float(t.double().pow(2).sum()) for t in s.grads))
    norm = torch.tensor(total, dtype=torch.float64)
    if s.op == "grad_norm":
        return norm
    return norm, s.flat.double() * min(1.0, s.max_norm / (total + 1e-6))
