"""A transformer block of a diffusion model on the library's operators, from the modulated norm to the gated residual.

    python examples/dit_block.py                     # a 64 x 64 latent, checked against float32 PyTorch, timed
    python examples/dit_block.py --grid 21 30 52 --heads 40 --mlp 13824 --no-check
    python examples/dit_block.py --grid 1 24 20 --train

    (h, n)  = gated_norm(x, scale, shift)                n in fp8 with its scales
    q, k, v = Fp8Linear(n)                               split into heads by view
    q, k    = axes_rope(q, k, positions)                 norm over head_dim, then rotation by frame, row and column
    o       = attn_fwd(q, k, v)                          written token by token, as the projection reads it
    (h, n)  = gated_norm(h, Fp8Linear(o), gate, scale, shift)
    h       = gated_norm(h, Fp8Linear(gelu(Fp8Linear(n))), gate)

Every step runs on the library's kernels but the activation function, forward and backward; a training step clips the gradients of what it
trains (the modulation and the gains) to a common norm.  Weights are random and frozen.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from xdit_amd import block, grad_ops, ops, usp  # noqa: E402

F = torch.nn.functional


def axes_of(head_dim):
    """head_dim's columns that frame, row and column turn: even thirds, what is left over goes to the frame."""
    side = head_dim // 6 * 2
    return (head_dim - 2 * side, side, side)


def grid_positions(frames, rows, cols, device):
    axes = torch.meshgrid(torch.arange(frames, device=device), torch.arange(rows, device=device), torch.arange(cols, device=device), indexing="ij")
    return torch.stack(axes, -1).reshape(-1, 3)


class DiTBlock(torch.nn.Module):
    def __init__(self, heads, head_dim, mlp, dtype=torch.bfloat16, device="cuda", seed=0, train=False, fp32_attention=False):
        super().__init__()
        self.fp32_attention = fp32_attention   # of a training step
        C = heads * head_dim
        g = torch.Generator(device=device).manual_seed(seed)

        def linear(n, k):
            w = (torch.randn(n, k, generator=g, device=device) * k ** -0.5).to(dtype)
            return block.Fp8Linear(w, (0.1 * torch.randn(n, generator=g, device=device)).to(dtype), backward=train)

        self.heads, self.head_dim = heads, head_dim
        self.qkv, self.proj, self.up, self.down = linear(3 * C, C), linear(C, C), linear(mlp, C), linear(C, mlp)
        for name in ("q_gain", "k_gain"):
            gain = (1 + 0.1 * torch.randn(head_dim, generator=g, device=device)).to(dtype)
            setattr(self, name, torch.nn.Parameter(gain, requires_grad=train))
        freq, self.pairs = block.rope_frequencies(axes_of(head_dim), device=device)
        self.register_buffer("freq", freq)

    def forward(self, x, modulation, positions):
        """x (B, S, C); modulation (B, 6, C): shift, scale and gate of attention, then of the MLP."""
        B, S, C = x.shape
        shift1, scale1, gate1, shift2, scale2, gate2 = modulation.unsqueeze(2).unbind(1)
        train = torch.is_grad_enabled() and any(t.requires_grad for t in (x, modulation, self.q_gain))
        h, n = block.gated_norm(x, scale=scale1, shift=shift1, fp8=not train)
        qkv = self.qkv(n).view(B, S, 3, self.heads, self.head_dim)
        q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
        q, k = block.axes_rope(q, k, positions, self.freq, self.pairs, norm=True, q_weight=self.q_gain, k_weight=self.k_gain)
        if train:
            if self.fp32_attention:
                q, k, v = q.float(), k.float(), v.float()
            o = usp.attention(q, k, v).to(x.dtype).transpose(1, 2).reshape(B, S, C)
        else:
            o = torch.empty_like(x, memory_format=torch.contiguous_format)
            ops.attn_fwd(q, k, v, out=o.view(B, S, self.heads, self.head_dim).transpose(1, 2), return_lse=False)
        h, n = block.gated_norm(h, self.proj(o), gate1, scale2, shift2, fp8=not train)
        y = self.down(F.gelu(self.up(n), approximate="tanh"))
        return block.gated_norm(h, y, gate2, norm=None)[0]


def plain(m, x, modulation, positions, gains=None):
    """The block in float32 PyTorch: the same (already rounded) weights, activations that are never quantised."""
    def linear(p, t):
        scale = p.weight_scale.repeat_interleave(128, 0)[:p.out_features].repeat_interleave(128, 1)[:, :p.in_features]
        return t @ (p.weight.float() * scale).t() + p.bias

    x, modulation = x.float(), modulation.float()
    B, S, C = x.shape
    H, D = m.heads, m.head_dim
    gains = (m.q_gain.float(), m.k_gain.float()) if gains is None else gains
    shift1, scale1, gate1, shift2, scale2, gate2 = modulation.unsqueeze(2).unbind(1)
    q, k, v = (t.view(B, S, H, D).transpose(1, 2) for t in linear(m.qkv, F.layer_norm(x, (C,), eps=1e-6) * (1 + scale1) + shift1).chunk(3, -1))
    axis = torch.repeat_interleave(torch.arange(3, device=x.device), torch.tensor(m.pairs, device=x.device))
    angle = positions.double()[:, axis] * m.freq
    cos, sin = angle.cos().float(), angle.sin().float()

    def rotate(t, gain):
        t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * gain
        a, b = t[..., 0::2], t[..., 1::2]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)

    o = F.scaled_dot_product_attention(rotate(q, gains[0]), rotate(k, gains[1]), v).transpose(1, 2).reshape(B, S, C)
    h = x + gate1 * linear(m.proj, o)
    n = F.layer_norm(h, (C,), eps=1e-6) * (1 + scale2) + shift2
    return h + gate2 * linear(m.down, F.gelu(linear(m.up, n), approximate="tanh"))


def inputs(grid, heads, head_dim, batch=1, dtype=torch.bfloat16, device="cuda", seed=1):
    S, C = grid[0] * grid[1] * grid[2], heads * head_dim
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(batch, S, C, generator=g, device=device).to(dtype)
    return x, (0.5 * torch.randn(batch, 6, C, generator=g, device=device)).to(dtype), grid_positions(*grid, device)


def distance(a, b):
    """Size of a - b relative to b, over all elements."""
    return float((a.float() - b.float()).norm() / b.float().norm().clamp_min(1e-30))


def check(m, x, modulation, positions):
    """Relative distance of what the block adds to x from the float32 form's."""
    with torch.no_grad():
        got, want = m(x, modulation, positions), plain(m, x, modulation, positions)
    return distance(got.float() - x.float(), want - x.float())


def check_gradients(m, x, modulation, positions, seed=2):
    """The same for the gradients of sum(block(x) * r) -> {name: distance}."""
    r = torch.randn(x.shape, generator=torch.Generator(device=x.device).manual_seed(seed), device=x.device).to(x.dtype)
    x1, m1 = x.clone().requires_grad_(), modulation.clone().requires_grad_()
    got = torch.autograd.grad(m(x1, m1, positions), (x1, m1, m.q_gain, m.k_gain), r)
    x2, m2 = x.float().requires_grad_(), modulation.float().requires_grad_()
    gains = [t.detach().float().requires_grad_() for t in (m.q_gain, m.k_gain)]
    want = torch.autograd.grad(plain(m, x2, m2, positions, gains), (x2, m2, *gains), r.float())
    return {n: distance(a, b) for n, a, b in zip(("x", "modulation", "q_gain", "k_gain"), got, want)}


def training_step(m, x, modulation, positions, r, max_norm=1.0):
    """Gradients of sum(block(x) * r) to the modulation and the gains, clipped to a common norm -> (gradients, their norm before that)."""
    leaves = [modulation, m.q_gain, m.k_gain]
    grads = [g.contiguous() for g in torch.autograd.grad(m(x, modulation, positions), leaves, r)]
    return grads, grad_ops.clip_grads(grads, max_norm)


def timed(fn, n=10):
    """Milliseconds of a call among others."""
    for _ in range(3):
        fn()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(n):
        fn()
    end.record()
    end.synchronize()
    return start.elapsed_time(end) / n


def main():
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--grid", type=int, nargs=3, default=(1, 64, 64), help="frames, rows and columns of the latent")
    p.add_argument("--heads", type=int, default=16)
    p.add_argument("--head-dim", type=int, default=128)
    p.add_argument("--mlp", type=int, default=8192)
    p.add_argument("--batch", type=int, default=1)
    p.add_argument("--train", action="store_true", help="check the gradients and time a training step instead of the forward pass")
    p.add_argument("--fp32-attention", action="store_true", help="attention of a training step in float32, forward and backward")
    p.add_argument("--no-check", action="store_true")
    a = p.parse_args()
    m = DiTBlock(a.heads, a.head_dim, a.mlp, train=a.train, fp32_attention=a.fp32_attention)
    data = inputs(a.grid, a.heads, a.head_dim, a.batch)
    size = "%d tokens, %d heads of %d, MLP %d" % (data[0].shape[1], a.heads, a.head_dim, a.mlp)
    if a.train:
        if not a.no_check:
            print("gradients, relative distance to float32:", {n: round(d, 4) for n, d in check_gradients(m, *data).items()})
        x, modulation, positions = data
        modulation.requires_grad_()
        r = torch.randn_like(x)
        print("norm of the gradients: %.3f" % float(training_step(m, x, modulation, positions, r)[1]))
        print("%s: %.3f ms a training step" % (size, timed(lambda: training_step(m, x, modulation, positions, r))))
        return
    if not a.no_check:
        print("output, relative distance to float32: %.4f" % check(m, *data))
    with torch.no_grad():
        print("%s: %.3f ms a block" % (size, timed(lambda: m(*data))))


if __name__ == "__main__":
    main()
