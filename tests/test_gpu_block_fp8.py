"""The block-wise fp8 quantiser and the block-scaled fp8 product against the float64 oracle.

Quantiser: scale and bytes are those of fp32 divisions, compared bit for bit with torch's (whose division and cast round the same
way).  Product with exact sums: a block's 128 products are exact in fp32, their sum is off by at most 128 units of 2^-24 of the terms' sizes, the
scale's product by one, and every block's multiply-add (and every joined part's addition) by one of the sum so far; one rounding
to the output's dtype at the end.  Without: the matrix instructions add eight consecutive k at a time and cut each product at
2^-13 of the largest one's binade, so a group of eight adds at most 8 * 2^-13 of its largest product to that.
"""
import pytest
import torch

from oracle import block_oracle as O
from xdit_amd import block_ops, ops

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def quant_plain(x, rows):
    """fp32 divisions on the CPU."""
    x = x.float().cpu()
    M, K = x.shape
    mb, kb = -(-M // rows), -(-K // 128)
    p = torch.zeros(mb * rows, kb * 128)
    p[:M, :K] = x
    p = p.view(mb, rows, kb, 128)
    top = p.abs().amax((1, 3))
    scale = torch.where(top == 0, torch.ones_like(top), (top / 448.0).clamp(min=2.0 ** -126))
    return (p / scale[:, None, :, None]).view(mb * rows, kb * 128)[:M, :K].clamp(-448, 448).to(torch.float8_e4m3fn), scale


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,K", [(1, 8), (3, 136), (128, 128), (130, 1160), (257, 5120), (700, 640), (129, 264)])
def test_quantiser_has_the_bytes_of_a_division(gpu, dtype, M, K):
    g = torch.Generator().manual_seed(M + K)
    x = torch.randn(M, K, generator=g) * torch.exp(2 * torch.randn(K, generator=g))
    x[M // 2] = 0
    x[:, :K // 3] *= 1e-4 if dtype == torch.float16 else 1e-30
    x = x.to(dtype)
    wide = torch.full((M, K + 16), 3.0, dtype=dtype)
    wide[:, 8:8 + K] = x
    for rows in (1, 128):
        y, s = block_ops.fp8_block_quant(wide.to(gpu)[:, 8:8 + K], block_rows=rows)
        ry, rs = quant_plain(x, rows)
        assert y.is_contiguous() and s.shape == rs.shape
        assert torch.equal(s.cpu(), rs)
        assert torch.equal(y.cpu().view(torch.uint8), ry.view(torch.uint8))
    if M % 2 == 0:
        y3, s3 = block_ops.fp8_block_quant(x.to(gpu).view(2, M // 2, K))
        y, s = block_ops.fp8_block_quant(x.to(gpu))
        assert torch.equal(y3.view(M, K).view(torch.uint8), y.view(torch.uint8)) and torch.equal(s3.reshape(s.shape), s)


@pytest.mark.gpu
def test_quantiser_of_special_values(gpu):
    """Zeros keep scale 1, the smallest fp32 numbers a scale of 2^-126, the largest theirs; a NaN or an infinity spoils its own block."""
    x = torch.randn(4, 512)
    x[0, :128] = 0
    x[1, 128:256] = 1e-42
    x[2, 256:384] = 3.4e38
    x[3, 130] = float("nan")
    x[3, 400] = float("inf")
    y, s = block_ops.fp8_block_quant(x.to(gpu))
    ry, rs = quant_plain(x, 1)
    ok = torch.isfinite(rs)
    assert torch.equal(torch.isnan(s.cpu()), torch.isnan(rs)) and torch.equal(s.cpu()[ok], rs[ok]) and s[0, 0] == 1 and s[1, 1] == 2.0 ** -126 and torch.isinf(s[3, 3])
    fine = ok.repeat_interleave(128, 1)
    assert torch.equal(y.cpu().view(torch.uint8)[fine], ry.view(torch.uint8)[fine])
    assert torch.isnan(y[3, 128:256].float()).all() and torch.isnan(y[3, 400].float()) and (y[3, 384:400].float() == 0).all()
    t, ts = block_ops.fp8_block_quant(x.to(gpu), block_rows=128)
    assert torch.isfinite(ts[0, [0, 2]]).all() and torch.isnan(ts[0, 1]) and torch.isinf(ts[0, 3])


def operands(gpu, M, N, K, seed=0):
    g = torch.Generator(device=gpu).manual_seed(M * 7 + N * 13 + K + seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=gpu)  # noqa: E731
    x, xs = block_ops.fp8_block_quant(rn(M, K) * torch.exp(0.5 * rn(K)))
    w, ws = block_ops.fp8_block_quant(rn(N, K) * K ** -0.5, block_rows=128)
    return x, xs, w, ws, rn(N)


def check(got, x, xs, w, ws, bias, exact, tops=None):
    ref, size = O.block_matmul(x, xs, w, ws, bias)
    units = 128 + 2 + xs.shape[1] + 32
    err = (got.double() - ref).abs()
    bound = HALF[got.dtype] * ref.abs() * 1.01 + TINY[got.dtype] + units * 2.0 ** -24 * size
    if not exact:
        bound = bound + 2.0 ** -10 * (O.largest_of_eights(x, xs, w, ws) if tops is None else tops)
    assert bool((err <= bound).all()), (err - bound).max().item()


SHAPES = [(1, 1, 16), (1, 30, 2064), (2, 130, 128), (5, 257, 1152), (16, 640, 5120), (17, 96, 400), (33, 1000, 272), (64, 64, 64), (100, 1925, 1920), (128, 128, 1280),
          (129, 384, 1024), (226, 513, 640), (256, 256, 2560), (300, 777, 1488), (512, 1920, 144), (1000, 640, 640), (2050, 1152, 1152), (700, 2500, 5120)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product_against_oracle(gpu, M, N, K):
    x, xs, w, ws, bias = operands(gpu, M, N, K)
    tops = O.largest_of_eights(x, xs, w, ws)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        for b in (None, bias, bias.to(dtype)):
            for exact in (True, False):
                y = block_ops.fp8_block_matmul(x, xs, w, ws, bias=b, out_dtype=dtype, exact_sums=exact)
                assert y.shape == (M, N) and y.dtype == dtype
                check(y, x, xs, w, ws, b, exact, tops)
        default = block_ops.fp8_block_matmul(x, xs, w, ws, bias=b, out_dtype=dtype)
        assert torch.equal(default, block_ops.fp8_block_matmul(x, xs, w, ws, bias=b, out_dtype=dtype, exact_sums=dtype == torch.float32))
    again = block_ops.fp8_block_matmul(x, xs, w, ws, bias=bias.to(dtype), out_dtype=dtype)
    assert torch.equal(again, default)


@pytest.mark.gpu
@pytest.mark.parametrize("cus", [1, 3, 40, 256, 1000])
def test_product_planned_for_other_chips(gpu, cus, monkeypatch):
    """The launch rule at sizes on both sides of its choices: every plan gives the product."""
    monkeypatch.setitem(ops.TUNING, "cu_count", cus)
    for M, N, K in ((1, 500, 2048), (20, 333, 1024), (80, 400, 1920), (200, 640, 640), (600, 600, 768)):
        x, xs, w, ws, bias = operands(gpu, M, N, K, cus)
        for exact in (True, False):
            check(block_ops.fp8_block_matmul(x, xs, w, ws, bias=bias, exact_sums=exact), x, xs, w, ws, bias, exact)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(3, 200, 400), (150, 330, 656)])
def test_strides_and_neighbours(gpu, M, N, K):
    """Padded rows, scales of any strides, an output inside a larger tensor, (B, S, K) activations."""
    x, xs, w, ws, bias = operands(gpu, M, N, K)
    ref = block_ops.fp8_block_matmul(x, xs, w, ws, bias=bias)
    xp = torch.full((M, K + 48), 240.0, device=gpu).to(torch.float8_e4m3fn)
    wp = torch.full((N + 3, K + 32), float("nan"), device=gpu).to(torch.float8_e4m3fn)
    xp[:, 16:16 + K] = x
    wp[:N, :K] = w
    sp = torch.full((2 * M, 3 * xs.shape[1]), float("nan"), device=gpu)
    sp[::2, ::3] = xs
    out = torch.full((M, N + 7), 5.0, device=gpu, dtype=torch.bfloat16)
    y = block_ops.fp8_block_matmul(xp[:, 16:16 + K], sp[::2, ::3], wp[:N, :K], ws.t().contiguous().t(), bias=bias, out=out[:, 3:3 + N])
    assert torch.equal(y, ref) and bool((out[:, :3] == 5).all()) and bool((out[:, 3 + N:] == 5).all())
    if M % 3 == 0:
        y3 = block_ops.fp8_block_matmul(x.view(3, M // 3, K), xs.contiguous().view(3, M // 3, -1), w, ws, bias=bias)
        assert torch.equal(y3.view(M, N), ref)
    assert block_ops.fp8_block_matmul(x[:0], xs[:0], w, ws).shape == (0, N)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 40, 300])
def test_a_bad_row_stays_by_itself(gpu, M):
    x, xs, w, ws, bias = operands(gpu, M, 320, 1024)
    ref = block_ops.fp8_block_matmul(x, xs, w, ws)
    xs = xs.clone()
    xs[M // 2, 3] = float("nan")
    y = block_ops.fp8_block_matmul(x, xs, w, ws)
    assert torch.isnan(y[M // 2].float()).all()
    keep = torch.arange(M, device=gpu) != M // 2
    assert torch.equal(y[keep], ref[keep])


@pytest.mark.gpu
def test_gradient_to_the_input_through_the_transposed_weight(gpu):
    """dx = dy w: 128 x 128 blocks transpose exactly, so the same product serves, on the weight laid out once the other way."""
    M, N, K = 70, 384, 640
    _, _, w, ws, _ = operands(gpu, M, N, K)
    dy = torch.randn(M, N, device=gpu)
    d8, ds = block_ops.fp8_block_quant(dy)
    dx = block_ops.fp8_block_matmul(d8, ds, w.t().contiguous(), ws.t(), out_dtype=torch.float32)
    check(dx, d8, ds, w.t().contiguous(), ws.t(), None, True)
    full = w.double() * O.spread(ws.double(), 128, N, K)
    assert (dx.double() - dy.double() @ full).abs().max().item() <= 2.0 ** -4 * (dy.double().abs() @ full.abs()).max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 50, 600])
def test_streams_and_graph(gpu, M):
    x, xs, w, ws, bias = operands(gpu, M, 640, 2048)
    ref = block_ops.fp8_block_matmul(x, xs, w, ws, bias=bias)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    src = torch.randn(M, 2048, device=gpu)
    with torch.cuda.stream(side):
        assert torch.equal(block_ops.fp8_block_matmul(x, xs, w, ws, bias=bias), ref)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            q, s = block_ops.fp8_block_quant(src)
            y = block_ops.fp8_block_matmul(q, s, w, ws, bias=bias)
    for _ in range(3):
        src.mul_(-0.7)
        want = block_ops.fp8_block_matmul(*block_ops.fp8_block_quant(src), w, ws, bias=bias)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


@pytest.mark.gpu
def test_refusals(gpu):
    x, xs, w, ws, bias = operands(gpu, 4, 32, 256)
    q, f = block_ops.fp8_block_quant, block_ops.fp8_block_matmul
    src = torch.zeros(4, 256, device=gpu)
    for bad in (lambda: q(src, block_rows=64), lambda: q(src[0]), lambda: q(src.view(2, 2, 256), block_rows=128), lambda: q(src.double()), lambda: q(src[:, 1:9]),
                lambda: q(src[:, ::2]), lambda: f(x, xs[:, :1], w, ws), lambda: f(x, xs, w[:, :128], ws), lambda: f(x, xs, w, ws[:0]), lambda: f(x.float(), xs, w, ws),
                lambda: f(x, xs, w, ws, bias=bias[:3]), lambda: f(x, xs, w, ws, bias=bias.half()), lambda: f(x, xs, w, ws, out_dtype=torch.float64),
                lambda: f(x, xs.double(), w, ws), lambda: f(x, xs, w, ws, out=torch.zeros(4, 32, device=gpu)), lambda: f(x[:, 8:248], xs, w[:, 8:248], ws),
                lambda: f(x, xs, w, ws, out=torch.zeros(1, 32, device=gpu, dtype=torch.bfloat16).expand(4, 32)), lambda: f(x, None, w, ws)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        q(torch.zeros(2, 12, device=gpu))
    with pytest.raises(NotImplementedError):
        f(*q(torch.zeros(2, 24, device=gpu)), *q(torch.zeros(8, 24, device=gpu), block_rows=128))
    with pytest.raises(RuntimeError):
        q(src.cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,K,dtype", [(1, 14801, 1416, torch.bfloat16), (3, 5003, 1416, torch.float16), (1, 161003, 104, torch.float32), (2, 53, 260008, torch.bfloat16)])
def test_quantiser_of_many_blocks(gpu, B, S, K, dtype):
    """Large tensors, rows that are not next to each other, against the plain form and against the same rows a few at a time."""
    g = torch.Generator(device=gpu).manual_seed(S)
    wide = torch.randn(B, S, K + 24, generator=g, device=gpu).to(dtype)
    wide[:, 7] = 0
    x = wide[:, :, 16:16 + K]
    y, s = block_ops.fp8_block_quant(x)
    assert y.is_contiguous() and s.shape == (B, S, -(-K // 128))
    for b in range(B):
        for r0 in (0, S // 2, S - 19):
            part = x[b, r0:r0 + 19]
            ry, rs = quant_plain(part.cpu(), 1)
            py, ps = block_ops.fp8_block_quant(part)
            assert torch.equal(s[b, r0:r0 + 19].cpu(), rs) and torch.equal(y[b, r0:r0 + 19].cpu().view(torch.uint8), ry.view(torch.uint8))
            assert torch.equal(s[b, r0:r0 + 19], ps) and torch.equal(y[b, r0:r0 + 19].view(torch.uint8), py.view(torch.uint8))
    back = y.float() * s.repeat_interleave(128, -1)[..., :K]
    assert bool(((back - x.float()).abs() <= x.float().abs() / 16 + s.repeat_interleave(128, -1)[..., :K] * 2.0 ** -9).all())


@pytest.mark.gpu
@pytest.mark.parametrize("cus,M,N,K", [(5, 1300, 520, 640), (7, 2000, 520, 656), (12, 1900, 700, 1280), (20, 1500, 1100, 1920), (24, 3300, 700, 1024), (3, 777, 264, 512), (3, 485, 206, 1456), (2, 578, 132, 2736)])
def test_product_of_rows_beyond_whole_rounds(gpu, cus, M, N, K, monkeypatch):
    """Rows behind the last full round of large tiles may be a product of their own, in the last two cases with K in parts: results, offsets of every
    operand, padded outputs."""
    monkeypatch.setitem(ops.TUNING, "cu_count", cus)
    x, xs, w, ws, bias = operands(gpu, M, N, K)
    sp = torch.full((M, 2 * xs.shape[1]), float("nan"), device=gpu)[:, ::2]
    sp.copy_(xs)
    for exact in (True, False):
        y = block_ops.fp8_block_matmul(x, xs, w, ws, bias=bias, exact_sums=exact)
        check(y, x, xs, w, ws, bias, exact)
        wide = torch.full((M + 2, N + 24), 7.0, dtype=torch.bfloat16, device=gpu)
        block_ops.fp8_block_matmul(x, sp, w, ws, bias=bias, exact_sums=exact, out=wide[1:-1, 8:8 + N])
        assert torch.equal(wide[1:-1, 8:8 + N], y)
        wide[1:-1, 8:8 + N] = 7
        assert bool((wide == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("cus,M,N,K", [(12, 1900, 700, 1296), (2, 300, 520, 1936), (1, 500, 300, 144), (20, 1500, 1101, 1904)])
def test_large_tiles_with_a_ragged_last_block(gpu, cus, M, N, K, monkeypatch):
    monkeypatch.setitem(ops.TUNING, "cu_count", cus)
    x, xs, w, ws, bias = operands(gpu, M, N, K)
    for exact in (True, False):
        for dtype in (torch.bfloat16, torch.float32):
            check(block_ops.fp8_block_matmul(x, xs, w, ws, bias=bias, out_dtype=dtype, exact_sums=exact), x, xs, w, ws, bias, exact)


@pytest.mark.gpu
@pytest.mark.parametrize("stride", [1 << 24, 1 << 33, 16])
def test_a_single_row_of_any_stride(gpu, stride):
    """One row of x, one of w: the stride to the next row does not matter."""
    x, xs, w, ws, bias = operands(gpu, 1, 130, 400)
    far = torch.as_strided(x, (1, 400), (stride, 1))
    assert far.stride(0) == stride
    assert torch.equal(block_ops.fp8_block_matmul(far, xs, w, ws, bias=bias), block_ops.fp8_block_matmul(x, xs, w, ws, bias=bias))
    x, xs, w, ws, bias = operands(gpu, 70, 1, 400)
    far = torch.as_strided(w, (1, 400), (stride, 1))
    assert torch.equal(block_ops.fp8_block_matmul(x, xs, far, ws, bias=bias), block_ops.fp8_block_matmul(x, xs, w, ws, bias=bias))
