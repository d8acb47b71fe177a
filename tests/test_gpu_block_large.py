"""Tensors whose last rows lie beyond 2^31 elements and 2^32 bytes: they get the bits that the same rows get by themselves, and columns' sums
over all rows are those of the parts."""
import pytest
import torch

from xdit_amd import block_ops

pytestmark = pytest.mark.gpu
ROWS, C = 275000, 8192    # 2.25e9 elements


def same(a, b):
    bits = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[a.element_size()]
    assert torch.equal(a.contiguous().view(bits), b.contiguous().view(bits))


@pytest.fixture(scope="module")
def rows(gpu):
    x = torch.empty(1, ROWS, C, dtype=torch.bfloat16, device=gpu)
    g = torch.Generator(device=gpu).manual_seed(5)
    x[:, :1000].normal_(generator=g)
    for i in range(1000, ROWS, 1000):   # every thousand rows turned and scaled a little
        x[:, i:i + 1000] = x[:, :min(1000, ROWS - i)].roll(i // 1000, -1)
    yield x
    del x
    torch.cuda.empty_cache()


SPANS = (0, 131070, ROWS - 300)


def test_norm_and_its_gradient(gpu, rows):
    s = torch.linspace(-1, 1, C, device=gpu).view(1, 1, C)
    h, n, st = block_ops.gated_norm(rows, rows, s, s, s, return_stats=True)
    n8, sc = block_ops.gated_norm(rows, scale=s, norm="rms", fp8=True)[1]
    for a in SPANS:
        part = rows[:, a:a + 300]
        ph, pn, ps = block_ops.gated_norm(part, part, s, s, s, return_stats=True)
        same(h[:, a:a + 300], ph)
        same(n[:, a:a + 300], pn)
        same(st[:, a:a + 300], ps)
        p8, pc = block_ops.gated_norm(part, scale=s, norm="rms", fp8=True)[1]
        same(n8[:, a:a + 300], p8)
        same(sc[:, a:a + 300], pc)
    del n8
    r = block_ops.gated_norm_backward(n, rows, h, st, rows, s, s, s)
    total = 0
    for a in SPANS:
        part = [t[:, a:a + 300] for t in (n, rows, h)]
        p = block_ops.gated_norm_backward(*part, st[:, a:a + 300].contiguous(), part[1], s, s, s)
        same(r["dx"][:, a:a + 300], p["dx"])
        same(r["dy"][:, a:a + 300], p["dy"])
    for i in range(0, ROWS, 1000):   # dshift is the plain column sum of dn
        total = total + rows[:, i:i + 1000].double().sum(1, keepdim=True)
    size = sum(rows[:, i:i + 1000].double().abs().sum(1, keepdim=True) for i in range(0, ROWS, 1000))
    assert bool(((r["dshift"].double() - total).abs() <= (ROWS // 256 + 1300) * 2.0 ** -24 * size).all())   # a part's chain and the parts'


def test_rotation_and_its_gradient(gpu, rows):
    q = rows.view(1, ROWS, 64, 128).transpose(1, 2)
    f, pairs = block_ops.rope_frequencies((64, 64), device=gpu)
    pos = torch.stack([torch.arange(ROWS, device=gpu), torch.arange(ROWS, device=gpu) % 333], -1)
    y, _ = block_ops.axes_rope(q, None, pos, f, pairs, norm=True)
    d = block_ops.axes_rope_backward(q, None, pos, f, pairs, q, norm=True)[0]
    for a in SPANS:
        part = q[:, :, a:a + 300]
        same(y[:, :, a:a + 300], block_ops.axes_rope(part, None, pos[a:a + 300], f, pairs, norm=True)[0])
        same(d[:, :, a:a + 300], block_ops.axes_rope_backward(part, None, pos[a:a + 300], f, pairs, part, norm=True)[0])


def test_quantiser_and_product(gpu, rows):
    x8, s = block_ops.fp8_block_quant(rows[0])
    t8, ts = block_ops.fp8_block_quant(rows[0], 128)
    w, ws = block_ops.fp8_block_quant(torch.randn(320, C, device=gpu, generator=torch.Generator(device=gpu).manual_seed(1)), 128)
    y = block_ops.fp8_block_matmul(x8, s, w, ws)
    wide = torch.empty(ROWS, 8192, dtype=torch.bfloat16, device=gpu)
    block_ops.fp8_block_matmul(x8, s, w, ws, out=wide[:, 7800:8120])
    for a in (0, 131072, ROWS - ROWS % 128 - 256):
        part = rows[0, a:a + 256]
        p8, ps = block_ops.fp8_block_quant(part)
        same(x8[a:a + 256], p8)
        same(s[a:a + 256], ps)
        q8, qs = block_ops.fp8_block_quant(part, 128)
        same(t8[a:a + 256], q8)
        same(ts[a // 128:a // 128 + 2], qs)
        want = block_ops.fp8_block_matmul(p8, ps, w, ws)
        got = y[a:a + 256]
        # another plan may cut K: sums of 64 blocks in another order
        scale = want.double().abs().amax()
        assert float((got.double() - want.double()).abs().max()) <= 2.0 ** -7 * float(scale)
        same(wide[a:a + 256, 7800:8120], got)
    # the weight as the long operand
    ones, first = s.new_ones(2, C // 128), ROWS // 128 * 128 - 128
    full = block_ops.fp8_block_matmul(w[:2], ones, x8, ts)
    few = block_ops.fp8_block_matmul(w[:2], ones, x8[first:], ts[first // 128:])
    assert float((full[:, first:].double() - few.double()).abs().max()) <= 2.0 ** -7 * float(few.double().abs().max())
