"""The block-scaled product over operands and results of more than 2^31 elements, every row and element held to its own size.

Rows differ in scale by up to 2^40, so a scale or a piece of the wrong row shows whatever the size of the rows around it; bars as for small products."""
import pytest
import torch

from test_gpu_block_fp8 import check
from xdit_amd import block_ops

pytestmark = pytest.mark.gpu
ROWS, K = 275000, 8192    # row 262144 starts at byte 2^31
SPANS = (0, 262144 - 128, ROWS // 128 * 128 - 128)


def values(g, rows, gpu):
    return torch.randn(rows, K, generator=g, device=gpu).clamp(-4, 4).mul_(100).to(torch.float8_e4m3fn)


@pytest.fixture(scope="module")
def operands(gpu):
    g = torch.Generator(device=gpu).manual_seed(11)
    long = torch.empty(ROWS, K, dtype=torch.float8_e4m3fn, device=gpu)
    tile = values(g, 1000, gpu).view(torch.uint8)
    for i in range(0, ROWS, 1000):
        long[i:i + 1000].view(torch.uint8).copy_(tile.roll(i // 1000, -1)[:min(1000, ROWS - i)])
    row_scale = torch.exp2(torch.randint(-30, 10, (ROWS, 1), generator=g, device=gpu).float()) * (1 + torch.rand(ROWS, K // 128, generator=g, device=gpu))
    block_scale = torch.exp2(torch.randint(-30, 10, (-(-ROWS // 128), 1), generator=g, device=gpu).float()) * (1 + torch.rand(-(-ROWS // 128), K // 128, generator=g, device=gpu))
    yield g, long, row_scale, block_scale
    torch.cuda.empty_cache()


def test_many_rows(gpu, operands):
    g, x, xs, _ = operands
    w, ws = block_ops.fp8_block_quant(torch.randn(320, K, generator=g, device=gpu), 128)
    out = torch.empty(ROWS, 8192, dtype=torch.bfloat16, device=gpu)
    y = block_ops.fp8_block_matmul(x, xs, w, ws, out=out[:, 7800:8120])
    for a in SPANS:
        at = slice(a, min(ROWS, a + 256))
        check(y[at], x[at], xs[at], w, ws, None, False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_long_weight(gpu, operands, dtype):
    g, w, _, ws = operands
    x, xs = block_ops.fp8_block_quant(torch.randn(3, K, generator=g, device=gpu))
    y = block_ops.fp8_block_matmul(x, xs, w, ws, out_dtype=dtype)
    for a in SPANS:
        at = slice(a, min(ROWS, a + 256))
        check(y[:, at], x, xs, w[at], ws[a // 128:a // 128 + 2], None, dtype == torch.float32)
