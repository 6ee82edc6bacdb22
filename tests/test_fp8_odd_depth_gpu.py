"""Products on 256x256 tiles with an odd number of K blocks: infinities and NaN in the last block."""
import pytest
import torch

from dllm.ops import fp8
from test_fp8_gpu import rand

pytestmark = pytest.mark.gpu
DEV = "cuda"


def operands(M, N, nk, seed=1):
    """e5m2 rows with an infinity (both signs) and a NaN in the last block, against e4m3 rows whose codes there are the smallest
    (2^-9) and the largest ones, with ordinary blocks before them."""
    K = 128 * nk
    a, b = fp8.quantize_fp8(rand(M, K, seed).to(DEV), "e5m2"), fp8.quantize_fp8(rand(N, K, seed + 1).to(DEV))
    last = b.data.view(torch.uint8)[:, K - 128:]
    last.fill_(0x01)                                   # 2^-9
    last[1::3] = 0x81                                  # -2^-9
    last[2::3] = 0x7e                                  # 448
    rows = a.data.view(torch.uint8)
    rows[3, K - 5] = 0x7c                              # inf
    rows[M - 1, K - 100] = 0xfc                        # -inf
    rows[70, K - 128] = 0x7f                           # NaN
    return a, b


@pytest.mark.parametrize("nk", [1, 3, 5])
@pytest.mark.parametrize("swap", [False, True])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tile", [(256, 1), (128, 1), (64, 1)])
def test_infinity_in_the_last_block(monkeypatch, nk, swap, out, tile):
    a, b = operands(300, 290, nk)
    if swap:
        a, b = b, a
    monkeypatch.setattr(fp8, "_plan", lambda *_: tile)
    y = fp8.gemm_fp8(a, b, out_dtype=out).cpu()
    want = fp8.dequantize_fp8(a).cpu().double() @ fp8.dequantize_fp8(b).cpu().double().t()
    assert torch.isinf(want).sum() > 100 and torch.isnan(want).sum() > 100
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(y), inf) and torch.equal(y[inf].double(), want[inf])


def test_infinity_where_the_plan_takes_256_tiles():
    """As the plan chooses by itself: a whole round of 256x256 tiles, three K blocks, fp32 result."""
    M = N = 4096
    assert fp8._plan(M, N, 3, 1)[0] == 256
    a, b = operands(M, N, 3)
    y = fp8.gemm_fp8(a, b, out_dtype=torch.float32)
    want = fp8.dequantize_fp8(a) @ fp8.dequantize_fp8(b).t()
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(torch.isinf(y), torch.isinf(want))
    assert torch.isinf(want[3]).all() and torch.isinf(want[M - 1]).all() and torch.isnan(want[70]).all()
