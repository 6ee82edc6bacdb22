"""Block-scaled 8-bit operands: the format, the CPU forms, and every refusal (the checks are shared with the GPU path)."""
import math

import pytest
import torch

from dllm.ops import fp8

FMAX = {"e4m3": 448.0, "e5m2": 57344.0}
GRID = {"e4m3": (3, -6), "e5m2": (2, -14)}   # mantissa bits, smallest normal exponent


def grid_round(v: float, fmt: str) -> float:
    """Nearest number of the 8-bit grid, ties to even (the definition, in Python floats)."""
    bits, low = GRID[fmt]
    if v == 0 or math.isnan(v) or math.isinf(v):
        return v
    step = 2.0 ** (max(math.frexp(abs(v))[1] - 1, low) - bits)
    return round(v / step) * step


def block_exponent(vals, fmt: str) -> int:
    amax = max((abs(v) for v in vals if math.isfinite(v)), default=0.0)
    e = -127
    while amax > FMAX[fmt] * 2.0 ** e:
        e += 1
    return e


def oracle(x: torch.Tensor, fmt: str, tile: bool):
    """(values, exponents [k blocks][rows]) from the definition, element by element in 64 bits."""
    R, K = x.shape
    xs = x.double().tolist()
    kb = -(-K // 128)
    val = torch.zeros(R, K, dtype=torch.float64)
    ex = torch.zeros(kb, R, dtype=torch.int64)
    for b in range(kb):
        cols = range(128 * b, min(K, 128 * b + 128))
        for r0 in range(0, R, 128 if tile else 1):
            rows = range(r0, min(R, r0 + (128 if tile else 1)))
            e = block_exponent([xs[r][c] for r in rows for c in cols], fmt)
            for r in rows:
                ex[b, r] = e + 127
                for c in cols:
                    v = grid_round(xs[r][c] * 2.0 ** -e, fmt) if math.isfinite(xs[r][c]) else xs[r][c]
                    if fmt == "e4m3" and math.isinf(v):
                        v = math.nan
                    val[r, c] = v * 2.0 ** e if math.isfinite(v) else v
    return val, ex


def check_operand(q, x, fmt, tile):
    val, ex = oracle(x.cpu(), fmt, tile)
    assert torch.equal(q.scale.cpu().long(), ex)
    got = fp8.dequantize_fp8(q).double().cpu()
    val = val.float().double()   # read back in fp32: 3.3e38 rounds up to 2^128, which fp32 holds as inf only
    assert got.shape == val.shape and torch.equal(torch.nan_to_num(got, nan=1.25e30), torch.nan_to_num(val, nan=1.25e30))
    assert not q.data.cpu().float()[:, q.k:].any()   # zeros behind k


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("tile", [False, True])
@pytest.mark.parametrize("R,K", [(1, 1), (3, 130), (129, 127), (5, 256)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_matches_definition(fmt, tile, R, K, dtype):
    g = torch.Generator().manual_seed(R * 1000 + K)
    x = (torch.randn(R, K, generator=g) * torch.exp(2 * torch.randn(R, 1, generator=g))).to(dtype)
    check_operand(fp8.quantize_fp8(x, fmt, tile=tile), x, fmt, tile)
    check_operand(fp8.quantize_fp8_t(x, fmt, tile=tile), x.t(), fmt, tile)
    q, qt = fp8.quantize_fp8_both(x, fmt, "e5m2", tile=tile)
    check_operand(q, x, fmt, tile)
    check_operand(qt, x.t(), "e5m2", tile)


def special_values() -> torch.Tensor:
    """Blocks of zeros, subnormals, the largest numbers, values on and next to the format's borders, inf and NaN."""
    x = torch.zeros(12, 130)
    x[1] = 1e-42
    x[2] = 3.3e38
    x[3, :4] = torch.tensor([448.0, 448.0 * (1 + 2.0 ** -23), -448.0, 1.0])
    x[4, :3] = torch.tensor([57344.0, -57344.0 * (1 + 2.0 ** -23), 1.0])
    x[5, :3] = torch.tensor([float("nan"), 2.0, -3.0])
    x[6, :3] = torch.tensor([float("inf"), 2.0, -float("inf")])
    x[7] = float("nan")
    x[8] = float("inf")
    x[9, :6] = torch.tensor([17.0, 18.0, 19.0, 21.0, 22.0, 448.0])       # ties of the 3-bit mantissa
    x[10, :5] = torch.tensor([2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -9, 2.0 ** -7, 256.0])   # ties among e4m3 subnormals
    x[11, 129] = -0.0
    return x


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("tile", [False, True])
def test_quantize_special_values(fmt, tile):
    x = special_values()
    check_operand(fp8.quantize_fp8(x, fmt, tile=tile), x, fmt, tile)
    check_operand(fp8.quantize_fp8_t(x, fmt, tile=tile), x.t(), fmt, tile)


def test_empty_operands():
    q = fp8.quantize_fp8(torch.empty(0, 5))
    assert q.data.shape == (0, 128) and q.scale.shape == (1, 0) and fp8.dequantize_fp8(q).shape == (0, 5)
    z = fp8.quantize_fp8(torch.empty(4, 0))
    assert z.data.shape == (4, 0) and fp8.dequantize_fp8(z).shape == (4, 0)
    assert fp8.gemm_fp8(q, fp8.quantize_fp8(torch.ones(3, 5))).shape == (0, 3)
    out = fp8.gemm_fp8(z, fp8.quantize_fp8(torch.empty(2, 0)), torch.ones(4, 2), beta=0.5)
    assert torch.equal(out, torch.full((4, 2), 0.5))


def test_single_row_with_arbitrary_strides():
    """torch leaves the strides of a dimension of size one open: a transposed or sliced single row is an operand too."""
    q = fp8.quantize_fp8(torch.randn(6, 300))
    one = fp8.BlockFP8(q.data[2:3], q.scale[:, 2:3].t().contiguous().t(), 300)
    torch.testing.assert_close(fp8.gemm_fp8(one, q, out_dtype=torch.float32), fp8.gemm_fp8(q, q, out_dtype=torch.float32)[2:3])
    assert torch.equal(fp8.dequantize_fp8(one), fp8.dequantize_fp8(q)[2:3])


def test_gemm_epilogues():
    g = torch.Generator().manual_seed(2)
    a, b = torch.randn(7, 200, generator=g), torch.randn(5, 200, generator=g)
    qa, qb = fp8.quantize_fp8(a), fp8.quantize_fp8(b, "e5m2")
    acc = fp8.dequantize_fp8(qa) @ fp8.dequantize_fp8(qb).t()
    torch.testing.assert_close(fp8.gemm_fp8(qa, qb, out_dtype=torch.float32, alpha=0.5), 0.5 * acc)
    c = torch.ones(7, 5)
    torch.testing.assert_close(fp8.gemm_fp8(qa, qb, c, beta=2.0), acc + 2.0)
    h = torch.empty(7, 5)
    torch.testing.assert_close(fp8.gemm_fp8(qa, qb, out_dtype=torch.float32, epi="act", act="relu", aux_out=h),
                               acc.clamp(min=0))
    assert torch.equal(h, acc)
    torch.testing.assert_close(fp8.gemm_fp8(qa, qb, out_dtype=torch.float32, epi="dact", act="relu", aux=h), acc * (h > 0))


def test_linear_gradients_against_formula_and_differences():
    """linear_fp8's gradients are those of the product of the quantised operands; differences along x and w see them as long
    as the 8-bit rounding (half a step, 2^-4 relative e4m3, 2^-3 e5m2) stays below the tolerance."""
    g = torch.Generator().manual_seed(3)
    T, D, F = 40, 24, 30
    x, w, dy = torch.randn(T, D, generator=g), torch.randn(F, D, generator=g), torch.randn(T, F, generator=g)
    y, saved = fp8.linear_fp8(x, w, out_dtype=torch.float32)
    dx, dw = fp8.linear_fp8_bwd(dy, saved)
    wq = fp8.dequantize_fp8(saved.w_t).t()
    xq = fp8.dequantize_fp8(saved.x_t).t()
    torch.testing.assert_close(dx, fp8.dequantize_fp8(fp8.quantize_fp8(dy, "e5m2")) @ wq)
    torch.testing.assert_close(dw, fp8.dequantize_fp8(fp8.quantize_fp8_t(dy, "e5m2")) @ xq)
    # against differences of the unquantised loss <dy, x w^T> along a direction: three operands rounded, relative error of
    # each product at most 2^-3 + 2^-4 + 2^-7, summed in absolute value
    vx, vw = torch.randn(T, D, generator=g), torch.randn(F, D, generator=g)
    loss = lambda x_, w_: (dy.double() * (x_.double() @ w_.double().t())).sum()  # noqa: E731
    h = 1e-3
    for grad, num, mag in ((dx, (loss(x + h * vx, w) - loss(x - h * vx, w)) / (2 * h), (dy.abs() @ w.abs() * vx.abs()).sum()),
                           (dw, (loss(x, w + h * vw) - loss(x, w - h * vw)) / (2 * h),
                            (dy.abs().t() @ x.abs() * vw.abs()).sum())):
        v = vx if grad is dx else vw
        assert abs((grad.double() * v.double()).sum() - num) <= (2.0 ** -3 + 2.0 ** -4 + 2.0 ** -7) * mag
    acc = dw.clone()
    fp8.linear_fp8_bwd(dy, saved, acc, beta=1.0, need_dx=False)
    torch.testing.assert_close(acc, 2 * dw)


def test_refusals():
    x = torch.randn(4, 200)
    q = fp8.quantize_fp8(x)
    with pytest.raises(ValueError, match="unknown 8-bit format"):
        fp8.quantize_fp8(x, "e3m4")
    with pytest.raises(TypeError, match="2-D bf16 or fp32"):
        fp8.quantize_fp8(x.half())
    with pytest.raises(TypeError, match="2-D bf16 or fp32"):
        fp8.quantize_fp8(x[0])
    for shape in ((2 ** 31, 1), (1, 2 ** 31)):
        with pytest.raises(ValueError, match="rows and columns"):
            fp8.quantize_fp8(torch.zeros(1, 1).expand(shape))
    with pytest.raises(ValueError, match="must hold"):
        fp8.quantize_fp8(x, out=fp8.fp8_empty(4, 100))
    with pytest.raises(TypeError, match="float8"):
        fp8.dequantize_fp8(q._replace(data=q.data.view(torch.uint8)))
    with pytest.raises(ValueError, match="columns"):
        fp8.dequantize_fp8(q._replace(k=300))
    with pytest.raises(ValueError, match="scale must be"):
        fp8.dequantize_fp8(q._replace(scale=q.scale[:, :3]))
    with pytest.raises(ValueError, match="contiguous along"):
        fp8.dequantize_fp8(q._replace(scale=q.scale.t().contiguous().t()))
    for bad in (q._replace(data=q.data[:1].expand(q.rows, -1)), q._replace(scale=q.scale[:1].expand(len(q.scale), -1))):
        if bad.data.stride(0) == 0 or len(bad.scale) > 1:          # one row standing for all: the kernels step over rows
            with pytest.raises(ValueError, match="overlapping rows"):
                fp8.dequantize_fp8(bad)
    with pytest.raises(ValueError, match="out must be"):
        fp8.dequantize_fp8(q, out=torch.empty(4, 100))
    with pytest.raises(ValueError, match="inner dims"):
        fp8.gemm_fp8(q, fp8.quantize_fp8(torch.randn(4, 100)))
    with pytest.raises(ValueError, match="beta needs out"):
        fp8.gemm_fp8(q, q, beta=1.0)
    with pytest.raises(TypeError, match="bf16 or fp32"):
        fp8.gemm_fp8(q, q, torch.empty(4, 4, dtype=torch.float16))
    with pytest.raises(ValueError, match="out must be"):
        fp8.gemm_fp8(q, q, torch.empty(4, 5))
    with pytest.raises(ValueError, match="row-major"):
        fp8.gemm_fp8(q, fp8.quantize_fp8(torch.randn(6, 200)), torch.empty(6, 4).t())
    with pytest.raises(ValueError, match="row-major"):
        fp8.gemm_fp8(q, q, torch.empty(1, 4).expand(4, 4))
    with pytest.raises(ValueError, match="unknown epilogue"):
        fp8.gemm_fp8(q, q, epi="sgd")
    with pytest.raises(ValueError, match="needs an activation"):
        fp8.gemm_fp8(q, q, epi="act")
    with pytest.raises(ValueError, match="unknown activation"):
        fp8.gemm_fp8(q, q, epi="act", act="tanh")
    with pytest.raises(ValueError, match="needs aux"):
        fp8.gemm_fp8(q, q, epi="dact", act="relu")
    with pytest.raises(ValueError, match="no alpha"):
        fp8.gemm_fp8(q, q, epi="act", act="relu", alpha=2.0)
    with pytest.raises(ValueError, match="aux belongs"):
        fp8.gemm_fp8(q, q, aux=torch.empty(4, 4))
    with pytest.raises(TypeError, match="output dtype"):
        fp8.gemm_fp8(q, q, epi="act", act="relu", aux_out=torch.empty(4, 4))
    with pytest.raises(ValueError, match="x \\[T, D\\]"):
        fp8.linear_fp8(torch.randn(3, 4), torch.randn(5, 6))
    _, saved = fp8.linear_fp8(torch.randn(3, 4), torch.randn(5, 4))
    y, saved = fp8.linear_fp8(torch.randn(3, 5), torch.randn(7, 5))
    for kw in ({"beta": 1.0}, {"dx": torch.empty(3, 5), "need_dx": False}):
        with pytest.raises(ValueError, match="beta needs dw|need_dx"):
            fp8.linear_fp8_bwd(y.float(), saved, **kw)
    with pytest.raises(ValueError, match="dy must be"):
        fp8.linear_fp8_bwd(torch.randn(3, 4), saved)
