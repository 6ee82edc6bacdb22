"""8-bit products of operands whose rows lie far apart."""
import pytest
import torch

from dllm.ops import fp8
from test_fp8_gpu import rand

pytestmark = pytest.mark.gpu
DEV = "cuda"
PITCH = (fp8.MAX_PITCH // 128 + 1) * 128


def far(q: fp8.BlockFP8) -> fp8.BlockFP8:
    """The operand as the first columns of a very wide buffer."""
    buf = torch.empty(q.rows, PITCH, dtype=q.data.dtype, device=DEV)
    view = buf[:, :q.data.shape[1]]
    view.copy_(q.data)
    return fp8.BlockFP8(view, q.scale, q.k)


@pytest.mark.parametrize("M,N", [(20, 100), (64, 17), (300, 40)])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_far_rows(monkeypatch, M, N, out):
    a, b = fp8.quantize_fp8(rand(M, 300, 1).to(DEV), "e5m2"), fp8.quantize_fp8(rand(N, 300, 2).to(DEV))
    got = [fp8.gemm_fp8(x, y, out_dtype=out) for x, y in ((far(a), b), (a, far(b)))]
    monkeypatch.setattr(fp8, "_plan", lambda *_: (0, 1))
    want = fp8.gemm_fp8(a, b, out_dtype=out)
    assert all(torch.equal(t, want) for t in got)


def test_far_rows_on_both_sides_are_refused():
    a, b = fp8.quantize_fp8(rand(100, 256, 1).to(DEV)), fp8.quantize_fp8(rand(90, 256, 2).to(DEV))
    with pytest.raises(ValueError, match="bytes apart"):
        fp8.gemm_fp8(far(a), b)
    y, saved = fp8.linear_fp8(rand(100, 90, 3).to(DEV), rand(110, 90, 4).to(DEV))
    dy = rand(100, 110, 5).to(DEV)
    with pytest.raises(ValueError, match="bytes apart"):
        fp8.linear_fp8_bwd(dy, saved._replace(w_t=far(saved.w_t)))
    with pytest.raises(ValueError, match="bytes apart"):
        fp8.linear_fp8_bwd(dy, saved._replace(x_t=far(saved.x_t)), need_dx=False)
    want = fp8.linear_fp8_bwd(dy, saved, need_dx=False)[1]
    assert torch.equal(fp8.linear_fp8_bwd(dy, saved._replace(w_t=far(saved.w_t)), need_dx=False)[1], want)


def test_linear_of_very_long_rows():
    """A depth whose 8-bit rows lie far apart, few tokens: both directions are their separate operators."""
    T, D, F = 20, PITCH, 70
    x, w = (torch.randn(r, D, device=DEV).bfloat16() for r in (T, F))
    dy = torch.randn(T, F, device=DEV).bfloat16()
    y, saved = fp8.linear_fp8(x, w)
    xq, wq = fp8.quantize_fp8(x), fp8.quantize_fp8(w, tile=True)
    assert torch.equal(y, fp8.gemm_fp8(xq, wq))
    dx, dw = fp8.linear_fp8_bwd(dy, saved)
    dq, dt = fp8.quantize_fp8_both(dy, "e5m2", "e5m2")
    assert torch.equal(dx, fp8.gemm_fp8(dq, saved.w_t)) and torch.equal(dw, fp8.gemm_fp8(dt, saved.x_t, out_dtype=torch.float32))
    v, u = fp8.dequantize_fp8(xq).double(), fp8.dequantize_fp8(wq).double()
    want, mag = v @ u.t(), v.abs() @ u.abs().t()
    # the 8-bit instruction's groups of 8 lose less than 7 * 2^-13 of their sum |a||b|; D fp32 additions in 8 waves' chains of 32
    # instructions' sums each round by 2^-24 of the running sum, at most D / 8 / 32 of them; half a step of bf16
    assert ((y.double() - want).abs() <= (7 * 2.0 ** -13 + D / 256 * 2.0 ** -24) * mag + 2.0 ** -8 * want.abs()).all()
    with pytest.raises(ValueError, match="bytes apart"):
        fp8.linear_fp8(w, w)


@pytest.mark.parametrize("tile", [(256, 1), (128, 1), (64, 2)])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_farthest_rows_of_the_tiles(monkeypatch, tile, out):
    """Row strides at the limit: a tile's last row lies just below 2^31 bytes from its first."""
    pitch = fp8.MAX_PITCH // 128 * 128
    a, b = fp8.quantize_fp8(rand(300, 512, 1).to(DEV), "e5m2"), fp8.quantize_fp8(rand(270, 512, 2).to(DEV))
    monkeypatch.setattr(fp8, "_plan", lambda *_: tile)
    want = fp8.gemm_fp8(a, b, out_dtype=out)
    wide = []
    for q in (a, b):
        buf = torch.empty(q.rows, pitch, dtype=q.data.dtype, device=DEV)
        buf[:, :512].copy_(q.data)
        wide.append(fp8.BlockFP8(buf[:, :512], q.scale, q.k))
    assert torch.equal(fp8.gemm_fp8(wide[0], wide[1], out_dtype=out), want)
