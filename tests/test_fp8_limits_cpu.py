"""Sizes and row strides at the end of what the 8-bit products take: another kernel, or a refusal by name."""
import pytest
import torch

from dllm.ops import fp8

FAR = fp8.MAX_PITCH + 1
BF16, FP32 = 0, 1


def test_far_rows_take_the_kernel_for_few_rows():
    for out in (BF16, FP32):
        for M, N in ((40, 1000), (17, 17), (1000, 64), (64, 64)):
            for kb in (1, 8, 66000):
                assert fp8._plan(M, N, kb, out, FAR) == (0, 1)
        assert fp8._plan(40, 17000, 32, out)[0] == 64              # as near rows have it
        assert fp8._plan(100, 100, 0, out, FAR)[0] == 128           # without depth nothing is read


def test_far_rows_with_many_on_both_sides_are_refused():
    for M, N in ((65, 65), (100, 4096), (4096, 4096)):
        with pytest.raises(ValueError, match="bytes apart"):
            fp8._plan(M, N, 2, BF16, FAR)
    with pytest.raises(ValueError, match="bytes apart"):
        fp8._linear_workspace(100, FAR, 100, BF16)
    with pytest.raises(ValueError, match="bytes apart"):
        fp8._linear_bwd_workspace(100, 200, 300, BF16, FP32, FAR, 0)
    with pytest.raises(ValueError, match="bytes apart"):
        fp8._linear_bwd_workspace(100, 200, 300, -1, FP32, 0, FAR)
    assert fp8._linear_workspace(20, FAR, 100, BF16) > 20 * FAR
    assert fp8._linear_bwd_workspace(100, 200, 300, -1, FP32, FAR, 0) > 0      # (its wᵀ is not read)


def test_backward_without_dx_reserves_nothing_for_it():
    """The row-wise form of dy (T x F codes and their scales) and dx's K slices are needed for dx only."""
    def pad(n, to):
        return -(-n // to) * to

    for T, D, F in ((8192, 4096, 16384), (1000, 512, 1400), (1, 5, 7), (64, 4096, 16384)):
        columns = pad(F * pad(T, 128), 256) + pad(pad(T, 128) // 128 * F, 256)
        slices = fp8._plan(F, D, pad(T, 128) // 128, FP32)[1]
        assert fp8._linear_bwd_workspace(T, D, F, -1, FP32, 0, 0) == columns + (pad(4 * slices * F * D, 256) if slices > 1 else 0)
        assert fp8._linear_bwd_workspace(T, D, F, BF16, FP32, 0, 0) >= columns + T * pad(F, 128)


def test_more_rows_than_a_launch_counts_are_refused():
    top = 2 ** 27 - 16
    assert fp8._plan(1, top, 1, BF16) == (0, 1) and fp8._plan(top, 16, 1, FP32) == (0, 1)
    for M, N in ((1, top + 1), (top + 1, 16)):
        with pytest.raises(ValueError, match="rows on the other side"):
            fp8._plan(M, N, 1, BF16)


def test_pitch_limit_is_the_fetches_reach():
    """256 rows, and what one step of 128 bytes adds, stay below 2^31 bytes from the first."""
    assert 256 * fp8.MAX_PITCH + 4096 <= 2 ** 31 - 1 < 256 * (fp8.MAX_PITCH + 1) + 4096
    assert fp8._far(fp8.MAX_PITCH, 5) == 0 and fp8._far(7, FAR) == FAR


def test_one_target_for_both_orientations_is_refused():
    x, out, other = torch.randn(40, 40), fp8.fp8_empty(40, 40), fp8.fp8_empty(40, 40)
    for out_t in (out, out._replace(data=other.data), out._replace(scale=other.scale)):
        with pytest.raises(ValueError, match="share memory"):
            fp8.quantize_fp8_both(x, out=out, out_t=out_t)
    q, qt = fp8.quantize_fp8_both(x, out=out, out_t=other)
    assert torch.equal(fp8.dequantize_fp8(qt), fp8.dequantize_fp8(fp8.quantize_fp8(x.t())))
    none, none_t = fp8.quantize_fp8_both(torch.empty(0, 0))
    assert none.rows == none_t.rows == 0
