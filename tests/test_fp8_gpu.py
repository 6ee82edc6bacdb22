"""Block-scaled 8-bit operands on the GPU: codes and scales bit for bit against the CPU form, products against 64 bits."""
import pytest
import torch

from dllm.ops import fp8
from dllm.ops.activations import act_fwd, act_grad
from test_fp8_cpu import special_values

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rand(R, C, seed, dtype=torch.float32, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(R, C, generator=g) * torch.exp(spread * torch.randn(R, 1, generator=g))).to(dtype)


def same_operand(got, want):
    assert got.k == want.k and got.data.dtype == want.data.dtype
    assert torch.equal(got.scale.cpu(), want.scale)
    a, b = got.data.cpu().view(torch.uint8), want.data.view(torch.uint8)
    nan = lambda t, d: torch.isnan(d.float())  # noqa: E731  (a NaN's sign and payload are free)
    na, nb = nan(a, got.data.cpu()), nan(b, want.data)
    assert torch.equal(na, nb) and torch.equal(a[~na], b[~nb])


SIZES = [(1, 1), (1, 4096), (2, 129), (127, 128), (128, 127), (129, 257), (300, 1000), (1000, 77), (513, 640)]


@pytest.mark.parametrize("R,C", SIZES)
@pytest.mark.parametrize("tile", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fmt,fmt_t", [("e4m3", "e4m3"), ("e5m2", "e5m2"), ("e4m3", "e5m2")])
def test_quantize_bitwise(R, C, tile, dtype, fmt, fmt_t):
    x = rand(R, C, R + C, dtype, 2.0)
    xd = x.to(DEV)
    q, qt = fp8.quantize_fp8_both(xd, fmt, fmt_t, tile=tile)
    want, want_t = fp8.quantize_fp8(x, fmt, tile=tile), fp8.quantize_fp8_t(x, fmt_t, tile=tile)
    same_operand(q, want)
    same_operand(qt, want_t)
    same_operand(fp8.quantize_fp8(xd, fmt, tile=tile), want)
    same_operand(fp8.quantize_fp8_t(xd, fmt_t, tile=tile), want_t)
    for dt in (torch.float32, torch.bfloat16):
        assert torch.equal(fp8.dequantize_fp8(q, dt).cpu(), fp8.dequantize_fp8(want, dt))


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("tile", [False, True])
def test_quantize_special_values(fmt, tile):
    x = special_values()
    q, qt = fp8.quantize_fp8_both(x.to(DEV), fmt, fmt, tile=tile)
    same_operand(q, fp8.quantize_fp8(x, fmt, tile=tile))
    same_operand(qt, fp8.quantize_fp8_t(x, fmt, tile=tile))
    got, want = fp8.dequantize_fp8(q).cpu(), fp8.dequantize_fp8(fp8.quantize_fp8(x, fmt, tile=tile))
    assert torch.equal(torch.nan_to_num(got, nan=1.25e30), torch.nan_to_num(want, nan=1.25e30))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tile", [False, True])
@pytest.mark.parametrize("bits", [0x7f81, 0x7fc0, 0xff80, 0x0001])
def test_quantize_bit_patterns(dtype, tile, bits):
    """Signalling and quiet NaN, -inf and the smallest subnormal among ordinary values, in every position of a block's lanes:
    the block's scale and its other values are those of the CPU form."""
    x = rand(140, 260, 3, dtype)
    word = torch.tensor(bits << 16 if dtype == torch.float32 else bits, dtype=torch.int64)
    i = torch.arange(140)
    for c in (7, 70, 255):
        x.view(torch.int32 if dtype == torch.float32 else torch.int16)[i, (i + c) % 260] = \
            (word - 2 ** 32 if word >= 2 ** 31 else word).to(torch.int32) if dtype == torch.float32 else \
            (word - 2 ** 16 if word >= 2 ** 15 else word).to(torch.int16)
    for fmt in ("e4m3", "e5m2"):
        q, qt = fp8.quantize_fp8_both(x.to(DEV), fmt, fmt, tile=tile)
        same_operand(q, fp8.quantize_fp8(x, fmt, tile=tile))
        same_operand(qt, fp8.quantize_fp8_t(x, fmt, tile=tile))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_strided_and_misaligned(dtype):
    """Column slices (rows off the 16-byte grid), a transposed view, an expanded row, and writes that stay inside out."""
    base = rand(200, 300, 5, dtype)
    d = base.to(DEV)
    for cut in (slice(0, 299), slice(1, 300), slice(8, 264), slice(3, 4)):
        same_operand(fp8.quantize_fp8(d[:, cut]), fp8.quantize_fp8(base[:, cut].contiguous()))
        same_operand(fp8.quantize_fp8_t(d[3:, cut]), fp8.quantize_fp8_t(base[3:, cut].contiguous()))
    same_operand(fp8.quantize_fp8(d.t()), fp8.quantize_fp8(base.t().contiguous()))
    same_operand(fp8.quantize_fp8(d[:1].expand(5, 300)), fp8.quantize_fp8(base[:1].expand(5, 300).contiguous()))
    big = fp8.fp8_empty(210, 300, device=DEV)
    big.data.view(torch.uint8).fill_(7)
    big.scale.fill_(9)
    part = fp8.BlockFP8(big.data[5:205], big.scale[:, 5:205], 300)
    same_operand(fp8.quantize_fp8(d, out=part), fp8.quantize_fp8(base))
    rows = big.data.view(torch.uint8)
    assert (rows[:5] == 7).all() and (rows[205:] == 7).all() and (big.scale[:, :5] == 9).all() and (big.scale[:, 205:] == 9).all()


def product_check(got, qa, qb, alpha=1.0, beta=0.0, c=None, ref=None, mag_gain=1.0):
    """|error| <= K u sum|a||b| (any order of fp32 accumulation, u = 2^-24) + half an output step.  bf16 results come from the
    8-bit matrix instruction, which aligns the products of 8 neighbouring k to the largest and drops what lies under 2^-13
    of it: at most 7 of the 8 lose less than 2^-13 of the largest each, so less than 7 * 2^-13 of the group's sum|a||b|."""
    a, b = fp8.dequantize_fp8(qa).double().to(got.device), fp8.dequantize_fp8(qb).double().to(got.device)
    acc = a @ b.t()
    mag = abs(alpha) * (a.abs() @ b.abs().t())
    want = alpha * acc if ref is None else ref(acc)
    if beta:
        want = want + beta * c.double()
        mag = mag + abs(beta) * c.double().abs()
    u = 2.0 ** -24
    half = torch.finfo(got.dtype).eps / 2
    unit = (qa.k + 2) * u + (7 * 2.0 ** -13 if got.dtype == torch.bfloat16 else 0.0)
    tol = mag_gain * unit * mag + half * want.abs() * (1 + half) + 1e-38
    err = (got.double() - want).abs()
    assert (err <= tol).all(), f"worst {(err / tol).max().item():.3f} of the tolerance"


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 128, 128), (3, 5, 129), (16, 1000, 640), (64, 64, 256), (127, 129, 255),
                                   (128, 128, 384), (200, 333, 1537), (256, 256, 256), (300, 512, 2048), (512, 768, 1024),
                                   (1, 4096, 512), (33, 2000, 300), (1030, 260, 140), (65, 65, 100), (1000, 16, 700),
                                   (1000, 40, 1300), (17, 1000, 8200), (200, 70, 16500), (100, 100, 5000), (66, 513, 2500)])
@pytest.mark.parametrize("fa,fb", [("e4m3", "e4m3"), ("e5m2", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e5m2")])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_gemm(M, N, K, fa, fb, out):
    qa, qb = fp8.quantize_fp8(rand(M, K, 1).to(DEV), fa), fp8.quantize_fp8(rand(N, K, 2).to(DEV), fb, tile=True)
    product_check(fp8.gemm_fp8(qa, qb, out_dtype=out), qa, qb)
    c = rand(M, N, 3, out).to(DEV)
    c0 = c.clone()
    product_check(fp8.gemm_fp8(qa, qb, c, alpha=0.75, beta=-0.5), qa, qb, 0.75, -0.5, c0)


@pytest.mark.parametrize("M,N,K", [(5, 33000, 300), (40, 17000, 1000), (17000, 23, 1000), (50, 2049, 8200), (2817, 3001, 513), (33000, 5, 128), (4096, 2048, 256), (4, 32768, 640),
                                   (2900, 3100, 1100)])
@pytest.mark.parametrize("fa,fb", [("e4m3", "e4m3"), ("e5m2", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e5m2")])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_gemm_many_tiles(M, N, K, fa, fb, out):
    """Grids that fill the chip: the large-tile kernels, odd and even numbers of K blocks, edges in both directions."""
    qa, qb = fp8.quantize_fp8(rand(M, K, 1).to(DEV), fa), fp8.quantize_fp8(rand(N, K, 2).to(DEV), fb)
    buf = torch.full((M + 1, N), 5.0, dtype=out, device=DEV)
    product_check(fp8.gemm_fp8(qa, qb, buf[:M]), qa, qb)
    assert (buf[M] == 5).all()
    if fa == fb:
        c0 = buf[:M].clone()
        product_check(fp8.gemm_fp8(qa, qb, buf[:M], alpha=0.75, beta=-0.5), qa, qb, 0.75, -0.5, c0)
        h = torch.empty(M, N, dtype=out, device=DEV)
        a = fp8.gemm_fp8(qa, qb, out_dtype=out, epi="act", act="silu", aux_out=h)
        product_check(h, qa, qb)
        product_check(a, qa, qb, ref=lambda acc: act_fwd("silu", acc), mag_gain=1.13)
        d = fp8.gemm_fp8(qa, qb, out_dtype=out, epi="dact", act="silu", aux=h)
        product_check(d, qa, qb, ref=lambda acc: acc * act_grad("silu", h.double()), mag_gain=1.13)


@pytest.mark.parametrize("M,N,K", [(3, 70, 200), (256, 512, 256), (300, 300, 513)])
@pytest.mark.parametrize("act", ["relu", "silu", "gelu"])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_gemm_activation_epilogues(M, N, K, act, out):
    qa, qb = fp8.quantize_fp8(rand(M, K, 4, spread=0.3).to(DEV)), fp8.quantize_fp8(rand(N, K, 5, spread=0.3).to(DEV))
    h = torch.empty(M, N, dtype=out, device=DEV)
    a = fp8.gemm_fp8(qa, qb, out_dtype=out, epi="act", act=act, aux_out=h)
    product_check(h, qa, qb)
    # the activations' derivatives stay below 1.13 (silu 1.0999, gelu 1.129); their own fp32 evaluation adds a few ulp
    product_check(a, qa, qb, ref=lambda acc: act_fwd(act, acc), mag_gain=1.13)
    same = fp8.gemm_fp8(qa, qb, out_dtype=out, epi="act", act=act)
    assert torch.equal(a, same)
    got = fp8.gemm_fp8(qa, qb, out_dtype=out, epi="dact", act=act, aux=h)
    product_check(got, qa, qb, ref=lambda acc: acc * act_grad(act, h.double()), mag_gain=1.13)


def test_gemm_into_a_view_and_odd_strides():
    """out, aux and operands as slices of larger buffers; neighbours stay as they were."""
    qa, qb = fp8.quantize_fp8(rand(140, 260, 6).to(DEV)), fp8.quantize_fp8(rand(150, 260, 7).to(DEV))
    pa = fp8.BlockFP8(qa.data[3:133], qa.scale[:, 3:133], 260)
    pb = fp8.BlockFP8(qb.data[1:148], qb.scale[:, 1:148], 260)
    for ldc in (147, 149, 152, 160):
        for dt in (torch.bfloat16, torch.float32):
            buf = torch.full((132, ldc), 5.0, dtype=dt, device=DEV)
            product_check(fp8.gemm_fp8(pa, pb, buf[1:131, :147]), pa, pb)
            assert (buf[0] == 5).all() and (buf[131] == 5).all() and (buf[:, 147:] == 5).all()


def test_gemm_every_tile_and_slice(monkeypatch):
    """The plan's choices one by one on sizes that it would not choose them for."""
    for M, N, K in ((65, 70, 130), (300, 290, 1290), (257, 129, 2100)):
        qa, qb = fp8.quantize_fp8(rand(M, K, 1).to(DEV), "e5m2"), fp8.quantize_fp8(rand(N, K, 2).to(DEV))
        for tile, ksplit in ((64, 1), (128, 1), (256, 1), (64, 2), (128, 4), (64, 8), (128, 1)):
            if ksplit > 1 and K < 128 * ksplit:
                continue
            monkeypatch.setattr(fp8, "_plan", lambda *_: (tile, ksplit))
            for out in (torch.bfloat16, torch.float32):
                h = torch.empty(M, N, dtype=out, device=DEV)
                product_check(fp8.gemm_fp8(qa, qb, out_dtype=out), qa, qb)
                a = fp8.gemm_fp8(qa, qb, out_dtype=out, epi="act", act="relu", aux_out=h)
                product_check(h, qa, qb)
                assert torch.equal(a, h.clamp(min=0))


def test_gemm_no_depth():
    q, w = fp8.quantize_fp8(torch.empty(70, 0, device=DEV)), fp8.quantize_fp8(torch.empty(80, 0, device=DEV))
    assert torch.equal(fp8.gemm_fp8(q, w), torch.zeros(70, 80, dtype=torch.bfloat16, device=DEV))
    c = torch.ones(70, 80, device=DEV)
    assert torch.equal(fp8.gemm_fp8(q, w, c, beta=0.5), torch.full((70, 80), 0.5, device=DEV))
    one = fp8.quantize_fp8(torch.empty(1, 0, device=DEV))
    assert torch.equal(fp8.gemm_fp8(one, w), torch.zeros(1, 80, dtype=torch.bfloat16, device=DEV))


def test_single_row_with_arbitrary_strides():
    q = fp8.quantize_fp8(rand(6, 300, 11).to(DEV))
    for s in (q.scale[:, 2:3], q.scale[:, 2:3].t().contiguous().t()):
        one = fp8.BlockFP8(q.data[2:3], s, 300)
        product_check(fp8.gemm_fp8(one, q), one, q)
        product_check(fp8.gemm_fp8(q, one, out_dtype=torch.float32), q, one)
        assert torch.equal(fp8.dequantize_fp8(one), fp8.dequantize_fp8(q)[2:3])


def test_gemm_non_finite():
    """A NaN (or e5m2 infinity) reaches its row or column of the result only."""
    x, w = rand(130, 256, 8), rand(140, 256, 9)
    x[7, 200] = float("nan")
    x[9, 3] = float("inf")
    w[11, 130] = float("nan")
    qa, qb = fp8.quantize_fp8(x.to(DEV), "e5m2"), fp8.quantize_fp8(w.to(DEV))
    y = fp8.gemm_fp8(qa, qb, out_dtype=torch.float32).cpu()
    want = fp8.dequantize_fp8(qa).cpu().double() @ fp8.dequantize_fp8(qb).cpu().double().t()
    assert torch.equal(torch.isfinite(y), torch.isfinite(want)) and torch.equal(torch.isnan(y), torch.isnan(want))


@pytest.mark.parametrize("M,N", [(3, 70), (40, 90), (130, 300), (70, 5)])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_gemm_scale_nan(M, N, out):
    """Scale byte 255 stands for NaN: its block's row (column) of the result is NaN, the rest is untouched."""
    qa, qb = fp8.quantize_fp8(rand(M, 300, 8).to(DEV)), fp8.quantize_fp8(rand(N, 300, 9).to(DEV), "e5m2")
    clean = fp8.gemm_fp8(qa, qb, out_dtype=out)
    qa.scale[1, 2] = 255
    qb.scale[2, 4] = 255
    y = fp8.gemm_fp8(qa, qb, out_dtype=out)
    assert torch.isnan(y[2]).all() and torch.isnan(y[:, 4]).all() and torch.isnan(fp8.dequantize_fp8(qa)[2, 128:256]).all()
    rest = torch.ones(M, N, dtype=torch.bool, device=DEV)
    rest[2], rest[:, 4] = False, False
    assert torch.equal(y[rest], clean[rest])


def test_gemm_scale_extremes():
    """Scales from 2^-127 to 2^120: products far outside fp32 become 0 or inf as fp32 arithmetic would have them."""
    x = torch.cat([torch.full((20, 128), 1e-38), torch.full((20, 128), 1e30), torch.full((20, 128), 1.0),
                   torch.zeros(20, 128)])
    q = fp8.quantize_fp8(x.to(DEV))
    y = fp8.gemm_fp8(q, q, out_dtype=torch.float32).cpu().double()
    v = fp8.dequantize_fp8(q).cpu().double()
    want = v @ v.t()
    big, tiny = want.abs() > 3.4e38, want.abs() < 1.2e-38
    assert torch.isinf(y[big]).all() and (y[tiny].abs() < 1.2e-38).all()
    mid = ~big & ~tiny
    assert ((y - want).abs()[mid] <= 130 * 2.0 ** -24 * want[mid]).all()


@pytest.mark.parametrize("T,D,F", [(1, 33, 40), (200, 130, 257), (512, 256, 512)])
def test_linear(T, D, F):
    x, w, dy = rand(T, D, 1, torch.bfloat16), rand(F, D, 2, torch.bfloat16), rand(T, F, 3, torch.bfloat16)
    y, saved = fp8.linear_fp8(x.to(DEV), w.to(DEV))
    dx, dw = fp8.linear_fp8_bwd(dy.to(DEV), saved)
    product_check(y, fp8.quantize_fp8(x), fp8.quantize_fp8(w, tile=True))
    product_check(dx, fp8.quantize_fp8(dy, "e5m2"), fp8.quantize_fp8_t(w, tile=True))
    product_check(dw, fp8.quantize_fp8_t(dy, "e5m2"), fp8.quantize_fp8_t(x))
    assert dx.dtype == torch.bfloat16 and dw.dtype == torch.float32
    acc = dw.clone()
    assert fp8.linear_fp8_bwd(dy.to(DEV), saved, acc, beta=1.0, need_dx=False)[0] is None
    product_check(acc, fp8.quantize_fp8_t(dy, "e5m2"), fp8.quantize_fp8_t(x), beta=1.0, c=dw)


@pytest.mark.parametrize("T,D,F", [(1, 40, 33), (5, 1, 700), (333, 257, 129), (60, 2048, 4096), (1000, 512, 1400)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear_is_its_operators(T, D, F, dtype):
    """One call per direction, the bits of the separate calls; views in and out, either result type, no input gradient."""
    big = rand(T, D + 3, 1, dtype).to(DEV)
    x, w, dy = big[:, 1:D + 1], rand(D, F, 2, dtype).to(DEV).t(), rand(T, F, 3, dtype).to(DEV)
    xq, xt = fp8.quantize_fp8_both(x)
    wq, wt = fp8.quantize_fp8_both(w, tile=True)
    dq, dt = fp8.quantize_fp8_both(dy, "e5m2", "e5m2")
    for out in (torch.bfloat16, torch.float32):
        ybuf = torch.full((T, F + 5), 7.0, dtype=out, device=DEV)
        y, saved = fp8.linear_fp8(x, w, ybuf[:, 2:F + 2])
        assert torch.equal(y, fp8.gemm_fp8(xq, wq, out_dtype=out)) and (ybuf[:, :2] == 7).all() and (ybuf[:, F + 2:] == 7).all()
        same_operand(saved.x_t, fp8.BlockFP8(xt.data.cpu(), xt.scale.cpu(), T))
        same_operand(saved.w_t, fp8.BlockFP8(wt.data.cpu(), wt.scale.cpu(), F))
        acc = torch.ones(F, D, dtype=out, device=DEV)
        dx, dw = fp8.linear_fp8_bwd(dy, saved, acc, beta=0.5, dx=torch.empty(T, D, dtype=out, device=DEV))
        assert torch.equal(dx, fp8.gemm_fp8(dq, wt, out_dtype=out)) and dw is acc
        assert torch.equal(dw, fp8.gemm_fp8(dt, xt, torch.ones(F, D, dtype=out, device=DEV), beta=0.5))
    none, dw = fp8.linear_fp8_bwd(dy, saved, need_dx=False)
    assert none is None and torch.equal(dw, fp8.gemm_fp8(dt, xt, out_dtype=torch.float32))


def test_linear_captured_and_replayed():
    x, w, dy = (rand(r, c, i, torch.bfloat16).to(DEV) for i, (r, c) in enumerate(((200, 300), (500, 300), (200, 500))))

    def step():
        y, saved = fp8.linear_fp8(x, w)
        return (y, *fp8.linear_fp8_bwd(dy, saved))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        x.copy_(rand(200, 300, 20 + i))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_other_stream_and_graph():
    """The same bits on another stream, from a captured graph on replayed new inputs, and from the batch-size-one slice."""
    x, w = rand(300, 400, 1, torch.bfloat16).to(DEV), rand(200, 400, 2, torch.bfloat16).to(DEV)
    y0, _ = fp8.linear_fp8(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y1, _ = fp8.linear_fp8(x, w)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y0, y1)
    xs, dys = x.clone(), rand(300, 200, 3, torch.bfloat16).to(DEV)
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        graph.capture_begin()
        yg, saved = fp8.linear_fp8(xs, w)
        dxg, dwg = fp8.linear_fp8_bwd(dys, saved)
        graph.capture_end()
    torch.cuda.current_stream().wait_stream(s)
    for seed in (10, 11, 12):
        xn, dyn = rand(300, 400, seed, torch.bfloat16).to(DEV), rand(300, 200, seed + 50, torch.bfloat16).to(DEV)
        xs.copy_(xn)
        dys.copy_(dyn)
        graph.replay()
        y, sv = fp8.linear_fp8(xn, w)
        dx, dw = fp8.linear_fp8_bwd(dyn, sv)
        torch.cuda.synchronize()
        assert torch.equal(yg, y) and torch.equal(dxg, dx) and torch.equal(dwg, dw)


def test_repeats_are_bitwise():
    qa, qb = fp8.quantize_fp8(rand(260, 3000, 1).to(DEV)), fp8.quantize_fp8(rand(270, 3000, 2).to(DEV))
    first = fp8.gemm_fp8(qa, qb, out_dtype=torch.float32)
    for _ in range(3):
        assert torch.equal(first, fp8.gemm_fp8(qa, qb, out_dtype=torch.float32))


def test_misaligned_operand_is_refused():
    q = fp8.quantize_fp8(torch.randn(4, 256, device=DEV))
    flat = torch.empty(4 * 256 + 8, dtype=torch.uint8, device=DEV)[8:].view(4, 256).view(torch.float8_e4m3fn)
    with pytest.raises(ValueError, match="multiples of 16"):
        fp8.gemm_fp8(q._replace(data=flat), q)
    with pytest.raises(ValueError, match="operands on"):
        fp8.gemm_fp8(q, fp8.quantize_fp8(torch.randn(4, 256)))
