"""Newton-Schulz orthogonalisation and the Muon step on the GPU against 64 bits."""
import math

import pytest
import torch

from dllm.ops import muon
from dllm.ops.master import join_master, split_master
from test_muon_cpu import exact, relerr

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gradient(R, C, seed, kind="lowrank", batch=None):
    """Normal matrices, and gradient-like ones: few strong directions over noise (singular values over three decades)."""
    g = torch.Generator().manual_seed(seed)
    shape = (R, C) if batch is None else (batch, R, C)
    x = torch.randn(shape, generator=g)
    if kind == "lowrank":
        r = max(1, min(R, C) // 8)
        u = torch.randn((*shape[:-1], r), generator=g)
        v = torch.randn((*shape[:-2], r, C), generator=g)
        x = u @ v + 0.02 * x
    return x * 1e-3


def tolerance(x, steps=5, dtype=torch.float32):
    """Operands of 22 bits where the fp32 form has 24: at most four times the fp32 form's own error (a floor of 8 half
    steps of 22 bits where that error happens to vanish), plus half a step of the output."""
    ref = exact(x, steps)
    fp32 = relerr(muon._newton_schulz_torch(x.float(), steps, muon.NS_EPS), ref)
    return 4 * fp32 + 8 * 2.0 ** -23 + (torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0), ref


SIZES = [(1, 1), (1, 200), (200, 1), (16, 16), (101, 300), (300, 101), (128, 128), (129, 257), (256, 512), (640, 384),
         (64, 2000), (512, 512), (700, 1500), (1500, 700)]


@pytest.mark.parametrize("R,C", SIZES)
@pytest.mark.parametrize("kind", ["normal", "lowrank"])
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 5, 7])
def test_orthogonalize(R, C, kind, steps):
    x = gradient(R, C, R + C + steps, kind)
    tol, ref = tolerance(x, steps)
    got = muon.orthogonalize(x.to(DEV), steps)
    assert relerr(got, ref) <= tol


@pytest.mark.parametrize("R,C", [(300, 101), (256, 512)])
def test_orthogonalize_types_and_views(R, C):
    x = gradient(R, C, 3).bfloat16()
    tol, ref = tolerance(x.float(), 5, torch.bfloat16)
    d = x.to(DEV)
    out = muon.orthogonalize(d)
    assert out.dtype == torch.bfloat16 and relerr(out, ref) <= tol
    f = muon.orthogonalize(d, out=torch.empty(R, C, device=DEV))
    assert relerr(f, ref) <= tolerance(x.float())[0]
    wide = torch.zeros(R, C + 5, dtype=torch.bfloat16, device=DEV)
    wide[:, 2:C + 2] = d
    assert torch.equal(muon.orthogonalize(wide[:, 2:C + 2]), out)
    assert torch.equal(muon.orthogonalize(d.t().contiguous().t()), out)
    alias = d.clone()
    assert torch.equal(muon.orthogonalize(alias, out=alias), out) and torch.equal(alias, out)


def test_batch_is_bitwise_the_single_matrix():
    x = gradient(130, 260, 4, batch=3).to(DEV)
    out = muon.orthogonalize(x)
    for i in range(3):
        assert torch.equal(out[i], muon.orthogonalize(x[i]))
    assert torch.equal(out, muon.orthogonalize(x))


@pytest.mark.parametrize("R,C", [(200, 3000), (400, 2100)])
def test_batch_of_sliced_grams_is_bitwise_the_single_matrix(R, C):
    x = gradient(R, C, 4, batch=3).to(DEV)
    got = muon.orthogonalize(x)
    for i in range(3):
        assert torch.equal(got[i], muon.orthogonalize(x[i]))


def test_magnitudes_and_non_finite():
    """The result does not depend on the update's magnitude until eps = 1e-7 counts; zero stays zero; NaN and inf spoil their
    own matrix of a batch and no other."""
    x = gradient(96, 160, 5) * 1e3
    ref = muon.orthogonalize(x.to(DEV))
    for s in (2.0 ** 100, 2.0 ** 20):
        assert relerr(muon.orthogonalize((x * s).to(DEV)), ref.double().cpu()) <= 2.0 ** -18
    assert torch.equal(muon.orthogonalize(torch.zeros(40, 70, device=DEV)), torch.zeros(40, 70, device=DEV))
    b = torch.stack([x, x, x])
    b[1, 3, 5] = float("nan")
    b[2, 90, 100] = float("inf")
    out = muon.orthogonalize(b.to(DEV))
    assert torch.equal(out[0], ref) and torch.isnan(out[1]).all() and torch.isnan(out[2]).all()


@pytest.mark.parametrize("B,R,C", [(None, 64, 256), (None, 300, 101), (2, 129, 65)])
@pytest.mark.parametrize("gdt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step(B, R, C, gdt, nesterov):
    grad = gradient(R, C, 6, batch=B).to(gdt)
    mom, w = gradient(R, C, 7, batch=B) * 10, torch.randn((R, C) if B is None else (B, R, C), generator=torch.Generator().manual_seed(8))
    copy = torch.empty(w.shape, dtype=torch.bfloat16, device=DEV)
    wd, md = w.to(DEV), mom.to(DEV)
    hi, lo = (t.to(DEV) for t in split_master(w))
    ms = mom.to(DEV)
    kw = dict(lr=0.05, beta=0.9, nesterov=nesterov, wd=0.1, grad_scale=0.5)
    muon.muon_step_(wd, grad.to(DEV), md, copy=copy, **kw)
    muon.muon_split_step_(lo, hi, grad.to(DEV), ms, **kw)
    g = 0.5 * grad.double()
    m = 0.9 * mom.double() + g
    u = g + 0.9 * m if nesterov else m
    # momentum: two fp32 roundings of terms no larger than |0.9 m| + |g|
    assert ((md.double().cpu() - m).abs() <= 2 * 2.0 ** -24 * (0.9 * mom.double().abs() + g.abs())).all()
    rate = 0.05 * math.sqrt(max(1.0, R / C))
    for i in range(B or 1):
        ui = u if B is None else u[i]
        tol, o = tolerance(ui.float())
        # u itself is rounded to fp32 (2^-24 of its terms), which enters like one more rounding of the first step
        wi = w if B is None else w[i]
        want = wi.double() * (1 - 0.05 * 0.1) - rate * o
        err = (torch.linalg.norm((wd if B is None else wd[i]).double().cpu() - want)).item()
        assert err <= 2 * tol * rate * torch.linalg.norm(o).item() + 3 * 2.0 ** -24 * torch.linalg.norm(want).item()
    assert torch.equal(copy, wd.bfloat16())
    assert torch.equal(join_master(hi.cpu(), lo.cpu()), wd.cpu()) and torch.equal(ms, md)


def test_rows_behind_the_matrix_stay():
    """Views into larger flat buffers (the engine's): nothing outside the matrix is written."""
    n = 70 * 130
    flat = {k: torch.full((n + 300,), 3.0, device=DEV) for k in ("w", "m", "g")}
    flat["c"] = torch.full((n + 300,), 3.0, device=DEV, dtype=torch.bfloat16)
    view = {k: v[64:64 + n].view(70, 130) for k, v in flat.items()}
    for k, s in (("w", 1), ("m", 2), ("g", 3)):
        view[k].copy_(gradient(70, 130, s))
    muon.muon_step_(view["w"], view["g"], view["m"], lr=0.1, copy=view["c"])
    for v in flat.values():
        assert (v[:64] == 3).all() and (v[64 + n:] == 3).all()


def test_other_stream_and_graph():
    x = gradient(200, 333, 9).to(DEV)
    want = muon.orthogonalize(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = muon.orthogonalize(x)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    g, w, m = x.clone(), torch.randn(200, 333, device=DEV), torch.zeros(200, 333, device=DEV)
    we, me = w.clone(), m.clone()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        graph.capture_begin()
        muon.muon_step_(w, g, m, lr=0.02)
        graph.capture_end()
    torch.cuda.current_stream().wait_stream(s)
    for seed in (20, 21, 22):
        gn = gradient(200, 333, seed).to(DEV)
        g.copy_(gn)
        graph.replay()
        muon.muon_step_(we, gn, me, lr=0.02)
        torch.cuda.synchronize()
        assert torch.equal(w, we) and torch.equal(m, me)


@pytest.mark.parametrize("R,C", [(4096, 4224), (8192, 4096), (2900, 3100), (1024, 8200), (2048, 2048), (1300, 1300), (200, 5000),
                                 (5000, 260), (511, 2050), (150, 30000)])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_orthogonalize_large(R, C, out):
    """Sizes that take the larger tiles, against the iteration in 64 bits; memory that the workspace may get holds NaN."""
    x = gradient(R, C, R + C).to(DEV)
    ref = muon._newton_schulz_torch(x.double(), 5, muon.NS_EPS)
    err = lambda t: (torch.linalg.norm(t.double() - ref) / torch.linalg.norm(ref)).item()  # noqa: E731
    tol = 4 * err(muon._newton_schulz_torch(x, 5, muon.NS_EPS)) + 8 * 2.0 ** -23 + (2.0 ** -8 if out == torch.bfloat16 else 0.0)
    fill = torch.full((1 << 29,), float("nan"), device=DEV)
    del fill
    got = muon.orthogonalize(x, out=torch.empty(R, C, dtype=out, device=DEV))
    assert err(got) <= tol
