"""Newton-Schulz and the Muon step where the shorter side is above 128: a matrix's bits do not depend on its batch, and what is
not finite stays in its matrix."""
import pytest
import torch

from dllm.ops import muon
from dllm.ops.master import join_master, split_master
from test_muon_gpu import gradient

pytestmark = pytest.mark.gpu
DEV = "cuda"


# (batch, R, C): the cost model takes other tiles for the batch than for one matrix (64 for one; 128, 192 or 256 for these)
BATCHES = [(4, 1024, 4096), (16, 512, 512), (5, 1024, 1024), (64, 256, 256), (3, 2048, 2048), (16, 700, 640), (32, 512, 2048)]


@pytest.mark.parametrize("B,R,C", BATCHES)
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_batch_has_the_bits_of_the_single_matrix(B, R, C, out):
    g = torch.Generator(device=DEV).manual_seed(B + R)
    x = torch.randn(B, R, C, generator=g, device=DEV)
    got = muon.orthogonalize(x, out=torch.empty(B, R, C, dtype=out, device=DEV))
    for i in (0, B // 2, B - 1):
        one = muon.orthogonalize(x[i], out=torch.empty(R, C, dtype=out, device=DEV))
        assert torch.equal(got[i], one), f"matrix {i}: {(got[i] != one).float().mean().item():.4f} of the elements differ"


@pytest.mark.parametrize("B,R,C", [(4, 4096, 1024), (5, 1024, 1024), (16, 512, 640)])
def test_step_of_a_batch_has_the_bits_of_single_steps(B, R, C):
    g = torch.Generator(device=DEV).manual_seed(R)
    w, gr, m = (torch.randn(B, R, C, generator=g, device=DEV) for _ in range(3))
    hi, lo = split_master(w)
    ws, ms, copy, m2 = w.clone(), m.clone(), torch.empty(B, R, C, dtype=torch.bfloat16, device=DEV), m.clone()
    muon.muon_step_(w, gr, m, lr=0.1, wd=0.1, copy=copy)
    muon.muon_split_step_(lo, hi, gr, m2, lr=0.1, wd=0.1)
    assert torch.equal(copy, w.bfloat16()) and torch.equal(join_master(hi, lo), w) and torch.equal(m2, m)
    for i in (0, B - 1):
        muon.muon_step_(ws[i], gr[i], ms[i], lr=0.1, wd=0.1)
        assert torch.equal(ws[i], w[i]) and torch.equal(ms[i], m[i])


@pytest.mark.parametrize("R,C", [(200, 300), (300, 200), (640, 700), (200, 3000), (1024, 1024)])
def test_non_finite_updates_stay_in_their_matrix(R, C):
    """NaN and inf spoil the whole of their own matrix, its momentum only where they are, and nothing of the next matrix."""
    x = gradient(R, C, 5)
    ref = muon.orthogonalize(x.to(DEV))
    b = torch.stack([x, x, x, x])
    b[1, 3, 5] = float("nan")
    b[2, R - 10, C - 7] = float("inf")
    out = muon.orthogonalize(b.to(DEV))
    assert torch.isnan(out[1]).all() and torch.isnan(out[2]).all()
    assert torch.equal(out[0], ref) and torch.equal(out[3], ref)
    w, m = torch.ones(4, R, C, device=DEV), torch.zeros(4, R, C, device=DEV)
    muon.muon_step_(w, b.to(DEV), m, lr=0.1)
    assert torch.isnan(w[1]).all() and torch.isnan(w[2]).all() and torch.isfinite(w[0]).all() and torch.equal(w[0], w[3])
    bad = ~torch.isfinite(m)
    assert bad.sum() == 2 and bad[1, 3, 5] and bad[2, R - 10, C - 7]
