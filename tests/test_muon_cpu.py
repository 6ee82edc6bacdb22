"""Newton-Schulz orthogonalisation and the Muon step: the CPU forms and every refusal (checks shared with the GPU path)."""
import math

import pytest
import torch

from dllm.ops import muon
from dllm.ops.master import join_master, split_master


def exact(u: torch.Tensor, steps: int = 5) -> torch.Tensor:
    """The iteration on singular values, in 64 bits: U diag(p(...p(s))) V^T."""
    u = u.double()
    n = torch.linalg.matrix_norm(u)
    U, s, V = torch.linalg.svd(u / (n + 1e-7), full_matrices=False)
    a, b, c = muon.NS_COEFFS
    for _ in range(steps):
        s = s * (a + b * s ** 2 + c * s ** 4)
    return (U * s.unsqueeze(-2)) @ V


def relerr(x, y):
    return (torch.linalg.norm(x.double().cpu() - y) / torch.linalg.norm(y)).item()


# fp32 arithmetic, five steps: rounding noise (2^-24 per operation) grows by at most 3.45 a step, 3.45^5 = 489, and each step
# rounds about ten times: 489 * 10 * 2^-24 = 2.9e-4 of the largest singular value
TOL = 3e-4


@pytest.mark.parametrize("R,C", [(1, 1), (1, 7), (9, 1), (5, 5), (20, 33), (33, 20)])
@pytest.mark.parametrize("steps", [1, 3, 5])
def test_orthogonalize_cpu(R, C, steps):
    g = torch.Generator().manual_seed(R + C)
    x = torch.randn(R, C, generator=g)
    assert relerr(muon.orthogonalize(x, steps), exact(x, steps)) < TOL
    batch = torch.randn(3, R, C, generator=g)
    out = muon.orthogonalize(batch, steps)
    for i in range(3):
        assert relerr(out[i], exact(batch[i], steps)) < TOL
    assert muon.orthogonalize(x.bfloat16()).dtype == torch.bfloat16


def test_singular_values_end_near_one():
    x = torch.randn(40, 60, generator=torch.Generator().manual_seed(0))
    s = torch.linalg.svdvals(muon.orthogonalize(x))
    assert s.max() < 1.25 and s.min() > 0.5
    assert torch.equal(muon.orthogonalize(torch.zeros(3, 4)), torch.zeros(3, 4))


@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step_cpu(nesterov):
    g = torch.Generator().manual_seed(1)
    w, grad, mom = (torch.randn(24, 10, generator=g) for _ in range(3))
    w0, m0 = w.double(), mom.double()
    copy = torch.empty(24, 10, dtype=torch.bfloat16)
    muon.muon_step_(w, grad, mom, lr=0.1, beta=0.9, nesterov=nesterov, wd=0.5, copy=copy, grad_scale=0.25)
    m = 0.9 * m0 + 0.25 * grad.double()
    u = 0.25 * grad.double() + 0.9 * m if nesterov else m
    torch.testing.assert_close(mom.double(), m, rtol=2 ** -22, atol=2 ** -22)
    want = w0 * (1 - 0.1 * 0.5) - 0.1 * math.sqrt(2.4) * exact(u)
    assert relerr(w, want) < TOL and torch.equal(copy, w.bfloat16())


def test_muon_split_matches_fp32():
    g = torch.Generator().manual_seed(2)
    w, grad, mom = (torch.randn(2, 12, 30, generator=g) for _ in range(3))
    hi, lo = split_master(w)
    mom2 = mom.clone()
    muon.muon_step_(w, grad, mom, lr=0.02, wd=0.1)
    muon.muon_split_step_(lo, hi, grad, mom2, lr=0.02, wd=0.1)
    assert torch.equal(join_master(hi, lo), w) and torch.equal(mom, mom2)


def test_refusals():
    x = torch.randn(4, 6)
    for bad in (0, 21, -1):
        with pytest.raises(ValueError, match="steps must be"):
            muon.orthogonalize(x, bad)
    with pytest.raises(ValueError, match="batch"):
        muon.orthogonalize(x[0])
    with pytest.raises(TypeError, match="bf16 or fp32"):
        muon.orthogonalize(x.half())
    with pytest.raises(ValueError, match="out must be"):
        muon.orthogonalize(x, out=torch.empty(6, 4))
    with pytest.raises(ValueError, match="contiguous"):
        muon.orthogonalize(x, out=torch.empty(6, 4).t())
    with pytest.raises(TypeError, match="must be fp32"):
        muon.muon_step_(x.bfloat16(), x, x.clone(), lr=0.1)
    with pytest.raises(ValueError, match="grad must be"):
        muon.muon_step_(x, x[:2], x.clone(), lr=0.1)
    with pytest.raises(TypeError, match="momentum must be"):
        muon.muon_step_(x, x.clone(), x.bfloat16(), lr=0.1)
    with pytest.raises(ValueError, match="momentum must be contiguous"):
        muon.muon_step_(x, x.clone(), torch.randn(6, 4).t(), lr=0.1)
    with pytest.raises(TypeError, match="copy must be"):
        muon.muon_step_(x, x.clone(), x.clone(), lr=0.1, copy=x.clone())
    for w, g, m in ((x, x, x.clone()), (x, x.clone(), x)):
        with pytest.raises(ValueError, match="share memory"):
            muon.muon_step_(w, g, m, lr=0.1)
    both = torch.randn(7, 4)
    with pytest.raises(ValueError, match="share memory"):        # overlapping by all but a row
        muon.muon_step_(torch.randn(6, 4), both[:6], both[1:], lr=0.1)
    with pytest.raises(TypeError, match="int16 residual"):
        muon.muon_split_step_(x, x.bfloat16(), x, x.clone(), lr=0.1)
