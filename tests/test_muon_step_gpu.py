"""The Muon step where the shorter side is above 128 (segments of three steps, every tile) against the iteration in 64 bits."""
import math

import pytest
import torch

from dllm.ops import muon
from dllm.ops.master import join_master, split_master
from test_muon_gpu import gradient

pytestmark = pytest.mark.gpu
DEV = "cuda"


def iteration(u: torch.Tensor) -> torch.Tensor:
    """Five steps in u's own type, written from the formula."""
    a, b, c = 3.4445, -4.7750, 2.0315
    x = u / (u.square().sum().sqrt() + 1e-7)
    wide = x.shape[0] <= x.shape[1]
    for _ in range(5):
        s = x @ x.t() if wide else x.t() @ x
        p = b * s + c * (s @ s)
        p.diagonal().add_(a)
        x = p @ x if wide else x @ p
    return x


def norm(t: torch.Tensor) -> float:
    return torch.linalg.norm(t.double()).item()


# Three steps on one Gram matrix A (m x m, two fp16 planes: a rounding moves an element by up to 2^-23 of itself, and a step
# has three of them, of P, P A and (P A) P).  A rounding of A reaches P's next value times |b| = 4.8, and the next A times
# |a|^2 = 12: relative to the result (all singular values near 1, norm sqrt(m)) the roundings of the segment's first, second and
# third A count 4.8 * 144 / 3.44 = 200, 57 and 4.8 times their norm over sqrt(m).  |A_0| <= trace = 1, and the others' norms
# are at most sqrt(m): sqrt(3) * 2^-23 * (200 / sqrt(m) + 57 + 4.8), at m >= 129 at most 1.7e-5, and the second segment (two steps,
# 17 and 4.8) 4.5e-6: 2.1e-5.  To this come four times the fp32 iteration's own error, as for single steps.
SEGMENTS = 2.1e-5


def step_tolerance(u: torch.Tensor, o: torch.Tensor) -> float:
    return SEGMENTS + 4 * norm(iteration(u.float()).double() - o) / norm(o)


# the last product's tile (64, 128, 192, 256), wide, tall and odd sizes, sliced Gram matrices
STEPS = [(None, 129, 257), (None, 257, 129), (None, 256, 1024), (None, 1024, 256), (None, 700, 1500), (None, 1500, 700),
         (None, 300, 3000), (None, 3001, 200), (None, 1024, 4096), (None, 4096, 1024), (4, 1024, 4096), (4, 4096, 1024),
         (5, 1024, 1024), (None, 1023, 1025), (None, 2048, 2048), (2, 2048, 2048)]


@pytest.mark.parametrize("B,R,C", STEPS)
@pytest.mark.parametrize("kind", ["normal", "lowrank"])
def test_muon_step_against_64_bits(B, R, C, kind):
    """From a zero master the step hands out the orthogonalised update itself (fp32: 2^-24); from a full one the whole formula,
    fp32 and split, with their bf16 copies."""
    shape = (R, C) if B is None else (B, R, C)
    grad, mom = gradient(R, C, 6, kind, B).to(DEV), gradient(R, C, 7, kind, B).to(DEV) * 10
    w0 = torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(8), device=DEV)
    kw = dict(lr=0.05, beta=0.9, wd=0.1, grad_scale=0.5)
    zero, m = torch.zeros(shape, device=DEV), mom.clone()
    muon.muon_step_(zero, grad, m, scale=1 / 0.05, **kw)
    w, copy, mw = w0.clone(), torch.empty(shape, dtype=torch.bfloat16, device=DEV), mom.clone()
    muon.muon_step_(w, grad, mw, copy=copy, **kw)
    hi, lo = split_master(w0)
    ms = mom.clone()
    muon.muon_split_step_(lo, hi, grad, ms, **kw)
    assert torch.equal(copy, w.bfloat16()) and torch.equal(join_master(hi, lo), w)
    assert torch.equal(m, mw) and torch.equal(m, ms)
    g64 = 0.5 * grad.double()
    m64 = 0.9 * mom.double() + g64
    assert ((m.double() - m64).abs() <= 2 * 2.0 ** -24 * (0.9 * mom.double().abs() + g64.abs())).all()
    u64 = g64 + 0.9 * m64
    rate = 0.05 * math.sqrt(max(1.0, R / C))
    for i in range(B or 1):
        pick = lambda t: t if B is None else t[i]  # noqa: E731
        o = iteration(pick(u64))
        tol = step_tolerance(pick(u64), o)
        err = norm(pick(zero).double() + o) / norm(o)
        assert err <= tol + 2.0 ** -23
        want = pick(w0).double() * (1 - 0.05 * 0.1) - rate * o
        assert norm(pick(w).double() - want) <= tol * rate * norm(o) + 3 * 2.0 ** -24 * norm(want)
