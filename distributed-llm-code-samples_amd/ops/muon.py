"""Newton-Schulz orthogonalisation and the Muon optimizer step (``csrc/muon.hip`` on the GPU, torch on the CPU).

Muon replaces a 2-D weight's update U by the nearest matrix with all singular values near 1, from five steps of

    A = X·Xᵀ,   X <- a·X + (b·A + c·A²)·X,   (a, b, c) = (3.4445, -4.7750, 2.0315),   X_0 = U / (‖U‖_F + eps)

(singular values end between about 0.7 and 1.2).  It stands next to ``sgd_step_`` / ``adam_step_``; the reference has
plain SGD only (train_ffns.py:114).  Every parameter of an FFN stack is a hidden matrix, the kind Muon is meant for.

Accuracy: products of fp32 grade (two fp16 planes per matrix), fp32 or bf16 result; the same input gives the same bits,
alone or in a batch.  A NaN or inf anywhere in a matrix makes that matrix's result NaN; a zero matrix stays zero.
"""
from __future__ import annotations

import math

import torch

from .. import _native
from .fp8 import _on
from .master import join_master, set_master_

NS_COEFFS = (3.4445, -4.7750, 2.0315)
NS_STEPS = 5
NS_EPS = 1e-7
MAX_STEPS = 20


def _dims(t: torch.Tensor, name: str) -> tuple[int, int, int]:
    if t.dim() not in (2, 3):
        raise ValueError(f"{name} must be [R, C] or a batch [B, R, C] of matrices, got {tuple(t.shape)}")
    return (1, *t.shape) if t.dim() == 2 else tuple(t.shape)


def _check_steps(steps: int) -> None:
    if not 1 <= steps <= MAX_STEPS:
        raise ValueError(f"steps must be between 1 and {MAX_STEPS}, got {steps}")


def _check_dense(t: torch.Tensor, name: str, shape: torch.Size, dtypes: tuple, device) -> None:
    if t.shape != shape or t.device != device:
        raise ValueError(f"{name} must be {tuple(shape)} on {device}, got {tuple(t.shape)} on {t.device}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be one of {dtypes}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _workspace(B: int, R: int, C: int, steps: int, device) -> torch.Tensor:
    n = _native.lib().dllm_muon_workspace(B, R, C, steps) if max(B, R, C) < 2 ** 31 else 0
    if n <= 0:
        raise ValueError(f"matrices of {R}x{C} (batch {B}) are beyond the kernels' range: shorter side up to 65536, "
                         "longer up to 2097152, batch up to 65535")
    return torch.empty(n, dtype=torch.uint8, device=device)


def _newton_schulz_torch(u: torch.Tensor, steps: int, eps: float) -> torch.Tensor:
    a, b, c = NS_COEFFS
    dt = torch.float64 if u.dtype == torch.float64 else torch.float32
    x = u.to(dt)
    x = x / (x.square().sum(dim=(-2, -1), keepdim=True).sqrt() + eps)
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1)
    for _ in range(steps):
        g = torch.matmul(x, x.transpose(-2, -1))
        x = a * x + torch.matmul(b * g + c * torch.matmul(g, g), x)
    return x.transpose(-2, -1) if tall else x


def orthogonalize(x: torch.Tensor, steps: int = NS_STEPS, out: torch.Tensor | None = None,
                  eps: float = NS_EPS) -> torch.Tensor:
    """The orthogonalised ``x`` ([R, C] or a batch [B, R, C], bf16 or fp32); ``out``: x's shape, bf16 or fp32 (default: x's
    type).  ``out`` may be ``x``."""
    B, R, C = _dims(x, "x")
    _check_steps(steps)
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"orthogonalize takes bf16 or fp32, got {x.dtype}")
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _check_dense(out, "out", x.shape, (torch.bfloat16, torch.float32), x.device)
    if x.numel() == 0:
        return out
    if x.device.type != "cuda":
        out.copy_(_newton_schulz_torch(x, steps, eps))
        return out
    x = x.contiguous()
    with _on(x.device):
        ws = _workspace(B, R, C, steps, x.device)
        rc = _native.lib().dllm_orthogonalize(x.data_ptr(), _native.dtype_code(x.dtype), out.data_ptr(),
                                              _native.dtype_code(out.dtype), B, R, C, steps, float(eps), ws.data_ptr(),
                                              ws.numel(), _native.stream_ptr(x.device))
    _native.check(rc, f"dllm_orthogonalize({B}x{R}x{C})")
    return out


def muon_scale(rows: int, cols: int) -> float:
    """The update's factor for a ``[rows, cols]`` weight: ``sqrt(max(1, rows / cols))`` (equal change of the layer's output
    for wide and tall weights)."""
    return math.sqrt(max(1.0, rows / cols))


def _blocks_of(t: torch.Tensor, interleave: int) -> torch.Tensor:
    """[2, R, C] view-or-copy of the two matrices whose rows alternate in blocks of ``interleave``."""
    C = t.shape[1]
    return t.view(-1, 2, interleave, C).transpose(0, 1).reshape(2, -1, C)


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    pa, pb = a.data_ptr(), b.data_ptr()
    return pa < pb + b.numel() * b.element_size() and pb < pa + a.numel() * a.element_size()


def _step(grad, momentum, lr, beta, nesterov, wd, steps, eps, scale, grad_scale, interleave, master, copy, lo) -> None:
    ref = lo if master is None else master
    B, R, C = _dims(ref, "the weight")
    _check_steps(steps)
    _check_dense(ref, "the weight", ref.shape, (ref.dtype,), ref.device)
    _check_dense(grad, "grad", ref.shape, (torch.bfloat16, torch.float32), ref.device)
    _check_dense(momentum, "momentum", ref.shape, (torch.float32,), ref.device)
    if copy is not None:
        _check_dense(copy, "the bf16 copy", ref.shape, (torch.bfloat16,), ref.device)
    if interleave:
        if ref.dim() != 2 or interleave < 0 or R % (2 * interleave):
            raise ValueError(f"interleave = {interleave} needs a 2-D weight with rows in multiples of {2 * abs(interleave)}, "
                             f"got {tuple(ref.shape)}")
        B, R = 2, R // 2
    if ref.numel() == 0:
        return
    # the momentum is written while the gradient is read, and both are read again when the weights are written
    for t, what in ((grad, "grad"), (momentum, "momentum")):
        for u in (momentum, ref, copy) if t is grad else (ref, copy):
            if u is not None and _overlap(t, u):
                raise ValueError(f"{what} must not share memory with the other tensors")
    if copy is not None and _overlap(ref, copy):
        raise ValueError("the weight's tensors must not share memory")
    rate = lr * (muon_scale(R, C) if scale is None else scale)
    decay = 1.0 - lr * wd
    if ref.device.type != "cuda":
        g = grad.float() * grad_scale
        momentum.mul_(beta).add_(g)
        u = g + beta * momentum if nesterov else momentum
        if interleave:
            o = _newton_schulz_torch(_blocks_of(u, interleave), steps, eps)
            o = o.view(2, -1, interleave, C).transpose(0, 1).reshape(u.shape)
        else:
            o = _newton_schulz_torch(u, steps, eps)
        if master is not None:
            master.mul_(decay).sub_(rate * o)
            if copy is not None:
                copy.copy_(master)
        else:
            set_master_(copy, lo, join_master(copy, lo).mul_(decay).sub_(rate * o))
        return
    ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
    with _on(ref.device):
        ws = _workspace(B, R, C, steps, ref.device)
        rc = _native.lib().dllm_muon_step(grad.data_ptr(), _native.dtype_code(grad.dtype), momentum.data_ptr(), ptr(master),
                                          ptr(copy), ptr(lo), B, R, C, steps, float(eps), float(beta), int(nesterov),
                                          float(grad_scale), float(decay), float(rate), int(interleave), ws.data_ptr(),
                                          ws.numel(), _native.stream_ptr(ref.device))
    if rc:
        _native.check(rc, f"dllm_muon_step({B}x{R}x{C})")


def muon_step_(master: torch.Tensor, grad: torch.Tensor, momentum: torch.Tensor, lr: float, beta: float = 0.95,
               nesterov: bool = True, wd: float = 0.0, steps: int = NS_STEPS, eps: float = NS_EPS,
               copy: torch.Tensor | None = None, scale: float | None = None, grad_scale: float = 1.0,
               interleave: int = 0) -> None:
    """Muon on fp32 weights ``master`` [R, C] (or a batch [B, R, C] of equal shape, each its own matrix), in place:

    ``momentum = beta·momentum + g``, ``U = g + beta·momentum`` (``nesterov``) or ``momentum``, ``O = orthogonalize(U)``,
    ``master = (1 - lr·wd)·master - lr·scale·O``, ``copy = bf16(master)``,  with ``g = grad_scale·grad`` (bf16 or fp32).
    ``scale`` defaults to ``muon_scale(R, C)``.  ``interleave``: ``master`` [2 R, C] holds two matrices whose rows alternate
    in blocks of that many (the gated FFN's W13), each stepped as its own.  No two of the tensors may share memory."""
    if master.dtype != torch.float32:
        raise TypeError("master weights must be fp32")
    _step(grad, momentum, lr, beta, nesterov, wd, steps, eps, scale, grad_scale, interleave, master, copy, None)


def muon_split_step_(lo: torch.Tensor, hi: torch.Tensor, grad: torch.Tensor, momentum: torch.Tensor, lr: float,
                     beta: float = 0.95, nesterov: bool = True, wd: float = 0.0, steps: int = NS_STEPS,
                     eps: float = NS_EPS, scale: float | None = None, grad_scale: float = 1.0,
                     interleave: int = 0) -> None:
    """``muon_step_`` on a split master (``ops/master.py``): ``lo`` the int16 residual plane, ``hi`` the bf16 working copy."""
    if lo.dtype != torch.int16 or hi.dtype != torch.bfloat16 or lo.shape != hi.shape:
        raise TypeError("muon_split_step_ takes an int16 residual plane and its bf16 working copy")
    _step(grad, momentum, lr, beta, nesterov, wd, steps, eps, scale, grad_scale, interleave, None, hi, lo)
