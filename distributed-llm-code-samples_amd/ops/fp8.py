"""Block-scaled 8-bit floating point: quantiser, read-back, matrix product and the linear layer on them.

The reference trains in fp32 only (``linear_fwd`` / ``t_linear_bkwd``, train_ffns.py:41-45); this is the same three
products with 8-bit operands, which the gfx950 matrix cores run at twice the bf16 rate.

Format (``BlockFP8``): 8-bit codes (OCP e4m3 or e5m2) with one power-of-two scale per row and 128 consecutive k -- or per
128x128 tile, the same byte repeated on the tile's rows.  For a block with largest finite magnitude ``amax``

    e = the smallest integer >= -127 with amax <= FMAX * 2^e        (FMAX: e4m3 448, e5m2 57344)
    code = x * 2^-e rounded to nearest even,   stands for code * 2^e,   scale byte = e + 127

The division is exact, so every value is rounded once (by at most half a step: 2^-4 relative for normal e4m3 codes, 2^-3
for e5m2) and nothing finite saturates.  Non-finite elements do not enter ``amax``: NaN stays NaN, +-inf stays inf in e5m2
and becomes NaN in e4m3 (which has no infinity), and the rest of their block keeps its values.

GPU tensors run ``csrc/fp8.hip``; CPU tensors run the torch forms below (tests, oracle).
"""
from __future__ import annotations

import contextlib
import functools
from typing import NamedTuple

import torch

from .. import _native
from .activations import act_code, act_fwd, act_grad
from .gemm import EPIS

BLOCK = 128
MAX_DIM = 2 ** 31 - 2 * BLOCK      # the kernels count rows and columns in 32 bits
FORMATS = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_CODES = {torch.float8_e4m3fn: 0, torch.float8_e5m2: 1}
_TOP = {torch.float8_e4m3fn: 8, torch.float8_e5m2: 15}   # FMAX = 1.75 * 2^top


class BlockFP8(NamedTuple):
    """An 8-bit operand of logical shape ``[rows, k]``: ``data`` [rows, k rounded up to 128] (zeros behind ``k``) in a torch
    float8 type, ``scale`` uint8 [k blocks, rows] (exponent bytes, biased by 127)."""
    data: torch.Tensor
    scale: torch.Tensor
    k: int

    @property
    def rows(self) -> int:
        return self.data.shape[0]

    @property
    def device(self) -> torch.device:
        return self.data.device


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _fmt(fmt: str) -> torch.dtype:
    if fmt not in FORMATS:
        raise ValueError(f"unknown 8-bit format {fmt!r}; choose from {sorted(FORMATS)}")
    return FORMATS[fmt]


_HERE = contextlib.nullcontext()


def _on(device: torch.device):
    """Launches go to the tensors' device, whichever device is current."""
    return _HERE if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)


def fp8_empty(rows: int, k: int, fmt: str = "e4m3", device=None) -> BlockFP8:
    """Storage for a ``[rows, k]`` operand (uninitialised), for the quantisers' ``out``."""
    return BlockFP8(torch.empty((rows, _blocks(k) * BLOCK), dtype=_fmt(fmt), device=device),
                    torch.empty((_blocks(k), rows), dtype=torch.uint8, device=device), k)


def _ld(t: torch.Tensor) -> int:
    """Row stride of a view that ``_check_rows`` passed (torch leaves the stride of a single row arbitrary)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _check(q: BlockFP8, name: str) -> tuple[int, int, int, int, int]:
    """The operand as the kernels take it: (data, its row stride, scale, its row stride, format code)."""
    d, sc, k = q
    code = _CODES.get(d.dtype)
    if code is None or d.dim() != 2:
        raise TypeError(f"{name}: data must be a 2-D float8 tensor (e4m3fn or e5m2), got {d.dtype} {tuple(d.shape)}")
    rows, cols = d.shape
    if rows > MAX_DIM or cols > MAX_DIM:
        raise ValueError(f"{name}: up to {MAX_DIM} rows and columns, got {rows} and {cols}")
    kb = -(-k // BLOCK)
    if k < 0 or cols != kb * BLOCK:
        raise ValueError(f"{name}: data of k = {k} has {kb * BLOCK} columns, got {cols}")
    if sc.dtype != torch.uint8 or sc.shape != (kb, rows):
        raise ValueError(f"{name}: scale must be uint8 {(kb, rows)}, got {sc.dtype} {tuple(sc.shape)}")
    if sc.device != d.device:
        raise ValueError(f"{name}: data on {d.device}, scale on {sc.device}")
    ptr, (ld, s1), (lds, t1) = d.data_ptr(), d.stride(), sc.stride()
    ld, lds = ld if rows > 1 else cols, lds if kb > 1 else rows
    if rows and cols:
        if s1 != 1 or (rows > 1 and t1 != 1) or ld < cols or lds < rows:
            raise ValueError(f"{name}: data and scale must be contiguous along their last dimension, without overlapping rows; "
                             f"got strides {d.stride()} and {sc.stride()}")
        if d.is_cuda and (ptr % 16 or ld % 16):
            raise ValueError(f"{name}: data rows must start at multiples of 16 bytes")
    return ptr, ld, sc.data_ptr(), lds, code


def _pow2(e: torch.Tensor) -> torch.Tensor:
    """2^e in fp32, exactly, for integer -127 <= e <= 127."""
    normal = ((e + 127) << 23).to(torch.int32).view(torch.float32)
    return torch.where(e == -127, torch.full_like(normal, 2.0 ** -127), normal)


def _quantize_torch(x: torch.Tensor, dt: torch.dtype, tile: bool, out: BlockFP8) -> None:
    R, K = x.shape
    kb, rb = _blocks(K), _blocks(R)
    p = torch.zeros((rb * BLOCK if tile else R, kb * BLOCK), dtype=torch.float32, device=x.device)
    p[:R, :K] = x
    v = p.view(rb, BLOCK, kb, BLOCK) if tile else p.view(R, 1, kb, BLOCK)
    amax = torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v)).amax(dim=(1, 3), keepdim=True)
    bits = amax.contiguous().view(torch.int32)
    e = (((bits + 0x1FFFFF) >> 23) - _TOP[dt]).clamp(min=0) - 127
    q = v * _pow2(-e)
    if dt == torch.float8_e4m3fn:
        q = torch.where(torch.isinf(q), torch.full_like(q, float("nan")), q)
    out.data.copy_(q.reshape(p.shape)[:R].to(dt))
    out.scale.copy_((e + 127).to(torch.uint8).expand(v.shape[0], v.shape[1], kb, 1).reshape(-1, kb)[:R].t())


def _target(out: BlockFP8 | None, rows: int, k: int, fmt: str, device, name: str) -> tuple[BlockFP8, tuple]:
    """The output operand (made, or checked) and the kernels' form of it."""
    if out is None:
        out = fp8_empty(rows, k, fmt, device)
        return out, (out.data.data_ptr(), out.data.shape[1], out.scale.data_ptr(), rows, _CODES[out.data.dtype])
    arg = _check(out, name)
    if out.rows != rows or out.k != k or out.device != device:
        raise ValueError(f"{name} must hold {(rows, k)} on {device}, got {(out.rows, out.k)} on {out.device}")
    return out, arg


def _shape2(x: torch.Tensor) -> tuple[int, int]:
    if x.dim() != 2 or x.dtype not in _native.DT:
        raise TypeError(f"the quantiser takes 2-D bf16 or fp32 tensors, got {x.dtype} {tuple(x.shape)}")
    R, C = x.shape
    if R > MAX_DIM or C > MAX_DIM:
        raise ValueError(f"the quantiser takes up to {MAX_DIM} rows and columns, got {tuple(x.shape)}")
    return R, C


_NONE = (None, 0, None, 0, 0)


def _quantize(x: torch.Tensor, R: int, C: int, q: BlockFP8 | None, arg: tuple, qt: BlockFP8 | None, arg_t: tuple,
              tile: bool) -> None:
    if R == 0 or C == 0:
        return
    if not x.is_cuda:
        if q is not None:
            _quantize_torch(x, q.data.dtype, tile, q)
        if qt is not None:
            _quantize_torch(x.t(), qt.data.dtype, tile, qt)
        return
    if C > 1 and x.stride(1) != 1:
        x = x.contiguous()
    dev = x.device
    with _on(dev):
        rc = _native.lib().dllm_fp8_quantize(x.data_ptr(), _native.DT[x.dtype], x.stride(0), R, C, *arg[:4], *arg_t[:4], arg[4],
                                             arg_t[4], int(tile), _native.stream_ptr(dev))
    if rc:
        _native.check(rc, f"dllm_fp8_quantize({R}x{C})")


def quantize_fp8(x: torch.Tensor, fmt: str = "e4m3", *, tile: bool = False, out: BlockFP8 | None = None) -> BlockFP8:
    """The 8-bit form of ``x`` [R, K] (bf16 / fp32), scaled per row and 128 columns (``tile``: per 128x128 tile)."""
    R, C = _shape2(x)
    out, arg = _target(out, R, C, fmt, x.device, "out")
    _quantize(x, R, C, out, arg, None, _NONE, tile)
    return out


def quantize_fp8_t(x: torch.Tensor, fmt: str = "e4m3", *, tile: bool = False, out: BlockFP8 | None = None) -> BlockFP8:
    """The 8-bit form of ``xᵀ`` [K, R], scaled per column of ``x`` and 128 rows (``tile``: per 128x128 tile)."""
    R, C = _shape2(x)
    out, arg = _target(out, C, R, fmt, x.device, "out")
    _quantize(x, R, C, None, _NONE, out, arg, tile)
    return out


def quantize_fp8_both(x: torch.Tensor, fmt: str = "e4m3", fmt_t: str = "e4m3", *, tile: bool = False,
                      out: BlockFP8 | None = None, out_t: BlockFP8 | None = None) -> tuple[BlockFP8, BlockFP8]:
    """``(quantize_fp8(x, fmt), quantize_fp8_t(x, fmt_t))`` from one read of ``x``: a forward (or input-gradient) operand
    and the weight-gradient operand of the same tensor."""
    R, C = _shape2(x)
    out, arg = _target(out, R, C, fmt, x.device, "out")
    out_t, arg_t = _target(out_t, C, R, fmt_t, x.device, "out_t")
    if R and C and (arg[0] == arg_t[0] or arg[2] == arg_t[2]):   # both orientations are written at once
        raise ValueError("out and out_t must not share memory")
    _quantize(x, R, C, out, arg, out_t, arg_t, tile)
    return out, out_t


def dequantize_fp8(q: BlockFP8, dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values ``[rows, k]`` that ``q`` stands for, in bf16 or fp32: exact but where the type ends (a code that rounded up
    to 2^128 reads as inf; values among the type's subnormals are rounded)."""
    ptr, ld, sptr, lds, code = _check(q, "q")
    d, k = q.data, q.k
    rows, dev = d.shape[0], d.device
    dtype = dtype if out is None else out.dtype
    if dtype not in _native.DT:
        raise TypeError(f"dequantize_fp8 gives bf16 or fp32, not {dtype}")
    if out is None:
        out, ldo = torch.empty((rows, k), dtype=dtype, device=dev), k
    else:
        _check_rows(out, "out", (rows, k), dev)
        ldo = _ld(out)
    if rows == 0 or k == 0:
        return out
    if not d.is_cuda:
        kb = _blocks(q.k)
        e = q.scale.t().to(torch.int32) - 127
        s = torch.where(e == 128, torch.full_like(e, 0), e)
        v = q.data.float().view(q.rows, kb, BLOCK) * _pow2(s).unsqueeze(2)
        v = torch.where((e == 128).unsqueeze(2), torch.full_like(v, float("nan")), v)
        out.copy_(v.reshape(q.rows, -1)[:, :q.k])
        return out
    with _on(dev):
        rc = _native.lib().dllm_fp8_dequantize(ptr, ld, sptr, lds, code, out.data_ptr(), _native.DT[dtype], ldo, rows, k,
                                               _native.stream_ptr(dev))
    if rc:
        _native.check(rc, f"dllm_fp8_dequantize({rows}x{k})")
    return out


def _check_rows(t: torch.Tensor, name: str, shape: tuple, device) -> None:
    if t.shape != shape or t.device != device:
        raise ValueError(f"{name} must be {shape} on {device}, got {tuple(t.shape)} on {t.device}")
    if (shape[1] > 1 and t.stride(1) != 1) or (shape[0] > 1 and t.stride(0) < shape[1]):
        raise ValueError(f"{name} must be a row-major view without overlapping rows, got strides {t.stride()}")


MAX_PITCH = (2 ** 31 - 1 - 4096) // 256    # bytes between rows that the tiled kernels take; the one for few rows takes any


@functools.lru_cache(maxsize=4096)
def _plan(M: int, N: int, kb: int, out_code: int, pitch: int = 0) -> tuple[int, int]:
    """(output tile, or 0 for the kernel for few rows, K slices) of a product's sizes and result type.  ``pitch``: the larger
    row stride of the operands where it is above ``MAX_PITCH``."""
    p = _native.lib().dllm_fp8_gemm_plan(M, N, kb, out_code, pitch)
    if p < 0:
        raise ValueError(f"8-bit product of {M} x {N}: with more than 64 rows on both sides operand rows are up to {MAX_PITCH} "
                         f"bytes apart{f', got {pitch}' if pitch else ''}; with fewer, up to {2 ** 27 - 16} rows on the other side")
    return p & 0xFFFF, p >> 16


def _far(*pitches: int) -> int:
    """The largest row stride where it changes the choice of a kernel, else 0 (one cached plan for all others)."""
    p = max(pitches)
    return p if p > MAX_PITCH else 0


def gemm_fp8(a: BlockFP8, b: BlockFP8, out: torch.Tensor | None = None, *, out_dtype: torch.dtype = torch.bfloat16,
             alpha: float = 1.0, beta: float = 0.0, epi: str = "store", act: str = "none",
             aux: torch.Tensor | None = None, aux_out: torch.Tensor | None = None) -> torch.Tensor:
    """``C[M, N] = A[M, K] · B[N, K]ᵀ`` of two 8-bit operands (either format on either side), bf16 or fp32 ``out`` (any row
    stride).  Epilogues as in ``gemm``: ``"store"`` (``alpha·acc + beta·C``), ``"act"`` (``C = act(acc)``, ``aux_out =
    acc``) and ``"dact"`` (``C = acc · act'(aux)``).

    The result's type sets the arithmetic.  fp32: exact products and fp32 sums (about 5e-7 of the result at K = 8192), at
    the bf16 matrix rate.  bf16: the 8-bit matrix instruction, twice as fast, whose sums of 8 neighbouring products keep 13
    bits below the largest (about 4e-5 of the result, a hundredth of bf16's half step)."""
    aarg, barg = _check(a, "a"), _check(b, "b")
    ad, bd, k = a.data, b.data, a.k
    dev = ad.device
    if k != b.k:
        raise ValueError(f"gemm_fp8: inner dims differ ({k} vs {b.k})")
    if dev != bd.device:
        raise ValueError(f"gemm_fp8: operands on {dev} and {bd.device}")
    M, N = ad.shape[0], bd.shape[0]
    if out is None:
        if beta != 0.0:
            raise ValueError("gemm_fp8: beta needs out")
        out, ldc = torch.empty((M, N), dtype=out_dtype, device=dev), N
    else:
        _check_rows(out, "out", (M, N), dev)
        ldc, out_dtype = _ld(out), out.dtype
    oc = _native.DT.get(out_dtype)
    if oc is None:
        raise TypeError(f"gemm_fp8: out must be bf16 or fp32, got {out_dtype}")
    side = None
    if epi == "store":
        if aux is not None or aux_out is not None:
            raise ValueError("gemm_fp8: aux belongs to epilogue dact, aux_out to act")
        code = 0
    else:
        side = _check_epilogue(epi, act, alpha, beta, aux, aux_out, out)
        code = act_code(act)
    if M == 0 or N == 0:
        return out
    if not ad.is_cuda:
        return _gemm_torch(a, b, out, alpha, beta, epi, act, aux, aux_out)
    nk = ad.shape[1] // BLOCK
    tile, ksplit = _plan(M, N, nk, oc, _far(aarg[1], barg[1]))
    ws = torch.empty(ksplit * M * N, dtype=torch.float32, device=dev) if ksplit > 1 else None
    with _on(dev):
        rc = _native.lib().dllm_fp8_gemm(
            *aarg, *barg, out.data_ptr(), ldc, oc, aux.data_ptr() if aux is not None else None,
            aux_out.data_ptr() if aux_out is not None else None, _ld(side) if side is not None else 0, M, N, nk, alpha, beta,
            EPIS[epi], code, tile, ksplit, ws.data_ptr() if ws is not None else None, _native.stream_ptr(dev))
    if rc:
        _native.check(rc, f"dllm_fp8_gemm({epi},M={M},N={N},K={k})")
    return out


def _check_epilogue(epi, act, alpha, beta, aux, aux_out, out) -> torch.Tensor | None:
    if epi not in ("act", "dact"):
        raise ValueError(f"gemm_fp8: unknown epilogue {epi!r}; choose from store, act, dact")
    act_code(act)
    if act == "none":
        raise ValueError(f"gemm_fp8: epilogue {epi} needs an activation")
    if alpha != 1.0 or beta != 0.0:
        raise ValueError(f"gemm_fp8: epilogue {epi} takes no alpha / beta")
    if epi == "dact" and aux is None:
        raise ValueError("gemm_fp8: epilogue dact needs aux (pre-activation)")
    if (aux is not None) != (epi == "dact") or (aux_out is not None and epi != "act"):
        raise ValueError("gemm_fp8: aux belongs to epilogue dact, aux_out to act")
    side = aux if aux is not None else aux_out
    if side is not None:
        _check_rows(side, "aux" if aux is not None else "aux_out", tuple(out.shape), out.device)
        if side.dtype != out.dtype:
            raise TypeError("gemm_fp8: aux / aux_out must have the output dtype")
    return side


def _gemm_torch(a, b, out, alpha, beta, epi, act, aux, aux_out) -> torch.Tensor:
    acc = dequantize_fp8(a) @ dequantize_fp8(b).t()
    if epi == "store":
        out.copy_(alpha * acc + beta * out.float() if beta != 0.0 else alpha * acc)
    elif epi == "act":
        if aux_out is not None:
            aux_out.copy_(acc)
        out.copy_(act_fwd(act, acc))
    else:
        out.copy_(acc * act_grad(act, aux.float()))
    return out


# ----------------------------------------------------------------------------------------------------------------
# the linear layer on 8-bit operands
# ----------------------------------------------------------------------------------------------------------------
class LinearFP8(NamedTuple):
    """What ``linear_fp8`` keeps for its backward: xᵀ (weight gradient) and wᵀ (input gradient) in 8 bits."""
    x_t: BlockFP8
    w_t: BlockFP8


@functools.lru_cache(maxsize=4096)
def _linear_workspace(T: int, D: int, F: int, out_code: int) -> int:
    _plan(T, F, _blocks(D), out_code, _far(_blocks(D) * BLOCK))
    return _native.lib().dllm_linear_fp8_workspace(T, D, F, out_code)


@functools.lru_cache(maxsize=4096)
def _linear_bwd_workspace(T: int, D: int, F: int, dx_code: int, dw_code: int, ld_wt: int, ld_xt: int) -> int:
    if dx_code >= 0:
        _plan(T, D, _blocks(F), dx_code, _far(_blocks(F) * BLOCK, ld_wt))
    _plan(F, D, _blocks(T), dw_code, _far(_blocks(T) * BLOCK, ld_xt))
    return _native.lib().dllm_linear_fp8_bwd_workspace(T, D, F, dx_code, dw_code, ld_wt, ld_xt)


def _rows(x: torch.Tensor) -> torch.Tensor:
    return x if x.shape[1] <= 1 or x.stride(1) == 1 else x.contiguous()


def linear_fp8(x: torch.Tensor, w: torch.Tensor, out: torch.Tensor | None = None,
               out_dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, LinearFP8]:
    """``y = x·wᵀ`` (``linear_fwd`` train_ffns.py:41-42) with x [T, D] quantised per row and 128 columns and w [F, D] per
    128x128 tile, both e4m3.  Returns ``(y, saved)``; ``saved`` goes to ``linear_fp8_bwd``.  The same values as
    ``quantize_fp8_both`` and ``gemm_fp8`` give, in one call."""
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[1]:
        raise ValueError(f"linear_fp8: x [T, D] and w [F, D], got {tuple(x.shape)} and {tuple(w.shape)}")
    (T, D), (F, _) = _shape2(x), _shape2(w)
    dev = x.device
    if w.device != dev:
        raise ValueError(f"linear_fp8: x on {dev}, w on {w.device}")
    if not x.is_cuda or T == 0 or D == 0 or F == 0:
        xq, xt = quantize_fp8_both(x)
        wq, wt = quantize_fp8_both(w, tile=True)
        return gemm_fp8(xq, wq, out, out_dtype=out_dtype), LinearFP8(xt, wt)
    if out is None:
        out, ldo = torch.empty((T, F), dtype=out_dtype, device=dev), F
    else:
        _check_rows(out, "out", (T, F), dev)
        ldo, out_dtype = _ld(out), out.dtype
    oc = _native.DT.get(out_dtype)
    if oc is None:
        raise TypeError(f"linear_fp8: out must be bf16 or fp32, got {out_dtype}")
    x, w = _rows(x), _rows(w)
    n = _linear_workspace(T, D, F, oc)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    xt, wt = fp8_empty(D, T, "e4m3", dev), fp8_empty(D, F, "e4m3", dev)
    with _on(dev):
        rc = _native.lib().dllm_linear_fp8(
            x.data_ptr(), _native.DT[x.dtype], x.stride(0), w.data_ptr(), _native.DT[w.dtype], w.stride(0), T, D, F,
            xt.data.data_ptr(), xt.scale.data_ptr(), wt.data.data_ptr(), wt.scale.data_ptr(), out.data_ptr(), oc, ldo,
            ws.data_ptr(), n, _native.stream_ptr(dev))
    if rc:
        _native.check(rc, f"dllm_linear_fp8(T={T},D={D},F={F})")
    return out, LinearFP8(xt, wt)


def linear_fp8_bwd(dy: torch.Tensor, saved: LinearFP8, dw: torch.Tensor | None = None, *, beta: float = 0.0,
                   dx: torch.Tensor | None = None, need_dx: bool = True) -> tuple[torch.Tensor | None, torch.Tensor]:
    """``(dx, dw) = (dy·w, dyᵀ·x)`` (``t_linear_bkwd`` train_ffns.py:44-45) with dy [T, F] quantised to e5m2 (gradients
    need range more than digits): per row for dx, per column for dw.  ``dx`` has dy's type unless given, ``dw`` is fp32
    unless given; ``beta`` accumulates into ``dw``."""
    xt, wt = saved
    T, F, D = xt.k, wt.k, xt.rows
    if dy.dim() != 2 or dy.shape != (T, F):
        raise ValueError(f"linear_fp8_bwd: dy must be {(T, F)}, got {tuple(dy.shape)}")
    if dw is None and beta != 0.0:
        raise ValueError("linear_fp8_bwd: beta needs dw")
    if not need_dx and dx is not None:
        raise ValueError("linear_fp8_bwd: dx given with need_dx = False")
    _shape2(dy)
    dev = dy.device
    if not dy.is_cuda or T == 0 or D == 0 or F == 0:
        if need_dx:
            dq, dt = quantize_fp8_both(dy, "e5m2", "e5m2")
            dx = gemm_fp8(dq, wt, dx, out_dtype=dy.dtype)
        else:
            dt = quantize_fp8_t(dy, "e5m2")
        return dx, gemm_fp8(dt, xt, dw, out_dtype=torch.float32, beta=beta)
    xarg, warg = _check(xt, "saved.x_t"), _check(wt, "saved.w_t")
    if xt.device != dev or wt.device != dev or wt.rows != D:
        raise ValueError(f"linear_fp8_bwd: saved operands {xt.rows} x {T} on {xt.device}, {wt.rows} x {F} on {wt.device} "
                         f"for dy on {dev}")
    codes, args = [], []
    for t, name, shape, dtype in ((dx, "dx", (T, D), dy.dtype), (dw, "dw", (F, D), torch.float32)):
        if name == "dx" and not need_dx:
            codes.append(-1)
            args += [None, -1, 0]
            continue
        if t is None:
            t, ld = torch.empty(shape, dtype=dtype, device=dev), D
        else:
            _check_rows(t, name, shape, dev)
            ld, dtype = _ld(t), t.dtype
        if dtype not in _native.DT:
            raise TypeError(f"linear_fp8_bwd: {name} must be bf16 or fp32, got {dtype}")
        codes.append(_native.DT[dtype])
        args += [t.data_ptr(), codes[-1], ld]
        if name == "dx":
            dx = t
        else:
            dw = t
    dy = _rows(dy)
    n = _linear_bwd_workspace(T, D, F, *codes, _far(warg[1]), _far(xarg[1]))
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    with _on(dev):
        rc = _native.lib().dllm_linear_fp8_bwd(dy.data_ptr(), _native.DT[dy.dtype], dy.stride(0), T, D, F, *xarg, *warg, *args,
                                               beta, ws.data_ptr(), n, _native.stream_ptr(dev))
    if rc:
        _native.check(rc, f"dllm_linear_fp8_bwd(T={T},D={D},F={F})")
    return dx, dw
