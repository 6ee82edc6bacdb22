"""Measured cases of the 8-bit training operators and of the orthogonalised update.

* block-scaled 8-bit quantisation (``dllm.ops.fp8``: ``quantize_fp8`` / ``quantize_fp8_t`` / ``quantize_fp8_both``,
  ``dequantize_fp8``),
* matrix products of such operands (``gemm_fp8``) and a linear layer's forward and backward on them
  (``linear_fp8`` / ``linear_fp8_bwd``),
* Newton-Schulz orthogonalisation and the Muon update (``dllm.ops.muon``: ``orthogonalize``, ``muon_step_``).

``own`` selects the framework's operators; otherwise ``run`` computes the plain fp32 forms.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 128
FMAX = {"e4m3": 448.0, "e5m2": 57344.0}
DTYPES = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
FLOATS = {"bf16": torch.bfloat16, "fp32": torch.float32}
NS_A, NS_B, NS_C = 3.4445, -4.7750, 2.0315
NS_EPS = 1e-7


# ----------------------------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # one token's activation on its way into an 8-bit layer: a latency call
        {"name": "quantise one token", "op": "quantise", "rows": 1, "cols": 4096, "dtype": "bf16", "fmt": "e4m3",
         "tile": False, "both": False},
        # the flagship's activations: x for the forward product and its transpose for the weight gradient, in one call
        {"name": "quantise activations", "op": "quantise", "rows": 8192, "cols": 4096, "dtype": "bf16", "fmt": "e4m3",
         "tile": False, "both": True},
        # a weight of odd size in 128x128 tiles, for the forward and the input-gradient product, from its fp32 master
        {"name": "quantise odd weight", "op": "quantise", "rows": 1537, "cols": 1000, "dtype": "fp32", "fmt": "e4m3",
         "tile": True, "both": True},
        # one token through a layer whose weight was quantised before: reads the weight once
        {"name": "product one token", "op": "product", "M": 1, "N": 16384, "K": 4096, "fa": "e4m3", "fb": "e4m3",
         "out": "bf16", "beta": 0.0},
        # odd sizes in every dimension, gradient format on one side, fp32 result
        {"name": "product odd", "op": "product", "M": 333, "N": 1000, "K": 1537, "fa": "e5m2", "fb": "e4m3",
         "out": "fp32", "beta": 0.0},
        # the flagship layer's first forward product
        {"name": "product forward", "op": "product", "M": 8192, "N": 16384, "K": 4096, "fa": "e4m3", "fb": "e4m3",
         "out": "bf16", "beta": 0.0},
        # the flagship layer's weight gradient, accumulated in fp32 over micro-batches
        {"name": "product weight gradient", "op": "product", "M": 4096, "N": 16384, "K": 8192, "fa": "e5m2",
         "fb": "e4m3", "out": "fp32", "beta": 1.0},
        # a whole 8-bit linear layer of a small stack: forward, input gradient and weight gradient from bf16 tensors
        {"name": "linear small", "op": "linear", "T": 1000, "D": 512, "F": 1400},
        # the same for the flagship layer
        {"name": "linear flagship", "op": "linear", "T": 8192, "D": 4096, "F": 16384},
        # a small odd gradient, tall, fp32 result
        {"name": "orthogonalise odd", "op": "orthogonalise", "batch": 1, "rows": 300, "cols": 101, "dtype": "fp32"},
        # the Muon update of four layers' weights at once (model size 1024, FFN 4096): momentum, master, bf16 copy
        {"name": "muon step", "op": "muon", "batch": 4, "rows": 4096, "cols": 1024, "wd": 0.01},
        # one flagship gradient, bf16 in and out
        {"name": "orthogonalise flagship", "op": "orthogonalise", "batch": 1, "rows": 4096, "cols": 16384,
         "dtype": "bf16"},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    op = rng.choice(["quantise", "product", "product", "linear", "orthogonalise", "muon"])
    if op == "quantise":
        cols = _log_int(rng, 1, 8192)
        return {"op": op, "rows": _log_int(rng, 1, min(32768, 2 ** 25 // cols)), "cols": cols,
                "dtype": rng.choice(["bf16", "fp32"]), "fmt": rng.choice(["e4m3", "e5m2"]),
                "tile": rng.random() < 0.4, "both": rng.random() < 0.5}
    if op == "product":
        return {"op": op, "M": _log_int(rng, 1, 8192), "N": _log_int(rng, 8, 16384), "K": _log_int(rng, 16, 8192),
                "fa": rng.choice(["e4m3", "e5m2"]), "fb": rng.choice(["e4m3", "e5m2"]),
                "out": rng.choice(["bf16", "fp32"]), "beta": rng.choice([0.0, 0.0, 1.0])}
    if op == "linear":
        return {"op": op, "T": _log_int(rng, 1, 8192), "D": _log_int(rng, 32, 4096), "F": _log_int(rng, 32, 16384)}
    rows, cols = _log_int(rng, 1, 4096), _log_int(rng, 1, 4096)
    if rng.random() < 0.5:
        cols = max(1, min(16384, 4 * rows))
    batch = rng.choice([1, 1, 2, 3, 5]) if rows * cols <= 2 ** 21 else 1
    if op == "muon":
        return {"op": op, "batch": batch, "rows": rows, "cols": cols, "wd": rng.choice([0.0, 0.01])}
    return {"op": op, "batch": batch, "rows": rows, "cols": cols, "dtype": rng.choice(["fp32", "bf16"])}


# ----------------------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------------------
def _device() -> torch.device:
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _activations(shape, gen, std: float = 1.0) -> torch.Tensor:
    """Activations / output gradients: normal, with rows and channels of different size (a few large channels)."""
    x = torch.randn(shape, generator=gen, device=gen.device)
    x *= std * torch.exp(0.5 * torch.randn(shape[0], 1, generator=gen, device=gen.device))
    return x.mul_(torch.exp(0.7 * torch.randn(1, shape[1], generator=gen, device=gen.device)))


def _gradients(batch: int, rows: int, cols: int, gen) -> torch.Tensor:
    """Weight gradients: products of output gradients and activations over few effective directions, plus noise."""
    rank = max(1, min(rows, cols) // 4)
    dy = torch.randn(batch, rows, rank, generator=gen, device=gen.device)
    dy *= torch.exp(0.5 * torch.randn(batch, 1, rank, generator=gen, device=gen.device))
    x = torch.randn(batch, rank, cols, generator=gen, device=gen.device)
    g = torch.bmm(dy, x).mul_(1e-3)
    return g.add_(torch.randn(batch, rows, cols, generator=gen, device=gen.device), alpha=5e-4 * math.sqrt(rank))


def _operand(rows: int, k: int, fmt: str, gen) -> tuple[torch.Tensor, torch.Tensor]:
    """A quantised operand as a program holds it: 8-bit data [rows, K padded to 128] and exponent bytes [K blocks, rows]."""
    kb = -(-k // BLOCK)
    x = torch.zeros(rows, kb * BLOCK, device=gen.device)
    x[:, :k] = _activations((rows, k), gen)
    v = x.view(rows, kb, BLOCK)
    e = _block_exponent(v.abs().amax(dim=2), fmt)
    data = (v * _pow2(-e.unsqueeze(2))).view(rows, -1).to(DTYPES[fmt])
    return data, (e + 127).to(torch.uint8).t().contiguous()


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=_device())
    gen.manual_seed(int(seed))
    s = dict(case)
    op = case["op"]
    if op == "quantise":
        s["x"] = _activations((case["rows"], case["cols"]), gen).to(FLOATS[case["dtype"]])
    elif op == "product":
        s["a"], s["sa"] = _operand(case["M"], case["K"], case["fa"], gen)
        s["b"], s["sb"] = _operand(case["N"], case["K"], case["fb"], gen)
        if case["beta"]:
            s["c"] = torch.randn(case["M"], case["N"], generator=gen, device=gen.device).mul_(math.sqrt(case["K"])).to(
                FLOATS[case["out"]])
    elif op == "linear":
        T, D, F = case["T"], case["D"], case["F"]
        s["x"] = _activations((T, D), gen).bfloat16()
        s["w"] = (torch.randn(F, D, generator=gen, device=gen.device) / math.sqrt(D)).bfloat16()
        s["dy"] = _activations((T, F), gen, 1e-3).bfloat16()
    else:
        g = _gradients(case["batch"], case["rows"], case["cols"], gen)
        if op == "orthogonalise":
            s["x"] = (g if case["batch"] > 1 else g[0]).to(FLOATS[case["dtype"]])
        else:
            s["g"] = g
            s["m"] = _gradients(case["batch"], case["rows"], case["cols"], gen).mul_(10.0)
            s["w"] = torch.randn(g.shape, generator=gen, device=gen.device) / math.sqrt(case["cols"])
            s["copy"] = s["w"].bfloat16()
    return s


# ----------------------------------------------------------------------------------------------------------------
# plain forms (fp32)
# ----------------------------------------------------------------------------------------------------------------
def _pow2(e: torch.Tensor) -> torch.Tensor:
    """2^e in fp32, exactly, for integer -127 <= e <= 127 (a device's pow or exp2 may round)."""
    normal = ((e + 127) << 23).to(torch.int32).view(torch.float32)
    return torch.where(e == -127, torch.full_like(normal, 2.0 ** -127), normal)


def _block_exponent(amax: torch.Tensor, fmt: str) -> torch.Tensor:
    """The smallest e with amax <= FMAX * 2^e (FMAX = 0.875 * 2^top), at least -127; int32."""
    mant, ex = torch.frexp(amax)
    top = 9 if fmt == "e4m3" else 16
    return (ex - top + (mant > 0.875).to(ex.dtype)).clamp(min=-127)


def _values(x: torch.Tensor, fmt: str, tile: bool) -> torch.Tensor:
    """The values that the 8-bit form of x [R, K] stands for (fp32)."""
    R, K = x.shape
    rb, kb = -(-R // BLOCK), -(-K // BLOCK)
    p = torch.zeros(rb * BLOCK if tile else R, kb * BLOCK, device=x.device)
    p[:R, :K] = x
    v = p.view(rb, BLOCK, kb, BLOCK) if tile else p.view(R, 1, kb, BLOCK)
    e = _block_exponent(v.abs().amax(dim=(1, 3), keepdim=True), fmt)
    q = (v * _pow2(-e)).to(DTYPES[fmt]).float()
    return (q * _pow2(e)).view(p.shape)[:R, :K]


def _stands_for(data: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    rows, kp = data.shape
    e = scale.t().to(torch.int32) - 127
    return (data.float().view(rows, kp // BLOCK, BLOCK) * _pow2(e.unsqueeze(2))).view(rows, kp)


def _newton_schulz(u: torch.Tensor, steps: int = 5) -> torch.Tensor:
    x = u / (u.square().sum(dim=(-2, -1), keepdim=True).sqrt() + NS_EPS)
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1)
    for _ in range(steps):
        a = torch.matmul(x, x.transpose(-2, -1))
        x = NS_A * x + torch.matmul(NS_B * a + NS_C * torch.matmul(a, a), x)
    return x.transpose(-2, -1) if tall else x


MUON = {"lr": 0.02, "beta": 0.95}


def _plain(s: dict):
    op = s["op"]
    if op == "quantise":
        x = s["x"].float()
        if not s["both"]:
            return _values(x, s["fmt"], s["tile"]).bfloat16()
        return [_values(x, s["fmt"], s["tile"]).bfloat16(),
                _values(x.t(), s["fmt"], s["tile"]).bfloat16().contiguous()]
    if op == "product":
        c = torch.matmul(_stands_for(s["a"], s["sa"]), _stands_for(s["b"], s["sb"]).t())
        if s["beta"]:
            return s["c"].copy_(c.add_(s["c"].float(), alpha=s["beta"]))
        return c.to(FLOATS[s["out"]])
    if op == "linear":
        x, w, dy = s["x"].float(), s["w"].float(), s["dy"].float()
        wq = _values(w, "e4m3", True)
        y = torch.matmul(_values(x, "e4m3", False), wq.t())
        dx = torch.matmul(_values(dy, "e5m2", False), wq)
        dw = torch.matmul(_values(dy.t(), "e5m2", False), _values(x.t(), "e4m3", False).t())
        return [y.bfloat16(), dx.bfloat16(), dw]
    if op == "orthogonalise":
        return _newton_schulz(s["x"].float()).to(s["x"].dtype).contiguous()
    m, w = s["m"], s["w"]
    m.mul_(MUON["beta"]).add_(s["g"])
    o = _newton_schulz(s["g"] + MUON["beta"] * m)
    w.mul_(1.0 - MUON["lr"] * s["wd"]).sub_(o, alpha=MUON["lr"] * math.sqrt(max(1.0, s["rows"] / s["cols"])))
    s["copy"].copy_(w)
    return [w, m, s["copy"]]


# ----------------------------------------------------------------------------------------------------------------
# the framework's operators
# ----------------------------------------------------------------------------------------------------------------
def _own(s: dict):
    from dllm.ops import fp8, muon

    op = s["op"]
    if op == "quantise":
        if not s["both"]:
            return fp8.dequantize_fp8(fp8.quantize_fp8(s["x"], s["fmt"], tile=s["tile"]), torch.bfloat16)
        q, qt = fp8.quantize_fp8_both(s["x"], s["fmt"], s["fmt"], tile=s["tile"])
        return [fp8.dequantize_fp8(q, torch.bfloat16), fp8.dequantize_fp8(qt, torch.bfloat16)]
    if op == "product":
        a, b = fp8.BlockFP8(s["a"], s["sa"], s["K"]), fp8.BlockFP8(s["b"], s["sb"], s["K"])
        if s["beta"]:
            return fp8.gemm_fp8(a, b, out=s["c"], beta=s["beta"])
        return fp8.gemm_fp8(a, b, out_dtype=FLOATS[s["out"]])
    if op == "linear":
        y, saved = fp8.linear_fp8(s["x"], s["w"])
        dx, dw = fp8.linear_fp8_bwd(s["dy"], saved)
        return [y, dx, dw]
    if op == "orthogonalise":
        return muon.orthogonalize(s["x"])
    muon.muon_step_(s["w"], s["g"], s["m"], lr=MUON["lr"], beta=MUON["beta"], wd=s["wd"], copy=s["copy"])
    return [s["w"], s["m"], s["copy"]]


def run(state: dict):
    return _own(state) if own else _plain(state)


# ----------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------------------------
def _float_bytes(name: str) -> int:
    return 2 if name == "bf16" else 4


def work(case: dict) -> dict:
    op = case["op"]
    if op == "quantise":
        n = case["rows"] * case["cols"]
        ways = 2 if case["both"] else 1
        # x once, the values of each orientation as bf16 (the 8-bit form in between is the operator's own)
        return {"bytes": n * (_float_bytes(case["dtype"]) + 2 * ways), "flops": 2 * n * ways}
    if op == "product":
        M, N, K = case["M"], case["N"], case["K"]
        kb = -(-K // BLOCK)
        out = M * N * _float_bytes(case["out"]) * (2 if case["beta"] else 1)
        return {"bytes": (M + N) * (K + kb) + out, "flops": 2 * M * N * K}
    if op == "linear":
        T, D, F = case["T"], case["D"], case["F"]
        return {"bytes": 2 * (T * D + F * D + T * F) + 2 * (T * F + T * D) + 4 * F * D, "flops": 6 * T * D * F}
    b, m, n = case["batch"], min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
    flops = b * (3 * m * m * n + 17 * m * m * m)
    if op == "orthogonalise":
        return {"bytes": 2 * b * m * n * _float_bytes(case["dtype"]), "flops": flops}
    return {"bytes": b * m * n * (4 + 8 + 8 + 2), "flops": flops}


# ----------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ----------------------------------------------------------------------------------------------------------------
def _double_pow2(e: torch.Tensor) -> torch.Tensor:
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_values(x: torch.Tensor, fmt: str, tile: bool) -> torch.Tensor:
    """Block by block from the definition: power-of-two scale, then the nearest number of the 8-bit grid, ties to even."""
    x = x.double()
    R, K = x.shape
    rows = torch.arange(R, device=x.device) // (BLOCK if tile else 1)
    cols = torch.arange(K, device=x.device) // BLOCK
    nr, nc = int(rows[-1]) + 1, int(cols[-1]) + 1
    amax = torch.zeros(nr, nc, dtype=torch.float64, device=x.device)
    colmax = torch.zeros(R, nc, dtype=torch.float64, device=x.device)
    colmax.scatter_reduce_(1, cols.expand(R, K), x.abs(), "amax")
    amax.scatter_reduce_(0, rows.unsqueeze(1).expand(R, nc), colmax, "amax")
    e = torch.ceil(torch.log2(amax.clamp(min=1e-40) / FMAX[fmt]))
    e += (amax > FMAX[fmt] * _double_pow2(e)).double()              # log2 may round across a power of two
    e -= (amax <= FMAX[fmt] * _double_pow2(e - 1)).double()
    s = _double_pow2(e.clamp(min=-127))[rows][:, cols]
    v = x / s
    bits, low = (3, -6) if fmt == "e4m3" else (2, -14)
    mag = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** low)))
    mag -= (_double_pow2(mag) > v.abs().clamp(min=2.0 ** low)).double()
    mag += (_double_pow2(mag + 1) <= v.abs()).double()
    step = _double_pow2(mag - bits)
    return torch.round(v / step) * step * s


def _exact_operand(data: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    factor = _double_pow2(scale.to(torch.int64) - 127).repeat_interleave(BLOCK, dim=0).t()
    return data.double() * factor


def _exact_orthogonal(u: torch.Tensor) -> torch.Tensor:
    """The five quintic steps act on the singular values only; done on the products in 64 bits, matrix by matrix."""
    out = []
    for g in u.double().reshape(-1, *u.shape[-2:]):
        x = g / (torch.linalg.matrix_norm(g) + NS_EPS)
        wide = x.shape[0] <= x.shape[1]
        for _ in range(5):
            gram = x @ x.t() if wide else x.t() @ x
            p = NS_B * gram + NS_C * (gram @ gram)
            p.diagonal().add_(NS_A)
            x = p @ x if wide else x @ p
        out.append(x)
    return torch.stack(out).view(u.shape)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantise":
        q = _exact_values(s["x"], case["fmt"], case["tile"])
        return [q, _exact_values(s["x"].t(), case["fmt"], case["tile"]).contiguous()] if case["both"] else q
    if op == "product":
        c = _exact_operand(s["a"], s["sa"]) @ _exact_operand(s["b"], s["sb"]).t()
        return c + case["beta"] * s["c"].double() if case["beta"] else c
    if op == "linear":
        w = _exact_values(s["w"], "e4m3", True)
        y = _exact_values(s["x"], "e4m3", False) @ w.t()
        dx = _exact_values(s["dy"], "e5m2", False) @ w
        dw = _exact_values(s["dy"].t(), "e5m2", False) @ _exact_values(s["x"].t(), "e4m3", False).t()
        return [y, dx, dw]
    if op == "orthogonalise":
        return _exact_orthogonal(s["x"])
    g, w = s["g"].double(), s["w"].double()
    m = MUON["beta"] * s["m"].double() + g
    o = _exact_orthogonal(g + MUON["beta"] * m)
    w = w * (1.0 - MUON["lr"] * case["wd"]) - MUON["lr"] * math.sqrt(max(1.0, case["rows"] / case["cols"])) * o
    return [w, m, w]
