"""Device ops: MFMA GEMMs with fused FFN epilogues, RNG, fused optimizers (HIP on GPU, torch on CPU)."""
from .activations import act_fwd, act_grad  # noqa: F401
from .elementwise import adam_step_, cast_, rng_normal_, sgd_step_  # noqa: F401
from .gemm import gemm  # noqa: F401
from .fp8 import (BlockFP8, dequantize_fp8, fp8_empty, gemm_fp8, linear_fp8, linear_fp8_bwd, quantize_fp8,  # noqa: F401
                  quantize_fp8_both, quantize_fp8_t)
from .muon import muon_scale, muon_split_step_, muon_step_, orthogonalize  # noqa: F401
