// Block-scaled 8-bit floating point (OCP e4m3 / e5m2) on gfx950: operand format, quantiser and product arguments.
//
// An operand is data [R, Kp] (8-bit, row-major, Kp = K rounded up to 128, zeros behind K) and one exponent byte per row
// and 128 k, scale [Kp / 128][R]: element (r, k) stands for data[r][k] * 2^(scale[k / 128][r] - 127).  Powers of two,
// because the gfx950 matrix instruction applies them itself (v_mfma_scale_f32_16x16x128_f8f6f4, one instruction per
// 128 k: a block of 128 is exactly its depth), scaling costs no vector instruction in the main loop, and dividing by
// them is exact, so a value is rounded once.  K-block-major scales: a K step reads consecutive bytes of its rows.
#pragma once
#include "common.h"

namespace dllm {

enum Fp8Fmt : int { F8_E4M3 = 0, F8_E5M2 = 1 };   // also the matrix instruction's operand format codes

// 2^(b - 127) of an exponent byte (b = 255: NaN, b = 0: the subnormal 2^-127)
__device__ __forceinline__ float e8m0_to_f32(uint32_t b) {
  return b == 0 ? __uint_as_float(0x00400000u) : b == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(b << 23);
}
// exponent byte of a block with largest finite magnitude `amax` (bits): the smallest e with amax <= FMAX 2^e.  FMAX =
// 1.75 * 2^8 (e4m3: 448) or 1.75 * 2^15 (e5m2: 57344), so e = exponent(amax) - top, plus one where the mantissa passes 1.75
__device__ __forceinline__ uint32_t e8m0_of_amax(uint32_t bits, int fmt) {
  const int e = (int)((bits + 0x1fffffu) >> 23) - (fmt == F8_E4M3 ? 8 : 15);
  return (uint32_t)max(e, 0);
}
// 2^(127 - b): the exact reciprocal the quantiser multiplies by (b <= 247)
__device__ __forceinline__ float e8m0_inv(uint32_t b) { return __uint_as_float((254u - b) << 23); }

struct QuantArgs {
  const void* x; long ldx; int R, C;         // x [R, C] (elements)
  uint8_t* q; long ldq; uint8_t* sq; long ldsq;      // x's 8-bit form [R, C padded], scales [C blocks][R] (q may be null)
  uint8_t* qt; long ldqt; uint8_t* sqt; long ldsqt;  // x^T's [C, R padded], scales [R blocks][C] (qt may be null)
  int fmt, fmt_t, tile;
};

struct Fp8GemmArgs {
  const uint8_t* A; long lda; const uint8_t* SA; long ldsa;
  const uint8_t* B; long ldb; const uint8_t* SB; long ldsb;
  void* C; long ldc; const void* aux; void* aux_out; long ldaux;
  int M, N, nk;            // nk: 128-deep K steps
  float alpha, beta;
  int act;
  int tile, ksplit;        // output tile; K slices (fp32 sums of slice s at ws + s M N)
  float* ws;
};

}  // namespace dllm
