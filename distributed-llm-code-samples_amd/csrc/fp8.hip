// Block-scaled 8-bit quantiser, read-back and matrix product (fp8.h has the format).
#include <type_traits>

#include "fp8.h"
#include "nt8.h"

namespace dllm {

typedef __attribute__((ext_vector_type(8))) int i32x8_t;
typedef __attribute__((ext_vector_type(4))) int i32x4_t;
typedef __attribute__((ext_vector_type(2))) float f32x2_t;

// ----------------------------------------------------------------------------------------------
// quantiser: one block of 256 threads per 128x128 tile of x, one read of x for both orientations
//
// Thread (g, j) = (t / 16, t % 16) holds rows 8g .. 8g+7 and columns 8j .. 8j+7 of the tile in registers.  A row's 128
// columns sit in 16 neighbouring lanes (row scales: 4 lane exchanges), a column's 128 rows in 16 values of g (column
// scales: lane exchanges over the wave's four g, then LDS over the four waves).  x^T leaves through LDS so that its rows
// are written in whole 128-B lines.  Bound by HBM: reads x once and writes one byte per element and orientation.
// ----------------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<uint16_t>(uint16_t v) { return bf2f(v); }
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }

// magnitude bits of v, 0 for inf / NaN (the block's scale comes from its finite elements)
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}

// four values (already scaled into range) -> four 8-bit codes.  Rounds to nearest even; |v| <= FMAX by construction, so
// nothing finite saturates.  e4m3 has no infinity: inf becomes NaN; e5m2 keeps it.
template <int FMT>
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  int w = 0;
  if constexpr (FMT == F8_E4M3) {
    w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  } else {
    w = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, w, false);
    w = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, w, true);
  }
  return (uint32_t)w;
}
__device__ __forceinline__ uint32_t pack4f(int fmt, float a, float b, float c, float d) {
  return fmt == F8_E4M3 ? pack4<F8_E4M3>(a, b, c, d) : pack4<F8_E5M2>(a, b, c, d);
}

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void fp8_quantize_kernel(QuantArgs p) {
  constexpr int QT_LD = 128 + 16;   // LDS row of x^T codes (16-B aligned, off the 256-B bank period)
  __shared__ __attribute__((aligned(16))) uint8_t tbuf[128 * QT_LD];
  __shared__ uint32_t cmax[4][128];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int g = t >> 4, j = t & 15;
  const int tiles_c = (p.C + 127) >> 7;
  const int tr = blockIdx.x / tiles_c, tc = blockIdx.x - tr * tiles_c;
  const long r0 = (long)tr * 128, c0 = (long)tc * 128;
  const T* x = (const T*)p.x + r0 * p.ldx + c0;
  const int nr = (int)min((long)128, p.R - r0), nc = (int)min((long)128, p.C - c0);

  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 8 * g + i, c = 8 * j;
    if (r < nr && c < nc) {
      const T* s = x + (long)r * p.ldx + c;
      if (VEC && c + 8 <= nc) {
        if constexpr (sizeof(T) == 2) {
          const uint4 u = *(const uint4*)s;
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            v[i][2 * k] = __uint_as_float(w[k] << 16);
            v[i][2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
          }
        } else {
          const f32x4_t a = *(const f32x4_t*)s, b = *(const f32x4_t*)(s + 4);
#pragma unroll
          for (int k = 0; k < 4; ++k) { v[i][k] = a[k]; v[i][4 + k] = b[k]; }
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[i][k] = c + k < nc ? to_f32<T>(s[k]) : 0.f;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[i][k] = 0.f;
    }
  }

  uint32_t rowmax[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = max(m, finite_bits(v[i][k]));
    rowmax[i] = m;
  }
  uint32_t tilemax = 0;
  if (p.tile) {
#pragma unroll
    for (int i = 0; i < 8; ++i) tilemax = max(tilemax, rowmax[i]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) tilemax = max(tilemax, (uint32_t)__shfl_xor((int)tilemax, d));
    if (lane == 0) cmax[0][wave] = tilemax;
    __syncthreads();
    tilemax = max(max(cmax[0][0], cmax[0][1]), max(cmax[0][2], cmax[0][3]));
    __syncthreads();
  }

  if (p.q != nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t m = rowmax[i];
      if (p.tile) {
        m = tilemax;
      } else {
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
      }
      const uint32_t b = e8m0_of_amax(m, p.fmt);
      const float s = e8m0_inv(b);
      const int r = 8 * g + i;
      if (r < nr) {
        uint2 o;
        o.x = pack4f(p.fmt, v[i][0] * s, v[i][1] * s, v[i][2] * s, v[i][3] * s);
        o.y = pack4f(p.fmt, v[i][4] * s, v[i][5] * s, v[i][6] * s, v[i][7] * s);
        *(uint2*)(p.q + (r0 + r) * p.ldq + c0 + 8 * j) = o;
        if (j == 0) p.sq[(long)tc * p.ldsq + r0 + r] = (uint8_t)b;
      }
    }
  }

  if (p.qt != nullptr) {
    uint32_t cm[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) cm[k] = tilemax;
    if (!p.tile) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, finite_bits(v[i][k]));
        m = max(m, (uint32_t)__shfl_xor((int)m, 16));
        m = max(m, (uint32_t)__shfl_xor((int)m, 32));
        if (lane < 16) cmax[wave][8 * j + k] = m;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int c = 8 * j + k;
        cm[k] = max(max(cmax[0][c], cmax[1][c]), max(cmax[2][c], cmax[3][c]));
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t b = e8m0_of_amax(cm[k], p.fmt_t);
      const float s = e8m0_inv(b);
      uint2 o;
      o.x = pack4f(p.fmt_t, v[0][k] * s, v[1][k] * s, v[2][k] * s, v[3][k] * s);
      o.y = pack4f(p.fmt_t, v[4][k] * s, v[5][k] * s, v[6][k] * s, v[7][k] * s);
      *(uint2*)(tbuf + (8 * j + k) * QT_LD + 8 * g) = o;
      if (g == 0 && 8 * j + k < nc) p.sqt[(long)tr * p.ldsqt + c0 + 8 * j + k] = (uint8_t)b;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = 32 * i + (t >> 3), o = 16 * (t & 7);
      if (c < nc) *(uint4*)(p.qt + (c0 + c) * p.ldqt + r0 + o) = *(const uint4*)(tbuf + c * QT_LD + o);
    }
  }
}

// read-back: 8 codes and their block's exponent -> 8 values (exact in fp32 above the subnormals; bf16 rounds to even)
template <typename T>
__global__ __launch_bounds__(256) void fp8_dequantize_kernel(const uint8_t* q, long ldq, const uint8_t* sq, long ldsq,
                                                             T* out, long ldo, long R, int K, int fmt) {
  const int g8 = (K + 7) >> 3;
  const long n = R * g8;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    const long r = i / g8;
    const int c = (int)(i - r * g8) * 8;
    const uint2 w = *(const uint2*)(q + r * ldq + c);
    const float s = e8m0_to_f32(sq[(long)(c >> 7) * ldsq + r]);
    float v[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int u = (int)(h ? w.y : w.x);
      f32x2_t a, b;
      if (fmt == F8_E4M3) { a = __builtin_amdgcn_cvt_pk_f32_fp8(u, false); b = __builtin_amdgcn_cvt_pk_f32_fp8(u, true); }
      else { a = __builtin_amdgcn_cvt_pk_f32_bf8(u, false); b = __builtin_amdgcn_cvt_pk_f32_bf8(u, true); }
      v[4 * h] = a[0] * s; v[4 * h + 1] = a[1] * s; v[4 * h + 2] = b[0] * s; v[4 * h + 3] = b[1] * s;
    }
    T* o = out + r * ldo + c;
    if (c + 8 <= K && (((uintptr_t)o) & 15) == 0) {
      if constexpr (sizeof(T) == 2) {
        uint4 u;
        u.x = f2bf(v[0]) | ((uint32_t)f2bf(v[1]) << 16); u.y = f2bf(v[2]) | ((uint32_t)f2bf(v[3]) << 16);
        u.z = f2bf(v[4]) | ((uint32_t)f2bf(v[5]) << 16); u.w = f2bf(v[6]) | ((uint32_t)f2bf(v[7]) << 16);
        *(uint4*)o = u;
      } else {
        *(f32x4_t*)o = f32x4_t{v[0], v[1], v[2], v[3]};
        *(f32x4_t*)(o + 4) = f32x4_t{v[4], v[5], v[6], v[7]};
      }
    } else {
      for (int k = 0; k < 8 && c + k < K; ++k) {
        if constexpr (sizeof(T) == 2) o[k] = f2bf(v[k]);
        else o[k] = v[k];
      }
    }
  }
}

// ----------------------------------------------------------------------------------------------
// product C = alpha A B^T + beta C (and the activation epilogues), any M, N: 128x128 tile, 4 waves of 64x64
//
// Both operands are K-contiguous; a K step is one 128-byte line per row.  LDS rows of 128 B with the 16-B chunk index
// XOR-swizzled by (row >> 1) & 7, filled by LDS-DMA from swizzled source addresses and read by ds_read_b128 without bank
// conflicts.  A lane's 32 bytes of a fragment are chunks g and 4 + g (g = lane / 16) of its row, in A and B alike: a
// permutation of k inside the block, which the sum and the block's one scale do not see.  The operands are swapped in
// the matrix instruction (B first), so a lane ends with 4 consecutive columns of one row of C.
// ----------------------------------------------------------------------------------------------
__device__ __forceinline__ void lds_dma16(const uint8_t* src, DLLM_LDS char* dst) {
  __builtin_amdgcn_global_load_lds((const DLLM_GLB void*)src, (DLLM_LDS void*)dst, 16, 0, 0);
}

template <int FB, int FA>
__device__ __forceinline__ f32x4_t mfma_f8(i32x8_t b, i32x8_t a, f32x4_t c, int sb, int sa) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, c, FB, FA, 0, sb, 0, sa);
}

// The 8-bit matrix instruction adds the products of 8 neighbouring k with 13 bits below the largest of them (measured: a
// product under 2^-13 of its neighbour is lost whole, the sums of 8 then add up in fp32): about 4e-5 of the result, a
// hundredth of bf16's half step 2^-8 but hundreds of fp32's.  So a bf16 result is computed on it, and an fp32 result on
// the bf16 instruction, which keeps fp32 sums (5e-7 at K = 8192): codes times their scale are bf16 numbers, exactly
// (8 exponent bits; only values under 2^-126 may round), so the operands convert in registers on their way from LDS.
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
template <int FMT>
__device__ __forceinline__ void codes_to_bf16(i32x8_t q, float s, bf16x8_t (&o)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bf16x2_t v[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int w = q[2 * i + h];
      if constexpr (FMT == F8_E4M3) {
        v[2 * h] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, false);
        v[2 * h + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, true);
      } else {
        v[2 * h] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, s, false);
        v[2 * h + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, s, true);
      }
    }
    o[i] = bf16x8_t{v[0][0], v[0][1], v[1][0], v[1][1], v[2][0], v[2][1], v[3][0], v[3][1]};
  }
}

template <typename OutT> __device__ __forceinline__ float ld_out(const void* p, long i) {
  if constexpr (sizeof(OutT) == 2) return bf2f(((const uint16_t*)p)[i]);
  else return ((const float*)p)[i];
}
template <typename OutT> __device__ __forceinline__ void st_out(void* p, long i, float v) {
  if constexpr (sizeof(OutT) == 2) ((uint16_t*)p)[i] = f2bf(v);
  else ((float*)p)[i] = v;
}

// epilogue of 4 consecutive columns n .. n+3 of row m
template <int EPI, typename OutT>
__device__ __forceinline__ void f8_epi4(const Fp8GemmArgs& p, int m, int n, f32x4_t v) {
  if (m >= p.M) return;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (n + r >= p.N) return;
    const long i = (long)m * p.ldc + n + r, ia = (long)m * p.ldaux + n + r;
    float o = v[r];
    if constexpr (EPI == EPI_STORE) {
      o *= p.alpha;
      if (p.beta != 0.f) o += p.beta * ld_out<OutT>(p.C, i);
    } else if constexpr (EPI == EPI_ACT) {
      if (p.aux_out) st_out<OutT>(p.aux_out, ia, o);
      o = act_fwd(p.act, o);
    } else {
      o *= act_grad(p.act, ld_out<OutT>(p.aux, ia));
    }
    st_out<OutT>(p.C, i, o);
  }
}

template <int EPI, typename OutT, int FA, int FB>
__global__ __launch_bounds__(256, 2) void fp8_gemm_128(Fp8GemmArgs p) {
  constexpr int TB = 128 * 128;
  __shared__ __attribute__((aligned(16))) char smem[4 * TB];   // [buffer][A, B]
  DLLM_LDS char* lds = (DLLM_LDS char*)smem;
  const int t = threadIdx.x, lane = t & 63;
  const int wid = __builtin_amdgcn_readfirstlane(t >> 6);
  const int tiles_n = (p.N + 127) >> 7;
  const int bid = xcd_remap(blockIdx.x, gridDim.x);
  const int m0 = (bid / tiles_n) * 128, n0 = (bid % tiles_n) * 128;
  const int i15 = lane & 15, g = lane >> 4, wr = wid >> 1, wc = wid & 1;

  // rows past the end re-load the last row: their products are never stored
  const uint8_t *ap[4], *bp[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int q = i * 4 + wid, row = 8 * q + (lane >> 3), c = ((lane & 7) ^ ((row >> 1) & 7)) * 16;
    ap[i] = p.A + (long)min(m0 + row, p.M - 1) * p.lda + c;
    bp[i] = p.B + (long)min(n0 + row, p.N - 1) * p.ldb + c;
  }
  auto stage = [&](int kt, int buf) {
    DLLM_LDS char* d = lds + buf * 2 * TB;
#pragma unroll
    for (int i = 0; i < 4; ++i) lds_dma16(ap[i] + (long)kt * 128, d + (i * 4 + wid) * 1024);
#pragma unroll
    for (int i = 0; i < 4; ++i) lds_dma16(bp[i] + (long)kt * 128, d + TB + (i * 4 + wid) * 1024);
  };
  auto frag = [&](const DLLM_LDS char* tile, int row) {
    const int f = (row >> 1) & 7;
    const i32x4_t lo = *(const DLLM_LDS i32x4_t*)(tile + row * 128 + ((g ^ f) << 4));
    const i32x4_t hi = *(const DLLM_LDS i32x4_t*)(tile + row * 128 + (((4 + g) ^ f) << 4));
    return i32x8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  int am[4], bn[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    am[i] = min(m0 + wr * 64 + i * 16 + i15, p.M - 1);
    bn[i] = min(n0 + wc * 64 + i * 16 + i15, p.N - 1);
  }

  f32x4_t acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[i][k] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  if (p.nk > 0) stage(0, 0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  for (int kt = 0; kt < p.nk; ++kt) {
    if (kt + 1 < p.nk) stage(kt + 1, (kt + 1) & 1);
    const DLLM_LDS char* As = lds + (kt & 1) * 2 * TB;
    int sa[4], sb[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sa[i] = p.SA[(long)kt * p.ldsa + am[i]];
      sb[i] = p.SB[(long)kt * p.ldsb + bn[i]];
    }
    i32x8_t fa[4], fb[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      fa[i] = frag(As, wr * 64 + i * 16 + i15);
      fb[i] = frag(As + TB, wc * 64 + i * 16 + i15);
    }
    if constexpr (sizeof(OutT) == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[i][k] = mfma_f8<FB, FA>(fb[k], fa[i], acc[i][k], sb[k], sa[i]);
    } else {
      bf16x8_t xb[4][4];
#pragma unroll
      for (int k = 0; k < 4; ++k) codes_to_bf16<FB>(fb[k], e8m0_to_f32(sb[k]), xb[k]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        bf16x8_t xa[4];
        codes_to_bf16<FA>(fa[i], e8m0_to_f32(sa[i]), xa);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[i][k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xb[k][q], xa[q], acc[i][k], 0, 0, 0);
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k)
      f8_epi4<EPI, OutT>(p, m0 + wr * 64 + i * 16 + i15, n0 + wc * 64 + k * 16 + 4 * g, acc[i][k]);
}

// ----------------------------------------------------------------------------------------------
// 256x256 tiles on the 8-phase loop (nt8.h), one matrix instruction per 16x16 fragment pair and K step.
//
// Scales: a lane's four A rows of a half are consecutive rows of C (nt8.h), so one 32-bit word of the K step's scale row
// holds them, and 16 bits its two B rows; the matrix instruction picks the byte (op_sel), so scaling costs two 4-byte and
// two 2-byte loads per K step and nothing else.  An odd number of K steps runs one more: the last step again, with scale
// bytes 0 on both sides, 2^-254 of it, which leaves every fp32 sum as it is.
// ----------------------------------------------------------------------------------------------
typedef uint32_t u32_any __attribute__((aligned(1)));
typedef uint16_t u16_any __attribute__((aligned(1)));

template <int FMT>
__device__ __forceinline__ bf16x8_t codes8(int w0, int w1, float s) {
  bf16x2_t v[4];
  if constexpr (FMT == F8_E4M3) {
    v[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, false); v[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, true);
    v[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, false); v[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, true);
  } else {
    v[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w0, s, false); v[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w0, s, true);
    v[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w1, s, false); v[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w1, s, true);
  }
  return bf16x8_t{v[0][0], v[0][1], v[1][0], v[1][1], v[2][0], v[2][1], v[3][0], v[3][1]};
}

// EXACT: fp32 sums -- codes times scale as bf16 on the bf16 instruction (see codes_to_bf16), converted in the shadow of the
// matrix instructions: 3 conversions (4 cycles each) per matrix instruction (16 cycles)
template <int FA, int FB, bool EXACT>
struct F8Trait {
  const uint8_t *sa, *sb;      // scale bytes of K step 0
  long ldsa, ldsb;
  int nk, nk2;
  uint32_t oa[2], ob[2];       // the lane's scale bytes in a scale row, per half
  uint32_t sh;                 // right shifts of the four words, 8 bits each: words that would pass the row's end start
                               // earlier (rows that far are never stored)
  int keep;                    // 0 if the current pair's second step is the one behind the last
  int wa[2][2], wb[2][2];      // [K step parity][half]; as loaded until the step's first phase shifts them

  __device__ __forceinline__ void begin(const Fp8GemmArgs& p, int m0, int n0, int wid, int lane) {
    sa = p.SA; sb = p.SB; ldsa = p.ldsa; ldsb = p.ldsb;
    nk = p.nk; nk2 = (p.nk + 1) >> 1;
    sh = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int ra = m0 + 128 * h + (wid >> 2) * 64 + 4 * (lane & 15), rb = n0 + 128 * h + (wid & 3) * 32 + 2 * (lane & 15);
      oa[h] = (uint32_t)min(ra, p.M - 4);
      ob[h] = (uint32_t)min(rb, p.N - 2);
      sh |= (uint32_t)min(8 * (ra - (int)oa[h]), 24) << (8 * h) | (uint32_t)min(8 * (rb - (int)ob[h]), 8) << (16 + 8 * h);
    }
    fetch<0>(0);
    fetch<1>(1);
  }
  __device__ __forceinline__ int step(int pair) const { return 2 * pair + 1 < nk ? 128 : 0; }
  __device__ __forceinline__ int advance(const char*& an, const char*& bn, int it) {
    keep = 2 * it + 1 < nk ? -1 : 0;
    if (it + 1 < nk2) {
      an += 256;
      bn += 256;
      return step(it + 1);
    }
    return step(it);
  }
  template <int ODD>
  __device__ __forceinline__ void fetch(int kt) {
    const int k = min(kt, nk - 1);
    const uint8_t *a = sa + (long)k * ldsa, *b = sb + (long)k * ldsb;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      wa[ODD][h] = (int)*(const u32_any*)(a + oa[h]);
      wb[ODD][h] = (int)*(const u16_any*)(b + ob[h]);
    }
  }
  template <class ODD> __device__ __forceinline__ void load(ODD, int it) { fetch<ODD::value>(2 * it + 2 + ODD::value); }

  template <int MT, int NT>
  static __device__ __forceinline__ void one(f32x4_t& c, const N8Frag& fa, const N8Frag& fb, int a, int b) {
    const i32x8_t x = __builtin_shufflevector(fa.lo, fa.hi, 0, 1, 2, 3, 4, 5, 6, 7);
    const i32x8_t y = __builtin_shufflevector(fb.lo, fb.hi, 0, 1, 2, 3, 4, 5, 6, 7);
    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(y, x, c, FB, FA, NT, b, MT, a);
  }
  template <int QM, int QN, int ODD>
  __device__ __forceinline__ void mma(f32x4_t (&c)[4][2], N8Frag (&fa)[4], N8Frag (&fb)[2]) {
    if constexpr (QM == 0 && QN == 0) {   // the step's first phase
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        wa[ODD][h] = (int)((uint32_t)wa[ODD][h] >> (sh >> (8 * h) & 31));
        wb[ODD][h] = (int)((uint32_t)wb[ODD][h] >> (sh >> (16 + 8 * h) & 31));
        if constexpr (ODD) { wa[ODD][h] &= keep; wb[ODD][h] &= keep; }
      }
    }
    const int a = wa[ODD][QM], b = wb[ODD][QN];
    if constexpr (EXACT) {
      // a fragment serves two phases; its conversion is repeated, not kept (32 more registers than there are)
#pragma unroll
      for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(fa[i].lo), "+v"(fa[i].hi));
#pragma unroll
      for (int i = 0; i < 2; ++i) asm volatile("" : "+v"(fb[i].lo), "+v"(fb[i].hi));
      auto scale = [](int w, int i) { return __uint_as_float(((uint32_t)w >> (8 * i) & 255u) << 23); };
      float sa4[4], sb2[2];
#pragma unroll
      for (int i = 0; i < 4; ++i) sa4[i] = scale(a, i);
      sb2[0] = scale(b, 0);
      sb2[1] = scale(b, 1);
      // quarter s of the fragments' codes (8 of 32); the next conversion is issued between a pair of matrix instructions
      // and the order is pinned: left to itself the compiler converts everything first and spills
      auto pick = [&](const N8Frag& f, int s, int k) { return s < 2 ? f.lo[2 * (s & 1) + k] : f.hi[2 * (s & 1) + k]; };
      auto cva = [&](int s, int mt) { return codes8<FA>(pick(fa[mt], s, 0), pick(fa[mt], s, 1), sa4[mt]); };
      auto cvb = [&](int s, int nt) { return codes8<FB>(pick(fb[nt], s, 0), pick(fb[nt], s, 1), sb2[nt]); };
      bf16x8_t y0 = cvb(0, 0), y1 = cvb(0, 1), x = cva(0, 0), yn0 = y0, yn1 = y1;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          bf16x8_t xn = x;
          c[mt][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(y0, x, c[mt][0], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
          if (mt < 3) xn = cva(s, mt + 1);
          else if (s < 3) xn = cva(s + 1, 0);
          __builtin_amdgcn_sched_barrier(0);
          c[mt][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(y1, x, c[mt][1], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
          if (s < 3 && mt == 1) yn0 = cvb(s + 1, 0);
          if (s < 3 && mt == 2) yn1 = cvb(s + 1, 1);
          __builtin_amdgcn_sched_barrier(0);
          x = xn;
        }
        y0 = yn0;
        y1 = yn1;
      }
      return;
    }
    one<0, 0>(c[0][0], fa[0], fb[0], a, b); one<0, 1>(c[0][1], fa[0], fb[1], a, b);
    one<1, 0>(c[1][0], fa[1], fb[0], a, b); one<1, 1>(c[1][1], fa[1], fb[1], a, b);
    one<2, 0>(c[2][0], fa[2], fb[0], a, b); one<2, 1>(c[2][1], fa[2], fb[1], a, b);
    one<3, 0>(c[3][0], fa[3], fb[0], a, b); one<3, 1>(c[3][1], fa[3], fb[1], a, b);
  }
};

// 8 columns n .. n + 7 of row m; `fast`: the tile is inside C and rows are 16-byte aligned
template <int EPI, typename OutT>
__device__ __forceinline__ void f8_epi8(const Fp8GemmArgs& p, bool fast, int m, int n, const float (&v)[8]) {
  if (!fast) {
    f8_epi4<EPI, OutT>(p, m, n, f32x4_t{v[0], v[1], v[2], v[3]});
    f8_epi4<EPI, OutT>(p, m, n + 4, f32x4_t{v[4], v[5], v[6], v[7]});
    return;
  }
  auto load = [](const void* base, long i, float (&x)[8]) {
    if constexpr (sizeof(OutT) == 2) {
      const uint4 u = *(const uint4*)((const uint16_t*)base + i);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[2 * k] = __uint_as_float(w[k] << 16);
        x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
      }
    } else {
      const f32x4_t a = *(const f32x4_t*)((const float*)base + i), b = *(const f32x4_t*)((const float*)base + i + 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) { x[k] = a[k]; x[4 + k] = b[k]; }
    }
  };
  auto store = [](void* base, long i, const float (&x)[8]) {
    if constexpr (sizeof(OutT) == 2) {
      uint4 u;
      u.x = f2bf(x[0]) | ((uint32_t)f2bf(x[1]) << 16); u.y = f2bf(x[2]) | ((uint32_t)f2bf(x[3]) << 16);
      u.z = f2bf(x[4]) | ((uint32_t)f2bf(x[5]) << 16); u.w = f2bf(x[6]) | ((uint32_t)f2bf(x[7]) << 16);
      *(uint4*)((uint16_t*)base + i) = u;
    } else {
      *(f32x4_t*)((float*)base + i) = f32x4_t{x[0], x[1], x[2], x[3]};
      *(f32x4_t*)((float*)base + i + 4) = f32x4_t{x[4], x[5], x[6], x[7]};
    }
  };
  const long i = (long)m * p.ldc + n, ia = (long)m * p.ldaux + n;
  float o[8];
  if constexpr (EPI == EPI_STORE) {
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = v[e] * p.alpha;
    if (p.beta != 0.f) {
      float c[8];
      load(p.C, i, c);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] += p.beta * c[e];
    }
  } else if constexpr (EPI == EPI_ACT) {
    if (p.aux_out) store(p.aux_out, ia, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = act_fwd(p.act, v[e]);
  } else {
    float h[8];
    load(p.aux, ia, h);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = v[e] * act_grad(p.act, h[e]);
  }
  store(p.C, i, o);
}

template <int EPI, typename OutT, int FA, int FB>
__global__ __launch_bounds__(512, 2) void fp8_gemm_256(Fp8GemmArgs p) {
  __shared__ __attribute__((aligned(16))) char smem[N8_LDS];
  DLLM_LDS char* lds = (DLLM_LDS char*)smem;
  const int t = threadIdx.x, lane = t & 63;
  const int wid = __builtin_amdgcn_readfirstlane(t >> 6);
  const int tiles_m = (p.M + 255) >> 8, tiles_n = (p.N + 255) >> 8;
  const int bid = xcd_remap(blockIdx.x, gridDim.x);
  const int width = 4 * tiles_n, first = bid / width * 4, gsz = min(tiles_m - first, 4);
  const int m0 = (first + bid % width % gsz) * 256, n0 = (bid % width / gsz) * 256;
  const int left_m = min(p.M - 1 - m0, 255), left_n = min(p.N - 1 - n0, 255);
  uint32_t ao[2][2], bo[2][2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    n8_offsets<true>(p.lda, h, left_m, wid, lane, ao[h]);
    n8_offsets<false>(p.ldb, h, left_n, wid, lane, bo[h]);
  }
  F8Trait<FA, FB, sizeof(OutT) == 4> tr;
  tr.begin(p, m0, n0, wid, lane);
  f32x4_t acc[2][2][4][2];
#pragma unroll
  for (int i = 0; i < 32; ++i) (&acc[0][0][0][0])[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  n8_loop(tr, lds, (const char*)p.A + (long)m0 * p.lda, (const char*)p.B + (long)n0 * p.ldb, tr.step(0), ao, bo, tr.nk2, wid,
          lane, acc);
  const bool fast = left_m == 255 && left_n == 255 && p.ldc % 8 == 0 && (uintptr_t)p.C % 16 == 0 && p.ldaux % 8 == 0 &&
                    (uintptr_t)p.aux % 16 == 0 && (uintptr_t)p.aux_out % 16 == 0;
#pragma unroll
  for (int qm = 0; qm < 2; ++qm)
#pragma unroll
    for (int qn = 0; qn < 2; ++qn)
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = acc[qm][qn][mt][e & 1][e >> 1];
        f8_epi8<EPI, OutT>(p, fast, m0 + n8_row(wid, lane, qm, mt), n0 + n8_col(wid, lane, qn), v);
      }
}

template <int EPI, typename OutT>
static hipError_t launch_fp8(const Fp8GemmArgs& p, int fa, int fb, hipStream_t s) {
  const long tiles = (long)((p.M + 127) / 128) * ((p.N + 127) / 128);
  if (tiles > 0x7fffffffL) return hipErrorInvalidValue;
  const dim3 grid((unsigned)tiles), block(256);
  {
    const long big = (long)((p.M + 255) / 256) * ((p.N + 255) / 256);
    if (p.nk > 0 && p.M >= 4 && p.N >= 2 && big >= 128) {
      const dim3 g2((unsigned)big), b2(512);
      if (fa == F8_E4M3 && fb == F8_E4M3) hipLaunchKernelGGL((fp8_gemm_256<EPI, OutT, F8_E4M3, F8_E4M3>), g2, b2, 0, s, p);
      else if (fa == F8_E4M3) hipLaunchKernelGGL((fp8_gemm_256<EPI, OutT, F8_E4M3, F8_E5M2>), g2, b2, 0, s, p);
      else if (fb == F8_E4M3) hipLaunchKernelGGL((fp8_gemm_256<EPI, OutT, F8_E5M2, F8_E4M3>), g2, b2, 0, s, p);
      else hipLaunchKernelGGL((fp8_gemm_256<EPI, OutT, F8_E5M2, F8_E5M2>), g2, b2, 0, s, p);
      return hipGetLastError();
    }
  }
  if (fa == F8_E4M3 && fb == F8_E4M3) hipLaunchKernelGGL((fp8_gemm_128<EPI, OutT, F8_E4M3, F8_E4M3>), grid, block, 0, s, p);
  else if (fa == F8_E4M3) hipLaunchKernelGGL((fp8_gemm_128<EPI, OutT, F8_E4M3, F8_E5M2>), grid, block, 0, s, p);
  else if (fb == F8_E4M3) hipLaunchKernelGGL((fp8_gemm_128<EPI, OutT, F8_E5M2, F8_E4M3>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((fp8_gemm_128<EPI, OutT, F8_E5M2, F8_E5M2>), grid, block, 0, s, p);
  return hipGetLastError();
}

}  // namespace dllm

using namespace dllm;

extern "C" {

// x [R, C] (DT_BF16 / DT_F32) -> q (x's rows) and / or qt (x^T's rows).  0, a hipError_t, or -1 for a bad argument.
int dllm_fp8_quantize(const void* x, int dtype, long ldx, int R, int C, void* q, long ldq, void* sq, long ldsq, void* qt,
                      long ldqt, void* sqt, long ldsqt, int fmt, int fmt_t, int tile, void* stream) {
  if (R <= 0 || C <= 0 || (q == nullptr && qt == nullptr) || (dtype != DT_BF16 && dtype != DT_F32)) return -1;
  if (fmt < 0 || fmt > 1 || fmt_t < 0 || fmt_t > 1) return -1;
  const long rb = ((long)R + 127) / 128, cb = ((long)C + 127) / 128;
  if (rb * cb > 0x7fffffffL || (x == nullptr)) return -1;
  if (q && (sq == nullptr || ldq < cb * 128 || ldq % 16 || (uintptr_t)q % 16 || ldsq < R)) return -1;
  if (qt && (sqt == nullptr || ldqt < rb * 128 || ldqt % 16 || (uintptr_t)qt % 16 || ldsqt < C)) return -1;
  QuantArgs p{x, ldx, R, C, (uint8_t*)q, ldq, (uint8_t*)sq, ldsq, (uint8_t*)qt, ldqt, (uint8_t*)sqt, ldsqt, fmt, fmt_t, tile};
  const int es = dtype == DT_BF16 ? 2 : 4;
  const bool vec = (uintptr_t)x % 16 == 0 && (ldx * es) % 16 == 0;
  const dim3 grid((unsigned)(rb * cb)), block(256);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == DT_BF16) {
    if (vec) hipLaunchKernelGGL((fp8_quantize_kernel<uint16_t, true>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((fp8_quantize_kernel<uint16_t, false>), grid, block, 0, s, p);
  } else {
    if (vec) hipLaunchKernelGGL((fp8_quantize_kernel<float, true>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((fp8_quantize_kernel<float, false>), grid, block, 0, s, p);
  }
  return (int)hipGetLastError();
}

int dllm_fp8_dequantize(const void* q, long ldq, const void* sq, long ldsq, int fmt, void* out, int dtype, long ldo, int R,
                        int K, void* stream) {
  if (R <= 0 || K <= 0 || fmt < 0 || fmt > 1 || (dtype != DT_BF16 && dtype != DT_F32)) return -1;
  if (ldq % 16 || (uintptr_t)q % 16 || ldq < ((long)K + 127) / 128 * 128 || ldsq < R || ldo < K) return -1;
  const long n = (long)R * ((K + 7) / 8);
  const dim3 grid((unsigned)min((n + 255) / 256, 4096L)), block(256);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == DT_BF16)
    hipLaunchKernelGGL(fp8_dequantize_kernel<uint16_t>, grid, block, 0, s, (const uint8_t*)q, ldq, (const uint8_t*)sq, ldsq,
                       (uint16_t*)out, ldo, (long)R, K, fmt);
  else
    hipLaunchKernelGGL(fp8_dequantize_kernel<float>, grid, block, 0, s, (const uint8_t*)q, ldq, (const uint8_t*)sq, ldsq,
                       (float*)out, ldo, (long)R, K, fmt);
  return (int)hipGetLastError();
}

// C [M, N] (out_dtype) from A [M, 128 nk], B [N, 128 nk].  epi: EPI_STORE / EPI_ACT / EPI_DACT.
int dllm_fp8_gemm(const void* A, long lda, const void* SA, long ldsa, int fa, const void* B, long ldb, const void* SB,
                  long ldsb, int fb, void* C, long ldc, int out_dtype, const void* aux, void* aux_out, long ldaux, int M,
                  int N, int nk, float alpha, float beta, int epi, int act, void* stream) {
  if (M <= 0 || N <= 0 || nk < 0 || nk > (1 << 24) || (out_dtype != DT_BF16 && out_dtype != DT_F32)) return -1;
  if (fa < 0 || fa > 1 || fb < 0 || fb > 1 || ldc < N) return -1;
  if (nk > 0 && ((uintptr_t)A % 16 || (uintptr_t)B % 16 || lda % 16 || ldb % 16 || lda < 128L * nk || ldb < 128L * nk ||
                 ldsa < M || ldsb < N))
    return -1;
  if (epi != EPI_STORE && epi != EPI_ACT && epi != EPI_DACT) return -1;
  if (epi != EPI_STORE && (act < ACT_RELU || act > ACT_GELU)) return -1;
  if (epi == EPI_DACT && aux == nullptr) return -1;
  if ((aux || aux_out) && ldaux < N) return -1;
  Fp8GemmArgs p{(const uint8_t*)A, lda, (const uint8_t*)SA, ldsa, (const uint8_t*)B, ldb, (const uint8_t*)SB, ldsb,
                C, ldc, aux, aux_out, ldaux, M, N, nk, alpha, beta, act};
  hipStream_t s = (hipStream_t)stream;
  const bool bf = out_dtype == DT_BF16;
  switch (epi) {
    case EPI_STORE: return (int)(bf ? launch_fp8<EPI_STORE, uint16_t>(p, fa, fb, s) : launch_fp8<EPI_STORE, float>(p, fa, fb, s));
    case EPI_ACT: return (int)(bf ? launch_fp8<EPI_ACT, uint16_t>(p, fa, fb, s) : launch_fp8<EPI_ACT, float>(p, fa, fb, s));
    default: return (int)(bf ? launch_fp8<EPI_DACT, uint16_t>(p, fa, fb, s) : launch_fp8<EPI_DACT, float>(p, fa, fb, s));
  }
}

}  // extern "C"
