// Block-scaled 8-bit quantiser, read-back and matrix product (fp8.h has the format).
#include <type_traits>

#include "fp8.h"
#include "nt8.h"

namespace dllm {

typedef __attribute__((ext_vector_type(8))) int i32x8_t;
typedef __attribute__((ext_vector_type(2))) float f32x2_t;

// 16-byte accesses at any element's address: the hardware takes them unaligned, so odd row lengths need no other path
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// ----------------------------------------------------------------------------------------------
// quantiser: one block of 256 threads per 128x128 tile of x, one read of x for both orientations
//
// Thread (g, j) = (t / 16, t % 16) holds rows 8g .. 8g+7 and columns 8j .. 8j+7 of the tile in registers.  A row's 128
// columns sit in 16 neighbouring lanes (row scales: 4 rotations within them), a column's 128 rows in 16 values of g (column
// scales: two lane exchanges that leave each of the wave's four g with two of the eight columns, then LDS over the four
// waves).  x^T leaves through LDS so that its rows are written in whole 128-B lines; its rows there are 33 words apart, which
// spreads both the writes and the reads over all banks.  Bound by HBM on large tensors: 8192 x 4096 bf16, both orientations,
// 28.6 us (4.7 TB/s; 42.8 with a row's load waited for before the next, exchanges through LDS and rows 36 words apart); a
// tile takes about 5 us, which bounds small ones.
// ----------------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<uint16_t>(uint16_t v) { return bf2f(v); }
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }

// magnitude bits of v (in the order of magnitudes, then inf, then NaN), and the same with 0 for inf / NaN: a block's scale
// comes from its finite elements.  Integers: a float maximum gives way to a signalling NaN
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = abs_bits(v);
  return b < 0x7f800000u ? b : 0u;
}

// max over the 16 lanes of a row, in all of them
__device__ __forceinline__ uint32_t max_row16(uint32_t m) {
  auto ror = [](uint32_t x, auto n) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + n.value, 0xf, 0xf, false); };
  m = max(m, ror(m, std::integral_constant<int, 8>{}));
  m = max(m, ror(m, std::integral_constant<int, 4>{}));
  m = max(m, ror(m, std::integral_constant<int, 2>{}));
  return max(m, ror(m, std::integral_constant<int, 1>{}));
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

typedef uint64_t u64_any __attribute__((aligned(1)));
// n <= 8 scale bytes (byte i of w) to p
__device__ __forceinline__ void put_scales(uint8_t* p, uint64_t w, int n) {
  if (n >= 8) {
    *(u64_any*)p = w;
  } else {
    for (int i = 0; i < n; ++i) p[i] = (uint8_t)(w >> (8 * i));
  }
}

template <typename T>
__global__ __launch_bounds__(256) void fp8_quantize_kernel(QuantArgs p) {
  constexpr int QT_LD = 33;         // words
  __shared__ uint32_t tbuf[128 * QT_LD];
  __shared__ __attribute__((aligned(16))) uint32_t cmax[4][128];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int g = t >> 4, j = t & 15;
  const int tiles_c = (p.C + 127) >> 7;
  const int tr = blockIdx.x / tiles_c, tc = blockIdx.x - tr * tiles_c;
  const long r0 = (long)tr * 128, c0 = (long)tc * 128;
  const T* x = (const T*)p.x + r0 * p.ldx + c0;
  const int nr = (int)min((long)128, p.R - r0), nc = (int)min((long)128, p.C - c0);

  float v[8][8];
  auto unpack = [&](int i, const u32x4_any& w) {     // 8 bf16
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[i][2 * k] = __uint_as_float(w[k] << 16);
      v[i][2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
    }
  };
  // all loads are on their way before the first is used; behind the last row or column the last one is loaded again
  if (32 * wave >= nr) {
#pragma unroll
    for (int i = 0; i < 64; ++i) (&v[0][0])[i] = 0.f;
  } else if (nc % 8 == 0) {
    const int c = min(8 * j, nc - 8);
    if constexpr (sizeof(T) == 2) {
      u32x4_any u[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] = *(const u32x4_any*)(x + (long)min(8 * g + i, nr - 1) * p.ldx + c);
#pragma unroll
      for (int i = 0; i < 8; ++i) unpack(i, u[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const f32x4_any* s = (const f32x4_any*)(x + (long)min(8 * g + i, nr - 1) * p.ldx + c);
        const f32x4_t a = s[0], b = s[1];
#pragma unroll
        for (int k = 0; k < 4; ++k) { v[i][k] = a[k]; v[i][4 + k] = b[k]; }
      }
    }
    if (nr < 128 || nc < 128) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) v[i][k] = 8 * g + i < nr && 8 * j < nc ? v[i][k] : 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const T* s = x + (long)min(8 * g + i, nr - 1) * p.ldx;
#pragma unroll
      for (int k = 0; k < 8; ++k) v[i][k] = to_f32<T>(s[min(8 * j + k, nc - 1)]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) v[i][k] = 8 * g + i < nr && 8 * j + k < nc ? v[i][k] : 0.f;
  }

  // maxima of the thread's rows and columns; where there is an inf or NaN among them, again over the finite elements
  uint32_t rowmax[8], colmax[8], all = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) rowmax[i] = colmax[i] = 0;
#pragma unroll
  for (int i = 0; i < 8; i += 2)
#pragma unroll
    for (int k = 0; k < 8; k += 2) {     // 2 x 2 at a time: four magnitudes are alive, not 64
      const uint32_t m00 = abs_bits(v[i][k]), m01 = abs_bits(v[i][k + 1]), m10 = abs_bits(v[i + 1][k]), m11 = abs_bits(v[i + 1][k + 1]);
      rowmax[i] = max(max(rowmax[i], m00), m01);
      rowmax[i + 1] = max(max(rowmax[i + 1], m10), m11);
      colmax[k] = max(max(colmax[k], m00), m10);
      colmax[k + 1] = max(max(colmax[k + 1], m01), m11);
    }
#pragma unroll
  for (int i = 0; i < 8; ++i) all = max(all, rowmax[i]);
  if (all >= 0x7f800000u) {
    all = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      rowmax[i] = colmax[i] = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        asm("" : "+v"(v[i][k]));           // (not the magnitudes from above, kept for here)
        rowmax[i] = max(rowmax[i], finite_bits(v[i][k]));
      }
      all = max(all, rowmax[i]);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
#pragma unroll
      for (int i = 0; i < 8; ++i) colmax[k] = max(colmax[k], finite_bits(v[i][k]));
    }
  }
  if (p.tile) {
    all = max_row16(all);
    all = max(all, (uint32_t)__shfl_xor((int)all, 16));
    all = max(all, (uint32_t)__shfl_xor((int)all, 32));
    if (lane == 0) cmax[0][wave] = all;
    __syncthreads();
    all = max(max(cmax[0][0], cmax[0][1]), max(cmax[0][2], cmax[0][3]));
    __syncthreads();
  }

  using E4 = std::integral_constant<int, F8_E4M3>;
  using E5 = std::integral_constant<int, F8_E5M2>;
  if (p.q != nullptr) {
    auto rows = [&](auto fmt) {
      uint64_t bytes = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t b = e8m0_of_amax(p.tile ? all : max_row16(rowmax[i]), fmt.value);
        const float s = e8m0_inv(b);
        bytes |= (uint64_t)b << (8 * i);
        const int r = 8 * g + i;
        uint2 o;
        o.x = pack4<fmt.value>(v[i][0] * s, v[i][1] * s, v[i][2] * s, v[i][3] * s);
        o.y = pack4<fmt.value>(v[i][4] * s, v[i][5] * s, v[i][6] * s, v[i][7] * s);
        if (r < nr) *(uint2*)(p.q + (r0 + r) * p.ldq + c0 + 8 * j) = o;
      }
      if (j == 0) put_scales(p.sq + (long)tc * p.ldsq + r0 + 8 * g, bytes, nr - 8 * g);
    };
    if (p.fmt == F8_E4M3) rows(E4{});
    else rows(E5{});
  }

  if (p.qt != nullptr) {
    if (!p.tile) {
      // over the wave's four g: each exchange keeps half of the columns, lane row g % 4 = 2 a + b ends with 4 a + 2 b and the
      // one after it
      typedef __attribute__((ext_vector_type(2))) uint32_t u32x2_t;
      uint32_t h[4], q[2];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const u32x2_t w = __builtin_amdgcn_permlane32_swap(colmax[k], colmax[4 + k], false, false);
        h[k] = max(w[0], w[1]);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const u32x2_t w = __builtin_amdgcn_permlane16_swap(h[k], h[2 + k], false, false);
        q[k] = max(w[0], w[1]);
      }
      *(uint2*)&cmax[wave][8 * j + 4 * (lane >> 5) + 2 * (lane >> 4 & 1)] = uint2{q[0], q[1]};
      __syncthreads();
    }
    auto columns = [&](auto fmt) {
      uint64_t bytes = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int c = 8 * j + k;
        const uint32_t b = e8m0_of_amax(p.tile ? all : max(max(cmax[0][c], cmax[1][c]), max(cmax[2][c], cmax[3][c])), fmt.value);
        const float s = e8m0_inv(b);
        bytes |= (uint64_t)b << (8 * k);
        uint32_t* o = tbuf + c * QT_LD + 2 * g;
        o[0] = pack4<fmt.value>(v[0][k] * s, v[1][k] * s, v[2][k] * s, v[3][k] * s);
        o[1] = pack4<fmt.value>(v[4][k] * s, v[5][k] * s, v[6][k] * s, v[7][k] * s);
      }
      if (g == 0) put_scales(p.sqt + (long)tr * p.ldsqt + c0 + 8 * j, bytes, nc - 8 * j);
    };
    if (p.fmt_t == F8_E4M3) columns(E4{});
    else columns(E5{});
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = 32 * i + (t >> 3), o = t & 7;
      const uint32_t* w = tbuf + c * QT_LD + 4 * o;
      if (c < nc) *(uint4*)(p.qt + (c0 + c) * p.ldqt + r0 + 16 * o) = uint4{w[0], w[1], w[2], w[3]};
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
    if (c + 8 <= K) {
      if constexpr (sizeof(T) == 2) {
        u32x4_any u;
        u.x = f2bf(v[0]) | ((uint32_t)f2bf(v[1]) << 16); u.y = f2bf(v[2]) | ((uint32_t)f2bf(v[3]) << 16);
        u.z = f2bf(v[4]) | ((uint32_t)f2bf(v[5]) << 16); u.w = f2bf(v[6]) | ((uint32_t)f2bf(v[7]) << 16);
        *(u32x4_any*)o = u;
      } else {
        *(f32x4_any*)o = f32x4_any{v[0], v[1], v[2], v[3]};
        *(f32x4_any*)(o + 4) = f32x4_any{v[4], v[5], v[6], v[7]};
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
// product C = alpha A B^T + beta C (and the activation epilogues), any M, N
//
// Both operands are K-contiguous; a K step of 128 is one 128-byte line per row.  A lane's 32 bytes of a fragment are 16-byte
// chunks g and 4 + g (g = lane / 16) of its row, in A and B alike: a permutation of k inside the block, which neither the
// sum nor the block's one scale sees.  The operands are swapped in the matrix instruction (B first), so a lane ends with
// consecutive columns of a row of C.  Three kernels: 256x256 tiles (8-phase loop), 128x128 and 64x64 tiles (one wave per
// quarter), and few rows or columns (operands straight to registers, K over the waves); fp8_plan picks.
// ----------------------------------------------------------------------------------------------
// The 8-bit matrix instruction adds the products of 8 neighbouring k with 13 bits below the largest of them (measured: a
// product under 2^-13 of its neighbour is lost whole, the sums of 8 then add up in fp32): about 4e-5 of the result, a
// hundredth of bf16's half step 2^-8 but hundreds of fp32's.  So a bf16 result is computed on it, and an fp32 result on
// the bf16 instruction, which keeps fp32 sums (5e-7 at K = 8192): codes times their scale are bf16 numbers, exactly
// (8 exponent bits; only values under 2^-126 may round), so the operands convert in registers on their way from LDS.
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
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

template <typename OutT> __device__ __forceinline__ float ld_out(const void* p, long i) {
  if constexpr (sizeof(OutT) == 2) return bf2f(((const uint16_t*)p)[i]);
  else return ((const float*)p)[i];
}
template <typename OutT> __device__ __forceinline__ void st_out(void* p, long i, float v) {
  if constexpr (sizeof(OutT) == 2) ((uint16_t*)p)[i] = f2bf(v);
  else ((float*)p)[i] = v;
}

// epilogue of element (m, n)
template <int EPI, typename OutT>
__device__ __forceinline__ void f8_epi1(const Fp8GemmArgs& p, int m, int n, float o) {
  const long i = (long)m * p.ldc + n, ia = (long)m * p.ldaux + n;
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

// ----------------------------------------------------------------------------------------------
// 256x256 tiles on the 8-phase loop (nt8.h), one matrix instruction per 16x16 fragment pair and K step.
//
// Scales: a lane's four A rows of a half are consecutive rows of C (nt8.h), so one 32-bit word of the K step's scale row
// holds them, and 16 bits its two B rows; the matrix instruction picks the byte (op_sel), so scaling costs two 4-byte and
// two 2-byte loads per K step and nothing else.  An odd number of K steps runs one more, the last step again, without effect: a
// bf16 result takes it with scale bytes 0 on both sides, 2^-254 of products whose infinities stay infinities, which leaves
// every sum as it is (jumping over its matrix instructions costs that kernel 270 bytes of spills); an fp32 result jumps over
// them, as codes times 2^-127 would be rounded to zero in bf16, and infinity times zero is NaN.
//
// 8192 x 16384 x 4096 bf16: 445 us (2470 TF; 2898 in a library product without scales): matrix units busy 62 % of the cycles, at a
// clock that power holds at 1.9 of 2.4 GHz, and at the tile boundary every block stores at once.  The activation epilogues
// add the second 268 MB and the function: relu 495, with aux_out 526, dact 559; gelu 591, 601, 643.  4096 x 16384 x 8192 fp32 with
// beta: 914 us (1200 TF; 1464 in a library bf16 product): matrix units busy half of the cycles at 2.2 GHz, the conversions
// issue between their instructions.  No LDS conflicts in either.
// ----------------------------------------------------------------------------------------------
typedef uint32_t u32_any __attribute__((aligned(1)));
typedef uint16_t u16_any __attribute__((aligned(1)));

// EXACT: fp32 sums -- codes times scale as bf16 on the bf16 instruction (see codes8), converted in the shadow of the
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
    if constexpr (ODD && EXACT) {
      if (keep == 0) return;
    }
    if constexpr (QM == 0 && QN == 0) {   // the step's first phase
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        wa[ODD][h] = (int)((uint32_t)wa[ODD][h] >> (sh >> (8 * h) & 31));
        wb[ODD][h] = (int)((uint32_t)wb[ODD][h] >> (sh >> (16 + 8 * h) & 31));
        if constexpr (ODD && !EXACT) { wa[ODD][h] &= keep; wb[ODD][h] &= keep; }
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

// 8 columns n .. n + 7 of row m; `inside`: the whole tile is inside C
template <int EPI, typename OutT>
__device__ __forceinline__ void f8_epi8(const Fp8GemmArgs& p, bool inside, int m, int n, const float (&v)[8]) {
  if (!inside) {
    if (m >= p.M) return;
    if (n + 8 > p.N) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (n + e < p.N) f8_epi1<EPI, OutT>(p, m, n + e, v[e]);
      return;
    }
  }
  auto load = [](const void* base, long i, float (&x)[8]) {
    if constexpr (sizeof(OutT) == 2) {
      const u32x4_any w = *(const u32x4_any*)((const uint16_t*)base + i);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[2 * k] = __uint_as_float(w[k] << 16);
        x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
      }
    } else {
      const f32x4_any a = *(const f32x4_any*)((const float*)base + i), b = *(const f32x4_any*)((const float*)base + i + 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) { x[k] = a[k]; x[4 + k] = b[k]; }
    }
  };
  auto store = [](void* base, long i, const float (&x)[8]) {
    if constexpr (sizeof(OutT) == 2) {
      u32x4_any u;
      u.x = f2bf(x[0]) | ((uint32_t)f2bf(x[1]) << 16); u.y = f2bf(x[2]) | ((uint32_t)f2bf(x[3]) << 16);
      u.z = f2bf(x[4]) | ((uint32_t)f2bf(x[5]) << 16); u.w = f2bf(x[6]) | ((uint32_t)f2bf(x[7]) << 16);
      *(u32x4_any*)((uint16_t*)base + i) = u;
    } else {
      *(f32x4_any*)((float*)base + i) = f32x4_any{x[0], x[1], x[2], x[3]};
      *(f32x4_any*)((float*)base + i + 4) = f32x4_any{x[4], x[5], x[6], x[7]};
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
  const bool inside = left_m == 255 && left_n == 255;
#pragma unroll
  for (int qm = 0; qm < 2; ++qm)
#pragma unroll
    for (int qn = 0; qn < 2; ++qn)
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = acc[qm][qn][mt][e & 1][e >> 1];
        f8_epi8<EPI, OutT>(p, inside, m0 + n8_row(wid, lane, qm, mt), n0 + n8_col(wid, lane, qn), v);
      }
}

// ----------------------------------------------------------------------------------------------
// 128x128 (F = 4) and 64x64 (F = 2) tiles: four waves, each 16F x 16F, a ring of 4 K steps of LDS
//
// For grids that 256x256 tiles leave part-empty.  A wave reads the next step's fragments while it computes the current
// step's; one barrier per step.  F = 4 is bound by LDS (64 KiB read and 32 KiB written per step, 768 of its about 830
// cycles), F = 2 by the latency of few steps.  Rows are permuted in LDS (slot 16 f + i holds row F i + f of the wave's
// piece): a lane's F rows are consecutive and one word holds their scales.  ksplit > 1: slice blockIdx.y of the K steps,
// fp32 partial sums to ws (fp8_join adds them).
// ----------------------------------------------------------------------------------------------
template <int EPI, typename OutT, int FA, int FB, int F>
__device__ __forceinline__ void fp8_w4_body(const Fp8GemmArgs& p, DLLM_LDS char* lds) {
  constexpr int TS = 32 * F, OPB = TS * 128, STAGE = 2 * OPB, STAGES = 4;
  constexpr bool EXACT = sizeof(OutT) == 4;
  const int t = threadIdx.x, lane = t & 63;
  const int wid = __builtin_amdgcn_readfirstlane(t >> 6);
  const int i15 = lane & 15, g = lane >> 4, wr = wid >> 1, wc = wid & 1;
  const int tiles_m = (p.M + TS - 1) / TS, tiles_n = (p.N + TS - 1) / TS;
  const int bid = xcd_remap(blockIdx.x, gridDim.x);
  const int width = 4 * tiles_n, first = bid / width * 4, gsz = min(tiles_m - first, 4);
  const int m0 = (first + bid % width % gsz) * TS, n0 = (bid % width / gsz) * TS;
  const int k0 = (int)((long)p.nk * blockIdx.y / p.ksplit), nk = (int)((long)p.nk * (blockIdx.y + 1) / p.ksplit) - k0;

  uint32_t ao[F], bo[F];
#pragma unroll
  for (int i = 0; i < F; ++i) {
    const int s = 8 * (wid + 4 * i) + (lane >> 3);
    const int w = s / (16 * F), in = s - w * 16 * F;
    const int row = w * 16 * F + F * (in & 15) + (in >> 4), c = (lane & 7) ^ ((s >> 1) & 7);
    ao[i] = (uint32_t)((long)min(row, p.M - 1 - m0) * p.lda + c * 16);
    bo[i] = (uint32_t)((long)min(row, p.N - 1 - n0) * p.ldb + c * 16);
  }
  const char* A = (const char*)p.A + (long)m0 * p.lda + (long)k0 * 128;
  const char* B = (const char*)p.B + (long)n0 * p.ldb + (long)k0 * 128;
  auto fetch = [&](int i, int kt, int slot) {       // piece i of the step (0 .. 2F - 1: A's, then B's); past the end: the last
    const long ko = (long)min(kt, nk - 1) * 128;
    DLLM_LDS char* d = lds + slot * STAGE;
    if (i < F) n8_dma(A + ko, ao[i], d + (wid + 4 * i) * 1024);
    else n8_dma(B + ko, bo[i - F], d + OPB + (wid + 4 * (i - F)) * 1024);
  };
  // scales: the lane's F rows of A and of B; a word that would pass the end of its row starts earlier and is shifted
  const int ra = m0 + wr * 16 * F + F * i15, rb = n0 + wc * 16 * F + F * i15;
  const int oa = max(0, min(ra, p.M - F)), ob = max(0, min(rb, p.N - F));
  const int sha = min(8 * (ra - oa), 8 * F - 8), shb = min(8 * (rb - ob), 8 * F - 8);
  auto scales = [&](const uint8_t* s, long ld, int kt, int off) {
    const uint8_t* q = s + (long)(k0 + min(kt, nk - 1)) * ld + off;
    if constexpr (F == 4) return (uint32_t)*(const u32_any*)q;
    else return (uint32_t)*(const u16_any*)q;
  };
  const uint32_t lb = (uint32_t)(uintptr_t)lds;
  const int sw = (i15 >> 1) & 7;
  const uint32_t la[2] = {lb + (wr * 16 * F + i15) * 128 + ((g ^ sw) << 4), lb + (wr * 16 * F + i15) * 128 + (((4 + g) ^ sw) << 4)};
  const uint32_t lbb[2] = {lb + OPB + (wc * 16 * F + i15) * 128 + ((g ^ sw) << 4),
                           lb + OPB + (wc * 16 * F + i15) * 128 + (((4 + g) ^ sw) << 4)};
  N8Frag xa[2][F], xb[2][F];
  uint32_t wa[2], wb[2];
  f32x4_t acc[F][F];
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int k = 0; k < F; ++k) acc[i][k] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  auto read = [&](auto par, auto j, uint32_t off) {   // read j of a step's 4F
    constexpr int f = j.value >> 1, h = j.value & 1;
    if constexpr (f < F) n8_read<f * 2048>(h ? xa[par.value][f].hi : xa[par.value][f].lo, la[h] + off);
    else n8_read<(f - F) * 2048>(h ? xb[par.value][f - F].hi : xb[par.value][f - F].lo, lbb[h] + off);
  };
  auto upto = [](auto n, auto f) {
    [&]<int... J>(std::integer_sequence<int, J...>) { (f(std::integral_constant<int, J>{}), ...); }(std::make_integer_sequence<int, decltype(n)::value>{});
  };
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using NR = std::integral_constant<int, 4 * F>;
  using NQ = std::integral_constant<int, F * F>;
  if (nk > 0) {
    wa[0] = scales(p.SA, p.ldsa, 0, oa);
    wb[0] = scales(p.SB, p.ldsb, 0, ob);
#pragma unroll
    for (int s = 0; s < STAGES; ++s)
#pragma unroll
      for (int i = 0; i < 2 * F; ++i) fetch(i, s, s);
    if constexpr (F == 4) asm volatile("s_waitcnt vmcnt(24)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(12)" ::: "memory");
    N8_BARRIER();
    upto(NR{}, [&](auto j) { read(I0{}, j, 0u); });
    N8_LDS_WAIT();
    int slot = 0;
    // step kt: its fragments are in registers and its LDS slot is free; read step kt + 1, fetch step kt + 4
    auto one = [&](auto par, auto other, int kt) {
      if constexpr (F == 4) asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
      N8_BARRIER();
      const int fs = slot;
      slot = slot + 1 == STAGES ? 0 : slot + 1;
      const uint32_t off = (uint32_t)(slot * STAGE);
      wa[other.value] = scales(p.SA, p.ldsa, kt + 1, oa);
      wb[other.value] = scales(p.SB, p.ldsb, kt + 1, ob);
      upto(NR{}, [&](auto j) { read(other, j, off); });
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 2 * F; ++i) fetch(i, kt + STAGES, fs);
      __builtin_amdgcn_sched_barrier(0);
      const uint32_t a = wa[par.value] >> sha, b = wb[par.value] >> shb;
      if constexpr (!EXACT) {
        upto(NQ{}, [&](auto q) {
          constexpr int i = q.value / F, k = q.value % F;
          const N8Frag &fa = xa[par.value][i], &fb = xb[par.value][k];
          const i32x8_t x = __builtin_shufflevector(fa.lo, fa.hi, 0, 1, 2, 3, 4, 5, 6, 7);
          const i32x8_t y = __builtin_shufflevector(fb.lo, fb.hi, 0, 1, 2, 3, 4, 5, 6, 7);
          acc[i][k] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(y, x, acc[i][k], FB, FA, k, (int)b, i, (int)a);
        });
      } else {
        auto scale = [](uint32_t w, int i) { return __uint_as_float((w >> (8 * i) & 255u) << 23); };
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          auto pick = [&](const N8Frag& f, int k) { return s < 2 ? f.lo[2 * (s & 1) + k] : f.hi[2 * (s & 1) + k]; };
          bf16x8_t y[F];
#pragma unroll
          for (int k = 0; k < F; ++k) y[k] = codes8<FB>(pick(xb[par.value][k], 0), pick(xb[par.value][k], 1), scale(b, k));
#pragma unroll
          for (int i = 0; i < F; ++i) {
            const bf16x8_t x = codes8<FA>(pick(xa[par.value][i], 0), pick(xa[par.value][i], 1), scale(a, i));
#pragma unroll
            for (int k = 0; k < F; ++k) acc[i][k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(y[k], x, acc[i][k], 0, 0, 0);
          }
        }
      }
      N8_LDS_WAIT();
    };
    for (int kt = 0; kt < nk; kt += 2) {
      one(I0{}, I1{}, kt);
      if (kt + 1 < nk) one(I1{}, I0{}, kt + 1);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }

  // lane: rows mb .. mb + F - 1, columns nb .. nb + 4F - 1 (column F r + k of them: acc[.][k][r])
  const int mb = m0 + wr * 16 * F + F * i15, nb = n0 + wc * 16 * F + 4 * F * g;
  const bool inside = n0 + TS <= p.N && m0 + TS <= p.M;
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int c8 = 0; c8 < F / 2; ++c8) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = acc[i][(8 * c8 + e) % F][(8 * c8 + e) / F];
      if (p.ksplit > 1) {
        const int m = mb + i, n = nb + 8 * c8;
        if (m < p.M) {
          float* o = p.ws + (long)blockIdx.y * p.M * p.N + (long)m * p.N + n;
          if (n + 8 <= p.N) {
            *(f32x4_any*)o = f32x4_any{v[0], v[1], v[2], v[3]};
            *(f32x4_any*)(o + 4) = f32x4_any{v[4], v[5], v[6], v[7]};
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (n + e < p.N) o[e] = v[e];
          }
        }
      } else {
        f8_epi8<EPI, OutT>(p, inside, mb + i, nb + 8 * c8, v);
      }
    }
}

constexpr int fp8_w4_lds(int f) { return 4 * 2 * 32 * f * 128; }
extern __shared__ __attribute__((aligned(16))) char fp8_dyn_lds[];
// Dynamic LDS (128 KiB, one block per CU) and a bound of two blocks: the compiler then stays within 256 registers.  Left with
// 512 it keeps the accumulators in the accumulation file and copies each one around its matrix instruction.
template <int EPI, typename OutT, int FA, int FB>
__global__ __launch_bounds__(256, 2) void fp8_gemm_128(Fp8GemmArgs p) {
  fp8_w4_body<EPI, OutT, FA, FB, 4>(p, (DLLM_LDS char*)fp8_dyn_lds);
}
template <int EPI, typename OutT, int FA, int FB>
__global__ __launch_bounds__(256, 2) void fp8_gemm_64(Fp8GemmArgs p) {
  __shared__ __attribute__((aligned(16))) char smem[fp8_w4_lds(2)];
  fp8_w4_body<EPI, OutT, FA, FB, 2>(p, (DLLM_LDS char*)smem);
}

// the K slices' sums, in the order of K, and the epilogue; a thread per element
template <int EPI, typename OutT>
__global__ __launch_bounds__(256) void fp8_join(Fp8GemmArgs p) {
  const long n = (long)p.M * p.N;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    float s = p.ws[i];
    for (int k = 1; k < p.ksplit; ++k) s += p.ws[(long)k * n + i];
    f8_epi1<EPI, OutT>(p, (int)(i / p.N), (int)(i % p.N), s);
  }
}

// ----------------------------------------------------------------------------------------------
// few rows of A (SWAP: of B), at most 16 MT: 16 rows of the other operand per block, the K steps dealt to its 8 waves
//
// Fragments go from memory to registers (a step's line of a row is read by the 4 lanes of its row), the waves' sums are
// added in LDS in the order of the waves.  At one row bound by reading the long operand (16384 x 4096 in 14.7 us, 4.6 TB/s);
// with more rows by reading the short operand again for every 16 rows of the long one, from L2: 16 rows 19.8 us, 64 rows 46.
// 64x64 tiles read it once per 64 (19.0 us), so fp8_plan takes them there; on a small long operand they leave CUs empty
// (1024 x 1024, 64 rows: 5.4 us here, 6.3 there).  A long operand of few rows has too few blocks: one row by 4096 x 16384 takes
// 19.1 us (256 blocks, 16 steps a wave), by 4096 x 4096 6.2 (floors 13.2 and 3.3).
// ----------------------------------------------------------------------------------------------
template <int EPI, typename OutT, int FA, int FB, int MT, bool SWAP>
__global__ __launch_bounds__(512) void fp8_gemm_rows(Fp8GemmArgs p) {
  __shared__ f32x4_t part[8][MT][64];
  constexpr bool EXACT = sizeof(OutT) == 4;
  constexpr int FS = SWAP ? FB : FA, FL = SWAP ? FA : FB;        // formats of the short and the long operand
  const int t = threadIdx.x, lane = t & 63, i15 = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const uint8_t *L = SWAP ? p.A : p.B, *SL = SWAP ? p.SA : p.SB, *S = SWAP ? p.B : p.A, *SS = SWAP ? p.SB : p.SA;
  const long ldl = SWAP ? p.lda : p.ldb, ldsl = SWAP ? p.ldsa : p.ldsb, lds = SWAP ? p.ldb : p.lda, ldss = SWAP ? p.ldsb : p.ldsa;
  const int nl = SWAP ? p.M : p.N, ns = SWAP ? p.N : p.M;
  const int l0 = blockIdx.x * 16, rl = min(l0 + i15, nl - 1);
  const uint8_t* lp = L + (long)rl * ldl + g * 16;
  int rs[MT];
  const uint8_t* sp[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    rs[i] = min(16 * i + i15, ns - 1);
    sp[i] = S + (long)rs[i] * lds + g * 16;
  }
  f32x4_t acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  auto load = [](const uint8_t* q) {
    const n8_i32x4 lo = *(const n8_i32x4*)q, hi = *(const n8_i32x4*)(q + 64);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  // the loads of D steps are on their way together: one step at a time waits for memory at each (32 rows by 4096 x 4096:
  // 10.5 us, now 8.7)
  constexpr int D = MT == 4 ? 2 : 4;
  for (int kt = w; kt < p.nk; kt += 8 * D) {
    i32x8_t fl[D], fs[D][MT];
    int sl[D], ss[D][MT];
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (kt + 8 * d >= p.nk) break;
      const int k = kt + 8 * d;
      fl[d] = load(lp + (long)k * 128);
      sl[d] = SL[(long)k * ldsl + rl];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        fs[d][i] = load(sp[i] + (long)k * 128);
        ss[d][i] = SS[(long)k * ldss + rs[i]];
      }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d = 0; d < D; ++d) {   // uses that stay here: the compiler moves loads down to their first use
      asm volatile("" : "+v"(fl[d]), "+v"(sl[d]));
#pragma unroll
      for (int i = 0; i < MT; ++i) asm volatile("" : "+v"(fs[d][i]), "+v"(ss[d][i]));
    }
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (kt + 8 * d >= p.nk) break;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        if constexpr (!EXACT) {
          acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fl[d], fs[d][i], acc[i], FL, FS, 0, sl[d], 0, ss[d][i]);
        } else {
          const float a = __uint_as_float((uint32_t)ss[d][i] << 23), b = __uint_as_float((uint32_t)sl[d] << 23);
#pragma unroll
          for (int s = 0; s < 4; ++s)
            acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes8<FL>(fl[d][2 * s], fl[d][2 * s + 1], b),
                                                             codes8<FS>(fs[d][i][2 * s], fs[d][i][2 * s + 1], a), acc[i], 0, 0, 0);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) part[w][i][lane] = acc[i];
  __syncthreads();
  if (w < MT) {
    f32x4_t v = part[0][w][lane];
#pragma unroll
    for (int k = 1; k < 8; ++k) v += part[k][w][lane];
    const int s = 16 * w + i15, l = l0 + 4 * g;               // lane: rows l .. l + 3 of the long operand, row s of the short
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int m = SWAP ? l + r : s, n = SWAP ? s : l + r;
      if (m < p.M && n < p.N) f8_epi1<EPI, OutT>(p, m, n, v[r]);
    }
  }
}

// ----------------------------------------------------------------------------------------------
// choice and launch
// ----------------------------------------------------------------------------------------------
template <int EPI, typename OutT, int FA, int FB>
static hipError_t launch_fp8_f(Fp8GemmArgs p, hipStream_t s) {
  const int few = min(p.M, p.N);
  if (p.tile == 0) {
    const bool swap = p.N < p.M;
    const dim3 grid((unsigned)((max(p.M, p.N) + 15) / 16)), block(512);
    auto go = [&](auto mt, auto sw) {
      hipLaunchKernelGGL((fp8_gemm_rows<EPI, OutT, FA, FB, decltype(mt)::value, decltype(sw)::value>), grid, block, 0, s, p);
    };
    using T = std::true_type;
    using N = std::false_type;
    auto by = [&](auto sw) {
      if (few <= 16) go(std::integral_constant<int, 1>{}, sw);
      else if (few <= 32) go(std::integral_constant<int, 2>{}, sw);
      else go(std::integral_constant<int, 4>{}, sw);
    };
    if (swap) by(T{});
    else by(N{});
    return hipGetLastError();
  }
  const int ts = p.tile;
  const long tiles = (long)((p.M + ts - 1) / ts) * ((p.N + ts - 1) / ts);
  if (tiles > 0x7fffffffL) return hipErrorInvalidValue;
  if (ts == 256) hipLaunchKernelGGL((fp8_gemm_256<EPI, OutT, FA, FB>), dim3((unsigned)tiles), dim3(512), 0, s, p);
  else if (ts == 128) {
    const hipError_t e = lds_opt_in((const void*)fp8_gemm_128<EPI, OutT, FA, FB>, fp8_w4_lds(4));
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((fp8_gemm_128<EPI, OutT, FA, FB>), dim3((unsigned)tiles, p.ksplit), dim3(256), fp8_w4_lds(4), s, p);
  }
  else hipLaunchKernelGGL((fp8_gemm_64<EPI, OutT, FA, FB>), dim3((unsigned)tiles, p.ksplit), dim3(256), 0, s, p);
  if (p.ksplit > 1) {
    const long n = (long)p.M * p.N;
    hipLaunchKernelGGL((fp8_join<EPI, OutT>), dim3((unsigned)min((n + 255) / 256, 2048L)), dim3(256), 0, s, p);
  }
  return hipGetLastError();
}

template <int EPI, typename OutT>
static hipError_t launch_fp8(const Fp8GemmArgs& p, int fa, int fb, hipStream_t s) {
  if (fa == F8_E4M3) return fb == F8_E4M3 ? launch_fp8_f<EPI, OutT, F8_E4M3, F8_E4M3>(p, s) : launch_fp8_f<EPI, OutT, F8_E4M3, F8_E5M2>(p, s);
  return fb == F8_E4M3 ? launch_fp8_f<EPI, OutT, F8_E5M2, F8_E4M3>(p, s) : launch_fp8_f<EPI, OutT, F8_E5M2, F8_E5M2>(p, s);
}

constexpr int FP8_FEW = 64;   // rows (or columns) that fp8_gemm_rows takes, at most
// its blocks of 512 threads count 16 long rows each, and a launch counts its threads in 32 bits
constexpr int FP8_LONG = (1 << 27) - 16;
// bytes from row to row that the tiles' fetches take: the buffer form reaches 2^31 bytes from a tile's first row
constexpr long FP8_PITCH = (0x7fffffffL - 4096) / 256;

// Tile (0: fp8_gemm_rows) and number of K slices: the least time for whole rounds of CUs, in microseconds measured on full
// rounds: a K step of 128 on one CU (bf16 results / fp32 results), a round's beginning and end, and the slices' partial sums
// at 1.5 TB/s.  Every choice was measured at six weights (1024 x 1024 to 16384 x 4096, both directions), nine numbers of rows (1 to
// 256) and both result types: the one it makes is the fastest or within 12 % of it in 104 of 108 cases, else 17 to 37 % off
// (at worst 2048 x 8192, 256 rows, bf16: 24.7 us, four slices of 64 tiles 18.0).
static void fp8_plan(int M, int N, int nk, bool exact, int& tile, int& ksplit) {
  struct { int ts, blocks; float fast, exact; } kinds[] = {{256, 1, 1.45f, 3.0f}, {128, 1, 0.42f, 0.75f}, {64, 2, 0.30f, 0.40f}};
  float best = 1e30f;
  tile = 128;
  ksplit = 1;
  const long cus = cu_count();
  const int few = (min(M, N) + 15) / 16 * 16;
  if (few <= FP8_FEW) {
    // a block reads its 16 long rows and all of the short operand, at about 30 KB/us on a CU
    const long blocks = (max(M, N) + 15) / 16;
    best = (float)((blocks + cus - 1) / cus) * (float)(few + 16) * (float)nk * (128.f / 30e3f) + 3.f;
    tile = 0;
    if (few == 16) return;
  }
  for (auto& k : kinds) {
    const long tiles = (long)((M + k.ts - 1) / k.ts) * ((N + k.ts - 1) / k.ts);
    for (int s = 1; s <= 8; s *= 2) {
      if (s > 1 && (k.ts == 256 || nk < 4 * s)) break;
      const float rounds = (float)((tiles * s + cus * k.blocks - 1) / (cus * k.blocks));
      float t = rounds * ((float)((nk + s - 1) / s) * (exact ? k.exact : k.fast) + 5.f);
      if (s > 1) t += 5.f + (float)M * (float)N * (float)(8 * s) / 1.5e6f;
      if (t < best) { best = t; tile = k.ts; ksplit = s; }
    }
  }
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
  const dim3 grid((unsigned)(rb * cb)), block(256);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == DT_BF16) hipLaunchKernelGGL(fp8_quantize_kernel<uint16_t>, grid, block, 0, s, p);
  else hipLaunchKernelGGL(fp8_quantize_kernel<float>, grid, block, 0, s, p);
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

// tile size (low 16 bits) and K slices (high 16) that dllm_fp8_gemm should be given; ksplit > 1 needs ksplit * M * N floats.
// `pitch`: the larger of the operands' row strides.  -1 for sizes that no kernel takes: a pitch above FP8_PITCH with more than
// FP8_FEW rows on both sides, more than FP8_LONG rows next to few
int dllm_fp8_gemm_plan(int M, int N, int nk, int out_dtype, long pitch) {
  int tile, ksplit;
  fp8_plan(M, N, nk, out_dtype == DT_F32, tile, ksplit);
  if (nk == 0 && tile == 256) tile = 128;
  if (tile != 0 && nk > 0 && pitch > FP8_PITCH) {
    if (min(M, N) > FP8_FEW) return -1;
    tile = 0;
    ksplit = 1;
  }
  if (tile == 0 && max(M, N) > FP8_LONG) return -1;
  return tile | ksplit << 16;
}

// C [M, N] (out_dtype) from A [M, 128 nk], B [N, 128 nk].  epi: EPI_STORE / EPI_ACT / EPI_DACT.
int dllm_fp8_gemm(const void* A, long lda, const void* SA, long ldsa, int fa, const void* B, long ldb, const void* SB,
                  long ldsb, int fb, void* C, long ldc, int out_dtype, const void* aux, void* aux_out, long ldaux, int M,
                  int N, int nk, float alpha, float beta, int epi, int act, int tile, int ksplit, float* ws,
                  void* stream) {
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
                C, ldc, aux, aux_out, ldaux, M, N, nk, alpha, beta, act, tile, ksplit, ws};
  if (tile == 0) {
    if (min(M, N) > FP8_FEW || max(M, N) > FP8_LONG || ksplit != 1) return -1;
  } else {
    // scale words span 4 (2) rows, which these have
    if (min(M, N) <= 16 || (tile != 64 && tile != 128 && tile != 256) || ksplit < 1 || ksplit > 8 || (ksplit > 1 && (ws == nullptr || tile == 256)))
      return -1;
    if ((nk > 0 && max(lda, ldb) > FP8_PITCH) || (nk == 0 && tile == 256)) return -1;
  }
  hipStream_t s = (hipStream_t)stream;
  const bool bf = out_dtype == DT_BF16;
  switch (epi) {
    case EPI_STORE: return (int)(bf ? launch_fp8<EPI_STORE, uint16_t>(p, fa, fb, s) : launch_fp8<EPI_STORE, float>(p, fa, fb, s));
    case EPI_ACT: return (int)(bf ? launch_fp8<EPI_ACT, uint16_t>(p, fa, fb, s) : launch_fp8<EPI_ACT, float>(p, fa, fb, s));
    default: return (int)(bf ? launch_fp8<EPI_DACT, uint16_t>(p, fa, fb, s) : launch_fp8<EPI_DACT, float>(p, fa, fb, s));
  }
}

// ---- the linear layer's calls: the quantisations and products of one direction, their temporaries in one workspace ----
struct LinWs {
  uint8_t *a, *sa, *b, *sb;    // two quantised operands [ra, pad128(ka)], [rb, pad128(kb)] and their scales
  float* part;                 // K slices' sums of whichever product runs
  long bytes;
};
static LinWs lin_ws(char* base, long ra, long ka, long rb, long kb, long part) {
  LinWs w;
  long o = 0;
  auto take = [&](long n) {
    char* p = base + o;
    o += (n + 255) / 256 * 256;
    return p;
  };
  const long na = (ka + 127) / 128, nb = (kb + 127) / 128;
  w.a = (uint8_t*)take(ra * na * 128); w.sa = (uint8_t*)take(na * ra);
  w.b = (uint8_t*)take(rb * nb * 128); w.sb = (uint8_t*)take(nb * rb);
  w.part = (float*)take(part * 4);
  w.bytes = o;
  return w;
}
// floats that a product's K slices need; operands in rows of `pitch` bytes
static long lin_part(int M, int N, int K, int odt, long pitch) {
  const int t = dllm_fp8_gemm_plan(M, N, (K + 127) / 128, odt, pitch) >> 16;
  return t > 1 ? (long)t * M * N : 0;
}
static long pad_k(int k) { return ((long)k + 127) / 128 * 128; }
static int lin_gemm(const uint8_t* A, long lda, const uint8_t* SA, long ldsa, int fa, const uint8_t* B, long ldb,
                    const uint8_t* SB, long ldsb, int fb, void* C, long ldc, int odt, int M, int N, int K, float beta, float* part,
                    void* stream) {
  const int nk = (K + 127) / 128, t = dllm_fp8_gemm_plan(M, N, nk, odt, max(lda, ldb));
  if (t < 0) return -1;
  return dllm_fp8_gemm(A, lda, SA, ldsa, fa, B, ldb, SB, ldsb, fb, C, ldc, odt, nullptr, nullptr, 0, M, N, nk, 1.f, beta, EPI_STORE,
                       ACT_NONE, t & 0xffff, t >> 16, part, stream);
}

// bytes of workspace of dllm_linear_fp8 (y of type odt) and of dllm_linear_fp8_bwd (dx, dw of types dxdt, dwdt, dxdt = -1: no dx;
// wt and xt in rows of ldwt and ldxt bytes)
long dllm_linear_fp8_workspace(int T, int D, int F, int odt) { return lin_ws(nullptr, T, D, F, D, lin_part(T, F, D, odt, pad_k(D))).bytes; }
static LinWs lin_bwd_ws(char* base, int T, int D, int F, int dxdt, int dwdt, long ldwt, long ldxt) {
  const long dw = lin_part(F, D, T, dwdt, max(pad_k(T), ldxt));
  if (dxdt < 0) return lin_ws(base, 0, 0, F, T, dw);
  return lin_ws(base, T, F, F, T, max(lin_part(T, D, F, dxdt, max(pad_k(F), ldwt)), dw));
}
long dllm_linear_fp8_bwd_workspace(int T, int D, int F, int dxdt, int dwdt, long ldwt, long ldxt) {
  return lin_bwd_ws(nullptr, T, D, F, dxdt, dwdt, ldwt, ldxt).bytes;
}

// y [T, F] = x [T, D] w [F, D]^T; leaves x^T [D, T] and w^T [D, F] in 8 bits (rows of pad128 codes, dense scales)
int dllm_linear_fp8(const void* x, int xdt, long ldx, const void* w, int wdt, long ldw, int T, int D, int F, void* xt, void* sxt,
                    void* wt, void* swt, void* y, int odt, long ldy, void* ws, long ws_bytes, void* stream) {
  if (T <= 0 || D <= 0 || F <= 0 || (odt != DT_BF16 && odt != DT_F32)) return -1;
  const LinWs l = lin_ws((char*)ws, T, D, F, D, lin_part(T, F, D, odt, pad_k(D)));
  if (ws == nullptr || (uintptr_t)ws % 256 || ws_bytes < l.bytes) return -1;
  const long pd = pad_k(D), pt = pad_k(T), pf = pad_k(F);
  int rc = dllm_fp8_quantize(x, xdt, ldx, T, D, l.a, pd, l.sa, T, xt, pt, sxt, D, F8_E4M3, F8_E4M3, 0, stream);
  if (rc == 0) rc = dllm_fp8_quantize(w, wdt, ldw, F, D, l.b, pd, l.sb, F, wt, pf, swt, D, F8_E4M3, F8_E4M3, 1, stream);
  if (rc == 0) rc = lin_gemm(l.a, pd, l.sa, T, F8_E4M3, l.b, pd, l.sb, F, F8_E4M3, y, ldy, odt, T, F, D, 0.f, l.part, stream);
  return rc;
}

// dx [T, D] = dy [T, F] w (skipped where dx is null), dw [F, D] = dy^T x + beta dw, from dy in e5m2
int dllm_linear_fp8_bwd(const void* dy, int ydt, long ldy, int T, int D, int F, const void* xt, long ldxt, const void* sxt,
                        long ldsxt, int fx, const void* wt, long ldwt, const void* swt, long ldswt, int fw, void* dx, int dxdt,
                        long lddx, void* dw, int dwdt, long lddw, float beta, void* ws, long ws_bytes, void* stream) {
  if (T <= 0 || D <= 0 || F <= 0 || (dwdt != DT_BF16 && dwdt != DT_F32) || (dx && dxdt != DT_BF16 && dxdt != DT_F32)) return -1;
  const LinWs l = lin_bwd_ws((char*)ws, T, D, F, dx ? dxdt : -1, dwdt, ldwt, ldxt);
  if (ws == nullptr || (uintptr_t)ws % 256 || ws_bytes < l.bytes || dw == nullptr) return -1;
  const long pt = pad_k(T), pf = pad_k(F);
  int rc = dllm_fp8_quantize(dy, ydt, ldy, T, F, dx ? l.a : nullptr, pf, dx ? l.sa : nullptr, T, l.b, pt, l.sb, F, F8_E5M2, F8_E5M2, 0,
                             stream);
  if (rc == 0 && dx)
    rc = lin_gemm(l.a, pf, l.sa, T, F8_E5M2, (const uint8_t*)wt, ldwt, (const uint8_t*)swt, ldswt, fw, dx, lddx, dxdt, T, D, F, 0.f,
                  l.part, stream);
  if (rc == 0)
    rc = lin_gemm(l.b, pt, l.sb, F, F8_E5M2, (const uint8_t*)xt, ldxt, (const uint8_t*)sxt, ldsxt, fx, dw, lddw, dwdt, F, D, T, beta,
                  l.part, stream);
  return rc;
}

}  // extern "C"
