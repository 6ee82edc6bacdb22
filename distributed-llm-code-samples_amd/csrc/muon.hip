// Newton-Schulz orthogonalisation of 2-D updates and the Muon optimizer step.
//
// X0 = U / (|U|_F + eps) with the shorter side m as rows (m <= n), then `steps` times
//     A = X X^T,   X <- P X,   P = a I + b A + c A^2,   (a, b, c) = (3.4445, -4.7750, 2.0315)
// which pulls every singular value of X towards 1 and keeps the singular vectors.  All P are polynomials of one symmetric
// matrix, so they commute and stay symmetric, and the next A is P A P: up to three steps run on the m x m side alone,
//     Q = P_k ... P_1,   A <- (P A) P
// and X is multiplied by Q once at the end of such a segment.  Segments cost less (for n = 4 m, counting symmetric products
// half: 19 products of m x m x m for 3 + 2 steps, 32.5 for single steps) and lose digits: a Gram matrix's small eigenvalues
// are squares of small singular values, and its rounding is amplified as they are (12 a step).  Errors against 64 bits, 16 x 16 to
// 4096 x 16384 (the same iteration in plain fp32): normal matrices 5e-7 to 3e-6 in single steps, 2e-6 to 3e-6 in segments (7e-7 to
// 9e-6); a few strong directions over noise, singular values over three decades, 4e-6 to 1.6e-5 and 8e-6 to 2.4e-5 (3e-6 to 4e-5).
// So a result handed out in fp32 runs single steps; a bf16 result (half a step 4e-3) and a weight update (which scales the
// result by the learning rate before adding it) run segments of three.
//
// Every matrix is held as two fp16 planes, v = 2^-s (hi + lo): 22 bits, fp32's to within two.  A product of two such
// matrices is hi hi + hi lo + lo hi on the fp16 matrix instructions with fp32 accumulation (the missing lo lo is 2^-22 of
// the product).  Single bf16 or fp16 planes would be three times cheaper and lose 2 to 20 % of the result (bf16), 0.1 to
// 3 % (fp16): gradients have singular values thousands of times smaller than the largest, and rounding noise of the large
// ones is amplified with them (3.44 a step).  The scales s are fixed: |X| <= 1.21, |A| <= 1.46, |P| <= 3.45, |Q| <= 41
// (three steps) bound every entry below fp16's 65504.
#include <type_traits>

#include "common.h"
#include "nt8.h"

namespace dllm {

typedef _Float16 f16;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4_t;
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));   // unaligned 16-byte accesses
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;
constexpr int SX = 15, SA = 15, SP = 14, SQ = 10;   // plane scales 2^s of X, A (and P A), P, products of P
constexpr int NS_SEGMENT = 3;                        // steps on one Gram matrix where the result allows it
constexpr int NS_PARTS = 256;                        // partial sums of squares per matrix

// The empty asm makes v one fp32 number: where v is a product, the compiler otherwise rounds it to fp16 directly for one use
// of h and by way of fp32 for another, and where the two differ hi + lo is off by a step of hi.
__device__ __forceinline__ void split16(float v, f16& h, f16& l) {
  asm("" : "+v"(v));
  h = (f16)v;
  l = (f16)(v - (float)h);
}

enum NsIn : int { NS_ORTH = 0, NS_MUON = 1 };

struct MuonIn {
  const void* g; int gdt;     // update (NS_ORTH) or gradient, [B][R][C], DT_BF16 / DT_F32
  float* mom;                 // momentum [B][R][C] (NS_MUON)
  float beta, gscale;
  int nesterov;
  int R, C;
  int il, B;                  // il > 0: the rows of the B matrices alternate in blocks of il (one [B R][C] tensor)
};
// first element of row r of matrix z
__device__ __forceinline__ long muon_row(int il, int B, int R, int C, int z, int r) {
  return (il ? ((long)(r / il) * B + z) * il + r % il : (long)z * R + r) * C;
}

__device__ __forceinline__ float ld_g(const MuonIn& p, long i) {
  return p.gdt == DT_BF16 ? bf2f(((const uint16_t*)p.g)[i]) : ((const float*)p.g)[i];
}

// u of element i after the momentum update
template <int KIND>
__device__ __forceinline__ float muon_u(const MuonIn& p, long i) {
  if constexpr (KIND == NS_ORTH) return ld_g(p, i);
  const float m = p.mom[i];
  return p.nesterov ? fmaf(p.beta, m, p.gscale * ld_g(p, i)) : m;
}

// four elements of g / of u at i
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
__device__ __forceinline__ f32x4_t ld_g4(const MuonIn& p, long i) {
  if (p.gdt != DT_BF16) return *(const f32x4_any*)((const float*)p.g + i);
  const u32x2_any w = *(const u32x2_any*)((const uint16_t*)p.g + i);
  return f32x4_t{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                 __uint_as_float(w.y & 0xffff0000u)};
}
template <int KIND>
__device__ __forceinline__ f32x4_t muon_u4(const MuonIn& p, long i) {
  if constexpr (KIND == NS_ORTH) return ld_g4(p, i);
  const f32x4_t m = *(const f32x4_any*)(p.mom + i);
  if (!p.nesterov) return m;
  const f32x4_t g = ld_g4(p, i);
  f32x4_t u;
#pragma unroll
  for (int k = 0; k < 4; ++k) u[k] = fmaf(p.beta, m[k], p.gscale * g[k]);
  return u;
}

// momentum update and the partial sums of u^2 (64-bit: gradients of any magnitude, and a sum that does not depend on how it
// is cut).  grid (NS_PARTS, B).  Bound by HBM: one read of g (and of the momentum, and its write)
template <int KIND>
__device__ __forceinline__ double muon_sumsq_part(const MuonIn& p, int z, long n) {
  double s = 0.0;
  const long chunk = (long)p.il * p.C;                       // contiguous elements of one matrix (0: all)
  auto at = [&](long i) { return p.il ? (i / chunk * p.B + z) * chunk + i % chunk : (long)z * n + i; };
  const long n4 = chunk % 4 == 0 ? n >> 2 : 0, stride = (long)gridDim.x * blockDim.x, t0 = (long)blockIdx.x * blockDim.x + threadIdx.x;
#pragma unroll 4
  for (long j = t0; j < n4; j += stride) {
    const long i = at(4 * j);
    if constexpr (KIND == NS_MUON) {
      const f32x4_t g = ld_g4(p, i);
      f32x4_t m = *(const f32x4_any*)(p.mom + i);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        m[k] = fmaf(p.beta, m[k], p.gscale * g[k]);
        const double u = (double)(p.nesterov ? fmaf(p.beta, m[k], p.gscale * g[k]) : m[k]);
        s += u * u;
      }
      *(f32x4_any*)(p.mom + i) = m;
    } else {
      const f32x4_t u = ld_g4(p, i);
#pragma unroll
      for (int k = 0; k < 4; ++k) s += (double)u[k] * (double)u[k];
    }
  }
  for (long j = 4 * n4 + t0; j < n; j += stride) {
    const long i = at(j);
    if constexpr (KIND == NS_MUON) p.mom[i] = fmaf(p.beta, p.mom[i], p.gscale * ld_g(p, i));
    const double u = (double)muon_u<KIND>(p, i);
    s += u * u;
  }
  return s;
}
template <int KIND>
__global__ __launch_bounds__(1024) void muon_sumsq_kernel(MuonIn p, double* part) {
  __shared__ double red[16];
  const int z = blockIdx.y;
  double s = muon_sumsq_part<KIND>(p, z, (long)p.R * p.C);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) s += __shfl_down(s, d);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += red[i];
    part[(long)blockIdx.y * NS_PARTS + blockIdx.x] = t;
  }
}

// X0 planes in both orientations: same [Rp][Cp] and transposed [Cp][Rp], zeros outside [R][C].  64x64 tiles, grid
// (Cp / 64, Rp / 64, B).  Bound by HBM: reads u once, writes four 2-byte planes
template <int KIND>
__global__ __launch_bounds__(256) void ns_split_kernel(MuonIn p, const double* part, float eps, f16* same, f16* tr, int Rp,
                                                       int Cp) {
  __shared__ double red[4];
  __shared__ float tile[64][65];
  const int t = threadIdx.x;
  double s = part[(long)blockIdx.z * NS_PARTS + t];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) s += __shfl_down(s, d);
  if ((t & 63) == 0) red[t >> 6] = s;
  __syncthreads();
  const double norm = sqrt((red[0] + red[1]) + (red[2] + red[3]));
  const float inv = (float)((double)(1 << SX) / (norm + (double)eps));
  const long plane = (long)Rp * Cp;
  f16* so = same + (long)blockIdx.z * 2 * plane;
  f16* to = tr + (long)blockIdx.z * 2 * plane;
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64, q = t >> 4, j = 4 * (t & 15);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + 16 * i + q, c = c0 + j;
    f32x4_t v = {0.f, 0.f, 0.f, 0.f};
    if (r < p.R && c < p.C) {
      const long o = muon_row(p.il, p.B, p.R, p.C, blockIdx.z, r) + c;
      if (c + 4 <= p.C) {
        v = muon_u4<KIND>(p, o);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (c + k < p.C) v[k] = muon_u<KIND>(p, o + k);
      }
    }
    f16x4_t h, l;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f16 hh, ll;
      split16(v[k] * inv, hh, ll);
      h[k] = hh;
      l[k] = ll;
      tile[16 * i + q][j + k] = v[k] * inv;
    }
    *(f16x4_t*)(so + (long)r * Cp + c) = h;
    *(f16x4_t*)(so + plane + (long)r * Cp + c) = l;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f16x4_t h, l;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f16 hh, ll;
      split16(tile[j + k][16 * i + q], hh, ll);
      h[k] = hh;
      l[k] = ll;
    }
    const long o = (long)(c0 + 16 * i + q) * Rp + r0 + j;
    *(f16x4_t*)(to + o) = h;
    *(f16x4_t*)(to + plane + o) = l;
  }
}

// ----------------------------------------------------------------------------------------------
// product of two plane pairs, C[M, N] = A[M, K] B[N, K]^T (both K-contiguous; every size a multiple of 128)
// ----------------------------------------------------------------------------------------------
enum NsEpi : int { NS_PLANES = 0, NS_PLANES_T = 1, NS_POLY = 2, NS_OUT = 3, NS_STEP = 4 };

struct NsGemm {
  const f16* A; long lda, pa, ba;      // hi plane; lo plane at + pa; next matrix of the batch at + ba
  const f16* B; long ldb, pb, bb;
  int M, N, K;
  float cs;                            // accumulator -> output scale
  f16* out; long ldo, po, bo;          // planes (NS_PLANES / NS_PLANES_T / NS_POLY)
  f16* outT; long ldt, pt, bt;         // transposed planes (NS_PLANES_T)
  const f16* aux; float cb, ca;        // NS_POLY: A's planes (out's layout), b's factor, a on the diagonal
  void* C; int cdt, R, Cc;             // NS_OUT: result [R][Cc] (DT_BF16 / DT_F32);  NS_STEP: rows / columns of W
  int il, nb;                          // NS_STEP: alternating rows, as in MuonIn
  float* w; uint16_t* copy; int16_t* lo; float decay, rate;   // NS_STEP: fp32 master (+ bf16 copy), or split (lo, copy)
  int ksplit; float* part;             // slices of K, each block's fp32 sums to part (ns_join adds them)
  int sym;                             // the product is symmetric: tiles on and below the diagonal, mirrored on writing
};

// columns n .. n + 7 of row m of the result: written out (NS_OUT), or into the weights (NS_STEP)
template <int EPI>
__device__ __forceinline__ void ns_result8(const NsGemm& p, int z, int m, int n, const float (&v)[8]) {
  if (m >= p.R || n >= p.Cc) return;
  const long o = muon_row(p.il, p.nb, p.R, p.Cc, z, m) + n;
  if (n + 8 <= p.Cc) {   // 16-byte accesses at any element's address
    if constexpr (EPI == NS_OUT) {
      if (p.cdt == DT_BF16) {
        u32x4_any u;
        u.x = f2bf(p.cs * v[0]) | (uint32_t)f2bf(p.cs * v[1]) << 16; u.y = f2bf(p.cs * v[2]) | (uint32_t)f2bf(p.cs * v[3]) << 16;
        u.z = f2bf(p.cs * v[4]) | (uint32_t)f2bf(p.cs * v[5]) << 16; u.w = f2bf(p.cs * v[6]) | (uint32_t)f2bf(p.cs * v[7]) << 16;
        *(u32x4_any*)((uint16_t*)p.C + o) = u;
      } else {
        *(f32x4_any*)((float*)p.C + o) = f32x4_any{p.cs * v[0], p.cs * v[1], p.cs * v[2], p.cs * v[3]};
        *(f32x4_any*)((float*)p.C + o + 4) = f32x4_any{p.cs * v[4], p.cs * v[5], p.cs * v[6], p.cs * v[7]};
      }
    } else if (p.lo != nullptr) {
      const u32x4_any wh = *(const u32x4_any*)(p.copy + o), wl = *(const u32x4_any*)((const uint16_t*)p.lo + o);
      uint32_t h[4] = {wh.x, wh.y, wh.z, wh.w}, l[4] = {wl.x, wl.y, wl.z, wl.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float a, b;
        split_join2(h[k], l[k], a, b);
        split_part2(fmaf(-p.rate, p.cs * v[2 * k], a * p.decay), fmaf(-p.rate, p.cs * v[2 * k + 1], b * p.decay), h[k], l[k]);
      }
      *(u32x4_any*)(p.copy + o) = u32x4_any{h[0], h[1], h[2], h[3]};
      *(u32x4_any*)((uint16_t*)p.lo + o) = u32x4_any{l[0], l[1], l[2], l[3]};
    } else {
      f32x4_any a = *(const f32x4_any*)(p.w + o), b = *(const f32x4_any*)(p.w + o + 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        a[k] = fmaf(-p.rate, p.cs * v[k], a[k] * p.decay);
        b[k] = fmaf(-p.rate, p.cs * v[4 + k], b[k] * p.decay);
      }
      *(f32x4_any*)(p.w + o) = a;
      *(f32x4_any*)(p.w + o + 4) = b;
      if (p.copy) {
        u32x4_any u;
        u.x = f2bf(a[0]) | (uint32_t)f2bf(a[1]) << 16; u.y = f2bf(a[2]) | (uint32_t)f2bf(a[3]) << 16;
        u.z = f2bf(b[0]) | (uint32_t)f2bf(b[1]) << 16; u.w = f2bf(b[2]) | (uint32_t)f2bf(b[3]) << 16;
        *(u32x4_any*)(p.copy + o) = u;
      }
    }
    return;
  }
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    if (n + r >= p.Cc) return;
    const float x = p.cs * v[r];
    if constexpr (EPI == NS_OUT) {
      if (p.cdt == DT_BF16) ((uint16_t*)p.C)[o + r] = f2bf(x);
      else ((float*)p.C)[o + r] = x;
    } else if (p.lo != nullptr) {
      const float w = split_join(p.copy[o + r], (uint16_t)p.lo[o + r]);
      uint16_t h, l;
      split_part(fmaf(-p.rate, x, w * p.decay), h, l);
      p.copy[o + r] = h;
      p.lo[o + r] = (int16_t)l;
    } else {
      const float w = fmaf(-p.rate, x, p.w[o + r] * p.decay);
      p.w[o + r] = w;
      if (p.copy) p.copy[o + r] = f2bf(w);
    }
  }
}

// 256x256 tiles on the 8-phase loop (nt8.h): the three plane pairs as one run of 3 K / 64 K steps
struct NsTrait {
  const char *a, *b;
  long pa, pb;          // bytes from the hi to the lo plane
  int per;              // pairs of K steps per plane pair
  int seg = 0, left;
  __device__ __forceinline__ int advance(const char*& an, const char*& bn, int) {
    if (--left > 0) {
      an += 256;
      bn += 256;
    } else if (seg < 2) {   // (hi, lo) -> (lo, hi) -> (hi, hi)
      an = a + (seg == 0 ? pa : 0);
      bn = b;
      ++seg;
      left = per;
    }
    return 128;
  }
  template <class ODD> __device__ __forceinline__ void load(ODD, int) {}
  template <int QM, int QN, int ODD>
  __device__ __forceinline__ void mma(f32x4_t (&c)[4][2], N8Frag (&fa)[4], N8Frag (&fb)[2]) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
          c[mt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, s ? fb[nt].hi : fb[nt].lo),
                                                             __builtin_bit_cast(f16x8_t, s ? fa[mt].hi : fa[mt].lo),
                                                             c[mt][nt], 0, 0, 0);
  }
};

// one row group of a lane: 8 columns n .. n + 7 of row m (v[e]), scaled and with the polynomial's other terms
template <int EPI>
__device__ __forceinline__ void ns_value8(const NsGemm& p, int z, int m, int n, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] *= p.cs;
  if constexpr (EPI == NS_POLY) {
    const long o = (long)z * p.bo + (long)m * p.ldo + n;
    const f16x8_t ah = *(const f16x8_t*)(p.aux + o), al = *(const f16x8_t*)(p.aux + p.po + o);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      v[e] += p.cb * ((float)ah[e] + (float)al[e]) + (m == n + e ? p.ca : 0.f);
  }
}

// The block's tile: matrix z and origin.  Blocks that run on one XCD (whose L2 they share) get consecutive tiles of all
// matrices in a row, and consecutive tiles lie close together: bands of rows, column by column -- of the whole matrix, or
// of its lower triangle (symmetric products).  32 tiles then need about 12 row panels, row by row they need 24 and the
// products are bound by what lies behind the L2.
template <int TS>
__device__ __forceinline__ void ns_tile(const NsGemm& p, int& z, int& m0, int& n0) {
  const int tm = (p.M + TS - 1) / TS, tn = (p.N + TS - 1) / TS, nt = p.sym ? tm * (tm + 1) / 2 : tm * tn;
  int t = xcd_remap(blockIdx.x, gridDim.x);
  z = t / nt;
  t -= z * nt;
  constexpr int H = 6;
  if (!p.sym) {
    const int band = t / (H * tn), h = min(tm - band * H, H), in = t - band * H * tn;
    m0 = (band * H + in % h) * TS;
    n0 = in / h * TS;
    return;
  }
  int r0 = 0;                                                    // first row of the band; r0 (r0 + 1) / 2 tiles before it
  while (r0 + H < tm && (r0 + H) * (r0 + H + 1) / 2 <= t) r0 += H;
  const int h = min(tm - r0, H);
  t -= r0 * (r0 + 1) / 2;
  int c = t / h, r = t - c * h;                                  // columns 0 .. r0 are h tiles high
  if (c > r0) {                                                  // the triangle at the band's end
    t -= (r0 + 1) * h;
    c = 1;
    while (t >= h - c) t -= h - c++;
    r = c + t;
    c += r0;
  }
  m0 = (r0 + r) * TS;
  n0 = c * TS;
}
static __host__ __device__ inline int ns_tiles(const NsGemm& p, int ts) {
  const int a = (p.M + ts - 1) / ts, b = (p.N + ts - 1) / ts;
  return p.sym ? a * (a + 1) / 2 : a * b;
}

// A symmetric product's elements above the diagonal, and whether the lane's rows from m and columns from n are written as
// they are (0), also mirrored (1), or left to the mirror (-1).  Above and below the diagonal the same number is rounded
// differently: the plane pairs are added in exchanged order, and (P A) P is symmetric only up to rounding.  So which of the
// two is taken goes by 64x64 blocks, whatever the tile: on the diagonal each its own, elsewhere the lower one.  The tile depends on
// the batch (ns_launch), a matrix's bits do not.  (Tiles are multiples of 64, no lane's rows or columns cross that border
// but those of 192x192 tiles, which ask row by row.)
template <int EPI>
__device__ __forceinline__ int ns_half(const NsGemm& p, int m, int n) {
  if (EPI != NS_PLANES && EPI != NS_POLY) return 0;
  if (!p.sym) return 0;
  const int d = (m >> 6) - (n >> 6);
  return d > 0 ? 1 : d < 0 ? -1 : 0;
}

// the tile's results from its accumulators
template <int EPI>
__device__ __forceinline__ void ns_finish(const NsGemm& p, int z, int m0, int n0, int wid, int lane,
                                          const f32x4_t (&acc)[2][2][4][2]) {
  constexpr bool PL = EPI == NS_PLANES || EPI == NS_PLANES_T || EPI == NS_POLY;
  f16* tp = EPI == NS_PLANES_T ? p.outT + (long)z * p.bt : p.out + (long)z * p.bo;
  const long ldt = EPI == NS_PLANES_T ? p.ldt : p.ldo, pt = EPI == NS_PLANES_T ? p.pt : p.po;
#pragma unroll
  for (int qm = 0; qm < 2; ++qm)
#pragma unroll
    for (int qn = 0; qn < 2; ++qn) {
      const int n = n0 + n8_col(wid, lane, qn), half = ns_half<EPI>(p, m0 + n8_row(wid, lane, qm, 0), n);
      if (half < 0) continue;
      f16x4_t th[8], tl[8];   // transposed planes: column n + e, rows of the four mt
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        const int m = m0 + n8_row(wid, lane, qm, mt);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = acc[qm][qn][mt][e & 1][e >> 1];
        if constexpr (PL) {
          ns_value8<EPI>(p, z, m, n, v);
          f16x8_t h, l;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            f16 hh, ll;
            split16(v[e], hh, ll);
            h[e] = hh;
            l[e] = ll;
            th[e][mt] = hh;
            tl[e][mt] = ll;
          }
          const long o = (long)z * p.bo + (long)m * p.ldo + n;
          *(f16x8_t*)(p.out + o) = h;
          *(f16x8_t*)(p.out + p.po + o) = l;
        } else {
          ns_result8<EPI>(p, z, m, n, v);
        }
      }
      if (EPI == NS_PLANES_T || half > 0) {
        const int m = m0 + n8_row(wid, lane, qm, 0);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const long q = (long)(n + e) * ldt + m;
          *(f16x4_t*)(tp + q) = th[e];
          *(f16x4_t*)(tp + pt + q) = tl[e];
        }
      }
    }
}

template <int EPI>
__global__ __launch_bounds__(512, 2) void ns_gemm_256(NsGemm p) {
  __shared__ __attribute__((aligned(16))) char smem[N8_LDS];
  DLLM_LDS char* lds = (DLLM_LDS char*)smem;
  const int t = threadIdx.x, lane = t & 63;
  const int wid = __builtin_amdgcn_readfirstlane(t >> 6);
  int z, m0, n0;
  ns_tile<256>(p, z, m0, n0);
  uint32_t ao[2][2], bo[2][2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    n8_offsets<true>(p.lda * 2, h, 255, wid, lane, ao[h]);
    n8_offsets<false>(p.ldb * 2, h, 255, wid, lane, bo[h]);
  }
  f32x4_t acc[2][2][4][2];
#pragma unroll
  for (int i = 0; i < 32; ++i) (&acc[0][0][0][0])[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  NsTrait tr;
  tr.a = (const char*)(p.A + (long)z * p.ba + (long)m0 * p.lda);
  tr.b = (const char*)(p.B + (long)z * p.bb + (long)n0 * p.ldb);
  tr.pa = p.pa * 2;
  tr.pb = p.pb * 2;
  tr.per = tr.left = p.K >> 7;
  n8_loop(tr, lds, tr.a, tr.b + tr.pb, 128, ao, bo, 3 * (p.K >> 7), wid, lane, acc);
  ns_finish<EPI>(p, z, m0, n0, wid, lane, acc);
}

// ----------------------------------------------------------------------------------------------
// 64x64 (F = 2), 128x128 (F = 4) and 192x192 (F = 6) tiles: four waves, one per SIMD, each 16F x 16F
//
// For products whose 256x256 tiles do not fill the CUs: a symmetric 4096 x 4096 product has 136 of those and takes one
// round on 256 CUs as the full 256 tiles do, but 253 of 192 x 192, one round of 0.56 of the work.
// STAGES K steps of LDS ring, filled by LDS-DMA that many steps ahead; per K step one barrier.  A wave reads the next step's
// fragments while it computes the current one's; reads and fetches are placed between matrix instructions (order pinned,
// reads first so that they are back by the step's end), so that the one wave of a SIMD keeps its matrix pipe busy.  Rows are permuted in LDS (slot 16 f + i holds row F i
// + f of the wave's piece), so a lane ends with F consecutive rows by 4F consecutive columns.
// ----------------------------------------------------------------------------------------------
template <int F> struct W4 {
  static constexpr int TS = 32 * F, OPB = TS * 128, STAGE = 2 * OPB;      // bytes of an operand's / a step's LDS
  static constexpr int STAGES = F == 6 ? 3 : 4;
  static constexpr int LDS = STAGES * STAGE;
};

// the tile's results from a lane's accumulators
template <int EPI, int F>
__device__ __forceinline__ void ns_w4_finish(const NsGemm& p, int z, int m0, int n0, int wid, int lane, const f32x4_t (&acc)[F][F]) {
  const int i15 = lane & 15, g = lane >> 4, wr = wid >> 1, wc = wid & 1;
  // lane: rows mb .. mb + F - 1, columns nb .. nb + 4F - 1 (column F r + k of them: acc[.][k][r])
  constexpr bool PL = EPI == NS_PLANES || EPI == NS_PLANES_T || EPI == NS_POLY;
  f16* tp = EPI == NS_PLANES_T ? p.outT + (long)z * p.bt : p.out + (long)z * p.bo;
  const long ldt = EPI == NS_PLANES_T ? p.ldt : p.ldo, pt = EPI == NS_PLANES_T ? p.pt : p.po;
  const int mb = m0 + wr * 16 * F + F * i15, nb = n0 + wc * 16 * F + 4 * F * g;
#pragma unroll
  for (int c8 = 0; c8 < F / 2; ++c8) {            // 8 columns at a time
    const int n = nb + 8 * c8;
    if (n >= p.N) continue;
    f16 th[8][F], tl[8][F];
#pragma unroll
    for (int i = 0; i < F; ++i) {
      const int m = mb + i;
      if (m < p.M && ns_half<EPI>(p, m, n) >= 0) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = acc[i][(8 * c8 + e) % F][(8 * c8 + e) / F];
        if constexpr (PL) {
          ns_value8<EPI>(p, z, m, n, v);
          f16x8_t h, l;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            f16 hh, ll;
            split16(v[e], hh, ll);
            h[e] = hh; l[e] = ll;
            th[e][i] = hh; tl[e][i] = ll;
          }
          const long o = (long)z * p.bo + (long)m * p.ldo + n;
          *(f16x8_t*)(p.out + o) = h;
          *(f16x8_t*)(p.out + p.po + o) = l;
        } else {
          ns_result8<EPI>(p, z, m, n, v);
        }
      }
    }
    if (EPI == NS_PLANES_T || ns_half<EPI>(p, mb + F - 1, n) > 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f16* o = tp + (long)(n + e) * ldt + mb;
#pragma unroll
        for (int i = 0; i < F; i += 2) {          // rows are even, M a multiple of 128: pairs are on one side of its end
          if (mb + i < p.M && (EPI == NS_PLANES_T || ns_half<EPI>(p, mb + i, n) > 0)) {   // (and of a 64x64 block's)
            typedef __attribute__((ext_vector_type(2))) _Float16 f16x2_t;
            *(f16x2_t*)(o + i) = f16x2_t{th[e][i], th[e][i + 1]};
            *(f16x2_t*)(o + pt + i) = f16x2_t{tl[e][i], tl[e][i + 1]};
          }
        }
      }
    }
  }
}

template <int EPI, int F>
__device__ __forceinline__ void ns_w4_body(const NsGemm& p, DLLM_LDS char* lds) {
  using W = W4<F>;
  const int t = threadIdx.x, lane = t & 63;
  const int wid = __builtin_amdgcn_readfirstlane(t >> 6);
  const int i15 = lane & 15, g = lane >> 4, wr = wid >> 1, wc = wid & 1;
  int z, m0, n0;
  ns_tile<W::TS>(p, z, m0, n0);
  // a lane's byte offsets of its pieces (rows past the end re-load the last row: their results are not written)
  uint32_t ao[F], bo[F];
#pragma unroll
  for (int i = 0; i < F; ++i) {
    const int s = 8 * (wid + 4 * i) + (lane >> 3);            // LDS slot 0 .. TS - 1
    const int w = s / (16 * F), in = s - w * 16 * F;          // wave piece, slot in it
    const int row = w * 16 * F + F * (in & 15) + (in >> 4), c = (lane & 7) ^ ((s >> 1) & 7);
    ao[i] = (uint32_t)((long)min(row, p.M - 1 - m0) * p.lda * 2 + c * 16);
    bo[i] = (uint32_t)((long)min(row, p.N - 1 - n0) * p.ldb * 2 + c * 16);
  }
  // slice blockIdx.y of the K steps (whole pairs of them)
  const int k0 = (p.K >> 7) * blockIdx.y / p.ksplit * 2, per = (p.K >> 7) * (blockIdx.y + 1) / p.ksplit * 2 - k0, nk = 3 * per;
  const char* A = (const char*)(p.A + (long)z * p.ba + (long)m0 * p.lda + (long)k0 * 64);
  const char* B = (const char*)(p.B + (long)z * p.bb + (long)n0 * p.ldb + (long)k0 * 64);
  // next step to fetch: (hi, lo), (lo, hi), (hi, hi); past the last one it stays there
  const char *fa = A, *fb = B + p.pb * 2;
  int fleft = per, fseg = 0;
  auto next = [&]() {
    if (--fleft > 0) {
      fa += 128;
      fb += 128;
    } else if (fseg < 2) {
      fa = A + (fseg == 0 ? p.pa * 2 : 0);
      fb = B;
      ++fseg;
      fleft = per;
    }
  };
  auto fetch_a = [&](int i, int slot) { n8_dma(fa, ao[i], lds + slot * W::STAGE + (wid + 4 * i) * 1024); };
  auto fetch_b = [&](int i, int slot) { n8_dma(fb, bo[i], lds + slot * W::STAGE + W::OPB + (wid + 4 * i) * 1024); };
  const uint32_t lb = (uint32_t)(uintptr_t)lds;
  const int sw = (i15 >> 1) & 7;
  const uint32_t ra[2] = {lb + (wr * 16 * F + i15) * 128 + ((g ^ sw) << 4), lb + (wr * 16 * F + i15) * 128 + (((4 + g) ^ sw) << 4)};
  const uint32_t rb[2] = {lb + W::OPB + (wc * 16 * F + i15) * 128 + ((g ^ sw) << 4),
                          lb + W::OPB + (wc * 16 * F + i15) * 128 + (((4 + g) ^ sw) << 4)};
  n8_i32x4 xa[2][2][F], xb[2][2][F];   // [step parity][half step][fragment]
  f32x4_t acc[F][F];
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int k = 0; k < F; ++k) acc[i][k] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // read j of a step's 4F: half step 0's A and B fragments, then half step 1's
  auto read = [&](auto par, auto j, uint32_t off) {
    constexpr int h = j.value / (2 * F), f = j.value % (2 * F);
    if constexpr (f < F) n8_read<f * 2048>(xa[par.value][h][f], ra[h] + off);
    else n8_read<(f - F) * 2048>(xb[par.value][h][f - F], rb[h] + off);
  };
  auto mma1 = [&](auto par, int q) {   // q-th of 2 F F
    const int h = q / (F * F), i = q % (F * F) / F, k = q % F;
    acc[i][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, xb[par.value][h][k]),
                                                       __builtin_bit_cast(f16x8_t, xa[par.value][h][i]), acc[i][k], 0, 0, 0);
  };
  auto upto = [](auto n, auto f) {
    [&]<int... J>(std::integer_sequence<int, J...>) { (f(std::integral_constant<int, J>{}), ...); }(std::make_integer_sequence<int, decltype(n)::value>{});
  };
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using NR = std::integral_constant<int, 4 * F>;
  using NF = std::integral_constant<int, 2 * F>;

#pragma unroll
  for (int s = 0; s < W::STAGES; ++s) {
#pragma unroll
    for (int i = 0; i < F; ++i) fetch_a(i, s);
#pragma unroll
    for (int i = 0; i < F; ++i) fetch_b(i, s);
    next();
  }
  auto landed = [] {   // all but the youngest STAGES - 2 steps (2F fetches each) in flight have landed
    if constexpr (F == 2) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    else if constexpr (F == 4) asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(12)" ::: "memory");
  };
  // (STAGES - 1) * 2F: step 0 has landed
  if constexpr (F == 2) asm volatile("s_waitcnt vmcnt(12)" ::: "memory");
  else asm volatile("s_waitcnt vmcnt(24)" ::: "memory");
  N8_BARRIER();
  upto(NR{}, [&](auto j) { read(I0{}, j, 0u); });
  N8_LDS_WAIT();
  int slot = 0;
  // step kt (fragments in registers, its LDS slot free): read step kt + 1, fetch step kt + STAGES into the freed slot
  auto one = [&](auto par, auto other) {
    landed();
    N8_BARRIER();
    const int fs = slot;
    slot = slot + 1 == W::STAGES ? 0 : slot + 1;
    const uint32_t off = (uint32_t)(slot * W::STAGE);
    constexpr int PR = F / 2 - 1;                  // matrix instructions per read (0, 1, 2), then two per fetch
    static_assert(4 * F * PR + 2 * F * 2 == 2 * F * F, "every matrix instruction of the step, once");
    upto(NR{}, [&](auto j) {
      read(other, j, off);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int q = 0; q < PR; ++q) mma1(par, j.value * PR + q);
      __builtin_amdgcn_sched_barrier(0);
    });
    upto(NF{}, [&](auto j) {
      if constexpr (j.value < F) fetch_a(j.value, fs);
      else fetch_b(j.value - F, fs);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int q = 0; q < 2; ++q) mma1(par, 4 * F * PR + j.value * 2 + q);
      __builtin_amdgcn_sched_barrier(0);
    });
    next();
    N8_LDS_WAIT();
  };
  for (int kt = 0; kt < nk; kt += 2) {
    one(I0{}, I1{});
    one(I1{}, I0{});
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

  if constexpr (F == 2 && EPI == NS_PLANES) {
    if (p.ksplit > 1) {
      f32x4_t* o = (f32x4_t*)p.part + ((long)blockIdx.y * gridDim.x + blockIdx.x) * (F * F * 256) + t;
#pragma unroll
      for (int i = 0; i < F * F; ++i) o[i * 256] = acc[i / F][i % F];
      return;
    }
  }
  ns_w4_finish<EPI, F>(p, z, m0, n0, wid, lane, acc);
}

// slices of a product's K added up in order, and its results; grid as the product's, without the slices
template <int EPI>
__global__ __launch_bounds__(256) void ns_join(NsGemm p) {
  const int t = threadIdx.x;
  int z, m0, n0;
  ns_tile<64>(p, z, m0, n0);
  f32x4_t acc[2][2];
  const f32x4_t* q = (const f32x4_t*)p.part + (long)blockIdx.x * 1024 + t;
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i >> 1][i & 1] = q[i * 256];
  for (int k = 1; k < p.ksplit; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i >> 1][i & 1] += q[(long)k * gridDim.x * 1024 + i * 256];
  ns_w4_finish<EPI, 2>(p, z, m0, n0, t >> 6, t & 63, acc);
}

// 128 x 128: dynamic LDS (128 KiB, one block per CU) and a bound of two blocks, so that the compiler stays within 256
// registers; left with 512 it keeps these 64 accumulators in the accumulation file and copies each one around its matrix
// instruction.  192 x 192 tiles (144 accumulators) need both files and get no copies.
extern __shared__ __attribute__((aligned(16))) char ns_dyn_lds[];
template <int EPI>
__global__ __launch_bounds__(256, 2) void ns_gemm_128(NsGemm p) { ns_w4_body<EPI, 4>(p, (DLLM_LDS char*)ns_dyn_lds); }
template <int EPI>
__global__ __launch_bounds__(256, 2) void ns_gemm_64(NsGemm p) {
  __shared__ __attribute__((aligned(16))) char smem[W4<2>::LDS];
  ns_w4_body<EPI, 2>(p, (DLLM_LDS char*)smem);
}
template <int EPI>
__global__ __launch_bounds__(256, 1) void ns_gemm_192(NsGemm p) {
  __shared__ __attribute__((aligned(16))) char smem[W4<6>::LDS];
  ns_w4_body<EPI, 6>(p, (DLLM_LDS char*)smem);
}

// Slices of K for the Gram matrix of an m x n matrix (padded sizes): where its 64x64 tiles leave CUs empty and K is long, one
// block's 3 n / 64 steps (0.24 us each) are shared by up to 16, for a launch that adds them up (6 us).  By the matrix's own
// sizes, so that a batch gives the bits of the single matrix.  Orthogonalising 256 x 4096 to fp32: 268 ->
// 157 us, 512 x 8192: 521 -> 321, 512 x 2048: 214 -> 173
static int ns_slices(long m, long n) {
  const long t = m / 64, tiles = t * (t + 1) / 2, per = n / 64;
  int s = 1;
  while (s < 16 && tiles * (2 * s) <= 256 && per >= 8 * (2 * s)) s *= 2;
  return s > 1 && 3.f * (float)per * 0.24f * (1.f - 1.f / (float)s) > 6.f ? s : 1;
}

template <int EPI>
static hipError_t ns_launch(NsGemm p, int B, hipStream_t s) {
  if (EPI == NS_PLANES && p.ksplit > 1) {
    const long grid = (long)B * ns_tiles(p, 64);
    if (grid > 0x7fffffffL) return hipErrorInvalidValue;
    hipLaunchKernelGGL((ns_gemm_64<NS_PLANES>), dim3((unsigned)grid, p.ksplit), dim3(256), 0, s, p);
    hipLaunchKernelGGL((ns_join<NS_PLANES>), dim3((unsigned)grid), dim3(256), 0, s, p);
    return hipGetLastError();
  }
  p.ksplit = 1;
  // the tile that needs the least time for whole rounds of CUs: microseconds of a 64-deep K step on one CU (measured on full
  // rounds: 128 x 128 is bound by LDS, 256 x 256 by the matrix units' power, busy 80 to 85 % of the cycles at 1.7 GHz, 192 x 192
  // half by it, 50 to 54 % at 2.0), and of a round's beginning and end
  const long cus = cu_count();
  const float steps = 3.f * (float)(p.K >> 6);
  auto time = [&](int ts, long per_cu, float step) {
    return (float)(((long)B * ns_tiles(p, ts) + cus * per_cu - 1) / (cus * per_cu)) * (steps * step + 5.f);
  };
  const bool whole = p.M % 256 == 0 && p.N % 256 == 0;
  const float t[4] = {time(64, 2, 0.24f), time(128, 1, 0.40f), time(192, 1, 0.85f), whole ? time(256, 1, 1.5f) : 1e30f};
  int best = 0;
  for (int i = 1; i < 4; ++i)
    if (t[i] < t[best]) best = i;
  const long grid = (long)B * ns_tiles(p, 64 * (best + 1));
  if (grid > 0x7fffffffL) return hipErrorInvalidValue;
  const dim3 g((unsigned)grid);
  if (best == 3) hipLaunchKernelGGL((ns_gemm_256<EPI>), g, dim3(512), 0, s, p);
  else if (best == 2) hipLaunchKernelGGL((ns_gemm_192<EPI>), g, dim3(256), 0, s, p);
  else if (best == 0) hipLaunchKernelGGL((ns_gemm_64<EPI>), g, dim3(256), 0, s, p);
  else {
    const hipError_t e = lds_opt_in((const void*)ns_gemm_128<EPI>, W4<4>::LDS);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((ns_gemm_128<EPI>), g, dim3(256), W4<4>::LDS, s, p);
  }
  return hipGetLastError();
}

static long pad128(long n) { return (n + 127) / 128 * 128; }

// workspace: partial sums, X and X^T planes (a second X^T when X is rewritten), six m x m plane pairs
struct NsSpace {
  long mp, np;              // sizes padded to 128
  long px, ps;              // elements of an X (or X^T) and of an m x m plane
  double* part;
  f16 *X, *XT, *XT2, *S[6];
  int slices;               // of the Gram matrix's K, and their sums
  float* sums;
  size_t bytes;
};
static NsSpace ns_space(char* base, int B, int R, int C, bool again) {
  NsSpace w;
  w.mp = pad128(min(R, C));
  w.np = pad128(max(R, C));
  w.px = w.mp * w.np;
  w.ps = w.mp * w.mp;
  size_t o = 0;
  auto take = [&](size_t n) {
    char* p = base + o;
    o += (n + 255) / 256 * 256;
    return p;
  };
  w.part = (double*)take((size_t)B * NS_PARTS * 8);
  w.X = (f16*)take((size_t)B * w.px * 4);
  w.XT = (f16*)take((size_t)B * w.px * 4);
  w.XT2 = again ? (f16*)take((size_t)B * w.px * 4) : nullptr;
  for (int i = 0; i < 6; ++i) w.S[i] = (f16*)take((size_t)B * w.ps * 4);
  w.slices = ns_slices(w.mp, w.np);
  const long t = w.mp / 64;
  w.sums = w.slices > 1 ? (float*)take((size_t)B * w.slices * (t * (t + 1) / 2) * 4096 * 4) : nullptr;
  w.bytes = o;
  return w;
}

#define NS_TRY(e)                                 \
  do {                                            \
    const hipError_t err_ = (e);                  \
    if (err_ != hipSuccess) return (int)err_;     \
  } while (0)

// ----------------------------------------------------------------------------------------------
// shorter side m <= 128: one launch per step
//
// A and P (128 x 128, padded with zeros) fit a block, so every block computes P for itself and applies it to its own columns
// of X, then leaves its part of the next A, the fp32 Gram matrix of the columns it just wrote; the next launch adds the
// parts up in their order.  Launches and their latency bound it: 300 x 101, five steps, 17 launches of the kernels above
// take 87 us, these 7 take 70; 16 x 16 87 and 48.
//
// X lives in operand order, "fragments": chunk (nt, kk) of a plane is 64 lanes x 8 values, lane (g, i) = (lane / 16,
// lane % 16) holding column 16 nt + i, rows 32 kk + 4 g + (0 .. 3) and 32 kk + 16 + 4 g + (0 .. 3).  That is what a lane has
// of two neighbouring results of the matrix instruction, so results become operands without leaving their lane; the order
// of rows inside a chunk is the same in both operands of every product, and the sum does not see it.
// Wave (rw, cw) owns rows 32 rw .. 32 rw + 31 and columns 32 cw .. 32 cw + 31 of A and P, 16 cw .. 16 cw + 15 of a slice.
// ----------------------------------------------------------------------------------------------
constexpr int NS_SMALL = 128;
constexpr int SM_SLICE = 64;          // columns of X at a time
constexpr int SM_BLOCKS = 256;        // blocks (parts of A) per matrix, at most
constexpr int SM_DIRECT = 8;          // parts that a step adds up by itself; more are added by a launch of their own
constexpr int SM_TLD = NS_SMALL + 4;  // LDS row of a slice in fp32
constexpr int SM_PART = NS_SMALL * NS_SMALL;

struct NsSmall {
  MuonIn in;
  const double* part;
  float eps;
  f16* X; long px;                    // fragment planes; px: elements of a plane; matrices 2 px apart
  const float* gin; int parts;        // parts of A to add, [matrix][parts][SM_PART], as the waves hold them
  float* gout;                        // [matrix][gridDim.x][SM_PART]
  int m, n, slices, tall;
};

struct SmFrag { f16x8_t h, l; };
__device__ __forceinline__ SmFrag sm_frag(const f32x4_t& a, const f32x4_t& b, float s) {
  SmFrag f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    f16 hh, ll;
    split16((e < 4 ? a[e] : b[e - 4]) * s, hh, ll);
    f.h[e] = hh;
    f.l[e] = ll;
  }
  return f;
}
// One of the four plane products of rows of a (4 g + r) and rows of b (i): lo lo, lo hi, hi lo into d, hi hi into c.  lo lo
// too: in a sum of few terms its 2^-22 does not average out, and five steps on one number end at 4.4e-7 (median) without it,
// 3.6e-7 with it and in fp32.  Callers run one product of four results before the next: one after the other on the same sum
// would wait for each (twice the time).
template <int S>
__device__ __forceinline__ void sm_mma(f32x4_t& c, f32x4_t& d, const SmFrag& a, const SmFrag& b) {
  f32x4_t& s = S == 3 ? c : d;
  s = __builtin_amdgcn_mfma_f32_16x16x32_f16(S & 2 ? a.h : a.l, S & 1 ? b.h : b.l, s, 0, 0, 0);
}
template <class F> __device__ __forceinline__ void sm_each(F f) {
  f(std::integral_constant<int, 0>{});
  f(std::integral_constant<int, 1>{});
  f(std::integral_constant<int, 2>{});
  f(std::integral_constant<int, 3>{});
}
__device__ __forceinline__ void sm_put(f16x8_t* base, int chunks, int c, int lane, const SmFrag& f) {
  base[c * 64 + lane] = f.h;
  base[(chunks + c) * 64 + lane] = f.l;
}
__device__ __forceinline__ SmFrag sm_get(const f16x8_t* base, int chunks, int c, int lane) {
  return SmFrag{base[c * 64 + lane], base[(chunks + c) * 64 + lane]};
}
// this wave's part of the Gram matrix of a slice whose fragments are in LDS, chunk nk * 8 + mt
__device__ __forceinline__ void sm_gram(const f16x8_t* gf, int rw, int cw, int lane, f32x4_t (&c)[2][2], f32x4_t (&d)[2][2]) {
#pragma unroll
  for (int nk = 0; nk < 2; ++nk) {
    const SmFrag a[2] = {sm_get(gf, 16, nk * 8 + 2 * rw, lane), sm_get(gf, 16, nk * 8 + 2 * rw + 1, lane)};
    const SmFrag b[2] = {sm_get(gf, 16, nk * 8 + 2 * cw, lane), sm_get(gf, 16, nk * 8 + 2 * cw + 1, lane)};
    sm_each([&](auto s) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sm_mma<s.value>(c[i >> 1][i & 1], d[i >> 1][i & 1], b[i & 1], a[i >> 1]);
    });
  }
}
__device__ __forceinline__ void sm_part_out(const NsSmall& p, int rw, int cw, int lane, const f32x4_t (&c)[2][2], const f32x4_t (&d)[2][2]) {
  f32x4_t* o = (f32x4_t*)(p.gout + ((long)blockIdx.y * gridDim.x + blockIdx.x) * SM_PART);
#pragma unroll
  for (int i = 0; i < 4; ++i) o[((2 * rw + (i >> 1)) * 8 + 2 * cw + (i & 1)) * 64 + lane] = c[i >> 1][i & 1] + d[i >> 1][i & 1];
}
__device__ __forceinline__ void sm_clear(f32x4_t (&c)[2][2]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) (&c[0][0])[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
}

// X_0 in fragments and its parts of A.  grid (blocks, matrices)
template <int KIND>
__global__ __launch_bounds__(1024) void ns_small_first(NsSmall p) {
  __shared__ __attribute__((aligned(16))) float tile[SM_SLICE * SM_TLD];
  __shared__ __attribute__((aligned(16))) f16x8_t gf[2 * 16 * 64];
  __shared__ double red[4];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, rw = w & 3, cw = w >> 2, i15 = lane & 15, g = lane >> 4, z = blockIdx.y;
  if (w < 4) {
    double s = p.part[(long)z * NS_PARTS + t];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) s += __shfl_down(s, d);
    if (lane == 0) red[w] = s;
  }
  __syncthreads();
  const double norm = sqrt((red[0] + red[1]) + (red[2] + red[3]));
  const float inv = (float)((double)(1 << SX) / (norm + (double)p.eps));
  f32x4_t c[2][2], d[2][2];
  sm_clear(c);
  sm_clear(d);
  for (int sl = blockIdx.x; sl < p.slices; sl += gridDim.x) {
    const int n0 = sl * SM_SLICE;
#pragma unroll
    for (int k = 0; k < SM_SLICE * NS_SMALL / 1024; ++k) {        // neighbouring threads along U's rows
      const int j = t + 1024 * k, n = p.tall ? j >> 7 : j & 63, m = p.tall ? j & 127 : j >> 6;
      float v = 0.f;
      if (m < p.m && n0 + n < p.n) {
        const int r = p.tall ? n0 + n : m, col = p.tall ? m : n0 + n;
        v = muon_u<KIND>(p.in, muon_row(p.in.il, p.in.B, p.in.R, p.in.C, z, r) + col) * inv;
      }
      tile[n * SM_TLD + m] = v;
    }
    __syncthreads();
    f16x8_t* x = (f16x8_t*)(p.X + (long)z * 2 * p.px);
    const float* q = tile + (16 * cw + i15) * SM_TLD + 32 * rw + 4 * g;
    sm_put(x, (int)(p.px >> 9), sl * 16 + cw * 4 + rw, lane, sm_frag(*(const f32x4_t*)q, *(const f32x4_t*)(q + 16), 1.f));
    f32x4_t a, b;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      a[r] = tile[(32 * (w >> 3) + 4 * g + r) * SM_TLD + 16 * (w & 7) + i15];
      b[r] = tile[(32 * (w >> 3) + 16 + 4 * g + r) * SM_TLD + 16 * (w & 7) + i15];
    }
    sm_put(gf, 16, w, lane, sm_frag(a, b, 1.f));
    __syncthreads();
    sm_gram(gf, rw, cw, lane, c, d);
    __syncthreads();
  }
  sm_part_out(p, rw, cw, lane, c, d);
}

// parts of A added up in order: every fourth one per wave, then the four waves.  grid (64 results, matrices)
__global__ __launch_bounds__(256) void ns_small_sum(const float* in, int parts, float* out) {
  __shared__ f32x4_t red[4][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const f32x4_t* q = (const f32x4_t*)(in + (long)blockIdx.y * parts * SM_PART) + blockIdx.x * 64 + lane;
  f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int k = w; k < parts; k += 4) s += q[(long)k * (SM_PART / 4)];
  red[w][lane] = s;
  __syncthreads();
  if (w == 0)
    ((f32x4_t*)(out + (long)blockIdx.y * SM_PART))[blockIdx.x * 64 + lane] = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
}

// one step.  EPI NS_PLANES: X <- P X in place, and its parts of the next A; NS_OUT / NS_STEP: the result.  Sixteen waves of
// little code: every instruction is fetched once per launch, at about 0.7 us a kilobyte, and four waves with four times the
// code each took 14 to 18 us a launch (these: 6 for 16 x 16, 12 for 300 x 101, of which LDS reads and matrix instructions are 7)
template <int EPI>
__global__ __launch_bounds__(1024) void ns_small_step(NsSmall p, NsGemm fin) {
  __shared__ __attribute__((aligned(16))) f16x8_t af[2 * 32 * 64];   // A's fragments, then P's: chunk kk * 8 + mt
  __shared__ __attribute__((aligned(16))) f16x8_t xf[2 * 16 * 64];   // the slice of X: chunk nt * 4 + kk
  __shared__ __attribute__((aligned(16))) f16x8_t gf[SM_SLICE * SM_TLD / 4];   // its new rows for A, or the result in fp32
  static_assert(SM_SLICE * SM_TLD / 4 >= 2 * 16 * 64, "both fit");
  const int t = threadIdx.x, lane = t & 63, i15 = lane & 15, g = lane >> 4, z = blockIdx.y;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6), rw = w & 3, cw = w >> 2;
  const int chunks = (int)(p.px >> 9);
  f16x8_t* x = (f16x8_t*)(p.X + (long)z * 2 * p.px);
  SmFrag xr = sm_get(x, chunks, blockIdx.x * 16 + w, lane);      // a sixteenth of the slice on its way to LDS
  f32x4_t a[2][2], c[2][2], d[2][2];
  sm_clear(a);
  const f32x4_t* q = (const f32x4_t*)(p.gin + (long)z * p.parts * SM_PART) + (2 * rw * 8 + 2 * cw) * 64 + lane;
  for (int k = 0; k < p.parts; k += 4) {                         // four parts on their way at a time
    f32x4_t v[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[j][i] = q[(long)min(k + j, p.parts - 1) * (SM_PART / 4) + ((i >> 1) * 8 + (i & 1)) * 64];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (k + j < p.parts)
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i >> 1][i & 1] += v[j][i];
  }
  const int kks = (p.m + 31) >> 5;                               // what lies behind row m is zero
  constexpr float SC = 1.f / (float)(1L << (2 * SX - SA));
  // one A for both terms of P: b A + c A^2 changes by (b + 2 c) of A's rounding near A = I, by 2 c if the terms' A differ
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const SmFrag f = sm_frag(a[i][0], a[i][1], SC);
    sm_put(af, 32, cw * 8 + 2 * rw + i, lane, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) a[i][e >> 2][e & 3] = (float)f.h[e] + (float)f.l[e];
  }
  sm_clear(c);
  sm_clear(d);
  __syncthreads();
#pragma unroll 1
  for (int kk = 0; kk < kks; ++kk) {
    const SmFrag f[2] = {sm_get(af, 32, kk * 8 + 2 * rw, lane), sm_get(af, 32, kk * 8 + 2 * rw + 1, lane)};
    const SmFrag b[2] = {sm_get(af, 32, kk * 8 + 2 * cw, lane), sm_get(af, 32, kk * 8 + 2 * cw + 1, lane)};
    sm_each([&](auto s) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sm_mma<s.value>(c[i >> 1][i & 1], d[i >> 1][i & 1], b[i & 1], f[i >> 1]);
    });
  }
  __syncthreads();                                               // A is read: each wave puts its part of P in its place
  constexpr float PC = NS_C / (float)(1L << (2 * SA - SP)), PB = NS_B / (float)(1L << (SA - SP)), PA = NS_A * (float)(1L << SP);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        c[i][j][r] = (c[i][j][r] + d[i][j][r]) * PC + PB * a[i][j][r] + (2 * rw + i == 2 * cw + j && 4 * g + r == i15 ? PA : 0.f);
    sm_put(af, 32, cw * 8 + 2 * rw + i, lane, sm_frag(c[i][0], c[i][1], 1.f));
  }
  constexpr float XC = 1.f / (float)(1L << SP);
  sm_clear(c);
  sm_clear(d);
  for (int sl = blockIdx.x; sl < p.slices; sl += gridDim.x) {
    sm_put(xf, 16, w, lane, xr);
    if (sl + gridDim.x < p.slices) xr = sm_get(x, chunks, (sl + gridDim.x) * 16 + w, lane);
    __syncthreads();
    // 32 rows by 16 columns of P X: u with row 4 g + r and column i per lane (X's operand order), y with row i and column
    // 4 g + r (the Gram matrix's); [small products][16 rows]
    f32x4_t u[2][2], y[2][2];
    sm_clear(u);
    sm_clear(y);
#pragma unroll 1
    for (int kk = 0; kk < kks; ++kk) {
      const SmFrag f[2] = {sm_get(af, 32, kk * 8 + 2 * rw, lane), sm_get(af, 32, kk * 8 + 2 * rw + 1, lane)};
      const SmFrag b = sm_get(xf, 16, cw * 4 + kk, lane);
      sm_each([&](auto s) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          sm_mma<s.value>(u[0][i], u[1][i], f[i], b);
          if constexpr (EPI == NS_PLANES) sm_mma<s.value>(y[0][i], y[1][i], b, f[i]);
        }
      });
    }
    if constexpr (EPI == NS_PLANES) {
      sm_put(x, chunks, sl * 16 + cw * 4 + rw, lane, sm_frag(u[0][0] + u[1][0], u[0][1] + u[1][1], XC));
      const SmFrag f = sm_frag(y[0][0] + y[1][0], y[0][1] + y[1][1], XC);   // columns 16 cw ..: half of chunk cw / 2
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f16x4_t* o = (f16x4_t*)(gf + ((cw >> 1) * 8 + 2 * rw + i) * 64 + lane) + (cw & 1);
        *o = f16x4_t{f.h[4 * i], f.h[4 * i + 1], f.h[4 * i + 2], f.h[4 * i + 3]};
        o[16 * 64 * 2] = f16x4_t{f.l[4 * i], f.l[4 * i + 1], f.l[4 * i + 2], f.l[4 * i + 3]};
      }
      __syncthreads();
      sm_gram(gf, rw, cw, lane, c, d);
    } else {
      float* tile = (float*)gf;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        *(f32x4_t*)(tile + (16 * cw + i15) * SM_TLD + 32 * rw + 16 * i + 4 * g) = u[0][i] + u[1][i];
      __syncthreads();
      const int n = p.tall ? t >> 4 : 8 * (t & 7), m = p.tall ? 8 * (t & 15) : t >> 3;   // 8 columns of one row of the result
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = p.tall ? tile[n * SM_TLD + m + e] : tile[(n + e) * SM_TLD + m];
      const int n0 = sl * SM_SLICE;
      ns_result8<EPI>(fin, z, p.tall ? n0 + n : m, p.tall ? m : n0 + n, v);
    }
    __syncthreads();
  }
  if constexpr (EPI == NS_PLANES) sm_part_out(p, rw, cw, lane, c, d);
}

struct SmSpace {
  int slices, blocks;
  long px;
  double* part;
  f16* X;
  float *g[2], *sum;
  size_t bytes;
};
static SmSpace sm_space(char* base, int B, int R, int C) {
  SmSpace w;
  w.slices = (max(R, C) + SM_SLICE - 1) / SM_SLICE;
  w.blocks = min(w.slices, SM_BLOCKS);
  w.px = (long)w.slices * SM_SLICE * NS_SMALL;
  size_t o = 0;
  auto take = [&](size_t n) {
    char* p = base + o;
    o += (n + 255) / 256 * 256;
    return p;
  };
  w.part = (double*)take((size_t)B * NS_PARTS * 8);
  w.X = (f16*)take((size_t)B * w.px * 4);
  for (int i = 0; i < 2; ++i) w.g[i] = (float*)take((size_t)B * w.blocks * SM_PART * 4);
  w.sum = (float*)take((size_t)B * SM_PART * 4);
  w.bytes = o;
  return w;
}

template <int KIND, int LAST>
static int ns_small_run(const MuonIn& in, NsGemm fin, int B, int steps, float eps, char* ws, hipStream_t s) {
  const SmSpace w = sm_space(ws, B, in.R, in.C);
  NsSmall p{in, w.part, eps, w.X, w.px, nullptr, 0, w.g[0], min(in.R, in.C), max(in.R, in.C), w.slices, in.R > in.C};
  const dim3 grid(w.blocks, B);
  hipLaunchKernelGGL((muon_sumsq_kernel<KIND>), dim3(NS_PARTS, B), dim3(1024), 0, s, in, w.part);
  NS_TRY(hipGetLastError());
  hipLaunchKernelGGL((ns_small_first<KIND>), grid, dim3(1024), 0, s, p);
  NS_TRY(hipGetLastError());
  fin.R = in.R; fin.Cc = in.C; fin.il = in.il; fin.nb = in.B;
  fin.cs = 1.f / (float)(1L << (SP + SX));
  for (int k = 0; k < steps; ++k) {
    p.gin = w.g[k & 1];
    p.gout = w.g[~k & 1];
    p.parts = w.blocks;
    if (w.blocks > SM_DIRECT) {
      hipLaunchKernelGGL(ns_small_sum, dim3(64, B), dim3(256), 0, s, p.gin, p.parts, w.sum);
      NS_TRY(hipGetLastError());
      p.gin = w.sum;
      p.parts = 1;
    }
    if (k + 1 < steps) hipLaunchKernelGGL((ns_small_step<NS_PLANES>), grid, dim3(1024), 0, s, p, fin);
    else hipLaunchKernelGGL((ns_small_step<LAST>), grid, dim3(1024), 0, s, p, fin);
    NS_TRY(hipGetLastError());
  }
  return 0;
}

// the whole iteration; `fin` carries the last product's outputs
template <int KIND, int LAST>
static int ns_run(const MuonIn& in, NsGemm fin, int B, int steps, int seg, float eps, char* ws, hipStream_t s) {
  if (min(in.R, in.C) <= NS_SMALL) return ns_small_run<KIND, LAST>(in, fin, B, steps, eps, ws, s);
  const bool tall = in.R > in.C;
  // near-square matrices: single steps cost no more (7.5 n / m + 2.5 against 3 n / m + 7 products) and are more exact
  if (5L * max(in.R, in.C) <= 7L * min(in.R, in.C)) seg = 1;
  NsSpace w = ns_space(ws, B, in.R, in.C, steps > seg);
  const int mp = (int)w.mp, np = (int)w.np;
  const int Rp = tall ? np : mp, Cp = tall ? mp : np;
  hipLaunchKernelGGL((muon_sumsq_kernel<KIND>), dim3(NS_PARTS, B), dim3(1024), 0, s, in, w.part);
  NS_TRY(hipGetLastError());
  hipLaunchKernelGGL((ns_split_kernel<KIND>), dim3(Cp / 64, Rp / 64, B), dim3(256), 0, s, in, w.part, eps,
                     tall ? w.XT : w.X, tall ? w.X : w.XT, Rp, Cp);
  NS_TRY(hipGetLastError());

  auto square = [&](const f16* a, const f16* b, f16* out, float cs) {   // [mp, mp] from two [mp, mp]
    NsGemm p = {};
    p.A = a; p.lda = mp; p.pa = w.ps; p.ba = 2 * w.ps;
    p.B = b; p.ldb = mp; p.pb = w.ps; p.bb = 2 * w.ps;
    p.M = mp; p.N = mp; p.K = mp; p.cs = cs;
    p.out = out; p.ldo = mp; p.po = w.ps; p.bo = 2 * w.ps;
    p.sym = 1;
    return p;
  };
  auto e2 = [](int e) { return e >= 0 ? (float)(1L << e) : 1.f / (float)(1L << -e); };

  int left = steps;
  f16 *A = w.S[0], *A2 = w.S[1], *P = w.S[2], *T = w.S[3], *Q = w.S[4], *Q2 = w.S[5];
  f16 *XT = w.XT, *XTn = w.XT2;
  while (left > 0) {
    const int n = left > seg ? seg : left;
    left -= n;
    NsGemm gr = square(w.X, w.X, A, e2(SA - 2 * SX));
    gr.lda = gr.ldb = np; gr.pa = gr.pb = w.px; gr.ba = gr.bb = 2 * w.px; gr.K = np;
    gr.ksplit = w.slices; gr.part = w.sums;
    NS_TRY(ns_launch<NS_PLANES>(gr, B, s));
    int sq = SP;
    for (int i = 0; i < n; ++i) {
      f16* Pd = i == 0 ? Q : P;   // the first P is Q
      NsGemm po = square(A, A, Pd, NS_C * e2(SP - 2 * SA));
      po.aux = A; po.cb = NS_B * e2(SP - SA); po.ca = NS_A * e2(SP);
      NS_TRY(ns_launch<NS_POLY>(po, B, s));
      if (i + 1 < n) {
        NS_TRY(ns_launch<NS_PLANES>(square(Pd, A, T, e2(SA - SP - SA)), B, s));    // P A
        NS_TRY(ns_launch<NS_PLANES>(square(T, Pd, A2, e2(SA - SA - SP)), B, s));   // (P A) P
        f16* x = A; A = A2; A2 = x;
      }
      if (i > 0) {
        NS_TRY(ns_launch<NS_PLANES>(square(P, Q, Q2, e2(SQ - SP - sq)), B, s));
        f16* x = Q; Q = Q2; Q2 = x;
        sq = SQ;
      }
    }
    NsGemm ap = {};
    const f16 *qa = Q, *xa = XT;
    if (left > 0) {   // X <- Q X and its transpose
      ap.A = qa; ap.lda = mp; ap.pa = w.ps; ap.ba = 2 * w.ps;
      ap.B = xa; ap.ldb = mp; ap.pb = w.px; ap.bb = 2 * w.px;
      ap.M = mp; ap.N = np; ap.K = mp; ap.cs = e2(-sq);
      ap.out = w.X; ap.ldo = np; ap.po = w.px; ap.bo = 2 * w.px;
      ap.outT = XTn; ap.ldt = mp; ap.pt = w.px; ap.bt = 2 * w.px;
      NS_TRY(ns_launch<NS_PLANES_T>(ap, B, s));
      f16* x = XT; XT = XTn; XTn = x;
    } else {          // the result, in U's own orientation
      ap = fin;
      const f16 *a = tall ? xa : qa, *b = tall ? qa : xa;
      ap.A = a; ap.lda = mp; ap.pa = tall ? w.px : w.ps; ap.ba = 2 * ap.pa;
      ap.B = b; ap.ldb = mp; ap.pb = tall ? w.ps : w.px; ap.bb = 2 * ap.pb;
      ap.M = Rp; ap.N = Cp; ap.K = mp; ap.cs = e2(-sq - SX);
      ap.R = in.R; ap.Cc = in.C; ap.il = in.il; ap.nb = in.B;
      NS_TRY(ns_launch<LAST>(ap, B, s));
    }
  }
  return 0;
}

}  // namespace dllm

using namespace dllm;

extern "C" {

// bytes of workspace for B matrices [R, C]; 0 for sizes out of range
long dllm_muon_workspace(int B, int R, int C, int steps) {
  if (B <= 0 || B > 65535 || R <= 0 || C <= 0 || steps < 1 || steps > 20) return 0;
  if (pad128(min(R, C)) > 65536 || pad128(max(R, C)) > (1L << 21)) return 0;
  if (min(R, C) <= NS_SMALL) return (long)sm_space(nullptr, B, R, C).bytes;
  return (long)ns_space(nullptr, B, R, C, steps > 1).bytes;
}

// out [B][R][C] = the orthogonalised x
int dllm_orthogonalize(const void* x, int xdt, void* out, int odt, int B, int R, int C, int steps, float eps, void* ws,
                       long ws_bytes, void* stream) {
  const long need = dllm_muon_workspace(B, R, C, steps);
  if (need == 0 || ws == nullptr || ws_bytes < need || (uintptr_t)ws % 256) return -1;
  if ((xdt != DT_BF16 && xdt != DT_F32) || (odt != DT_BF16 && odt != DT_F32) || !x || !out) return -1;
  MuonIn in{x, xdt, nullptr, 0.f, 1.f, 0, R, C, 0, B};
  NsGemm fin = {};
  fin.C = out; fin.cdt = odt;
  return ns_run<NS_ORTH, NS_OUT>(in, fin, B, steps, odt == DT_F32 ? 1 : NS_SEGMENT, eps, (char*)ws, (hipStream_t)stream);
}

// momentum update, orthogonalisation and W <- decay W - rate O, on an fp32 master (w, optional bf16 copy) or a split one
// (lo, copy); gradient [B][R][C] bf16 / fp32, momentum fp32.  il > 0: the matrices' rows alternate in blocks of il
int dllm_muon_step(const void* g, int gdt, float* mom, float* w, void* copy, void* lo, int B, int R, int C, int steps,
                   float eps, float beta, int nesterov, float gscale, float decay, float rate, int il, void* ws,
                   long ws_bytes, void* stream) {
  if (il < 0 || (il > 0 && R % il)) return -1;
  const long need = dllm_muon_workspace(B, R, C, steps);
  if (need == 0 || ws == nullptr || ws_bytes < need || (uintptr_t)ws % 256) return -1;
  if ((gdt != DT_BF16 && gdt != DT_F32) || !g || !mom || (!w && !(lo && copy)) || (w && lo)) return -1;
  MuonIn in{g, gdt, mom, beta, gscale, nesterov, R, C, il, B};
  NsGemm fin = {};
  fin.w = w; fin.copy = (uint16_t*)copy; fin.lo = (int16_t*)lo; fin.decay = decay; fin.rate = rate;
  return ns_run<NS_MUON, NS_STEP>(in, fin, B, steps, NS_SEGMENT, eps, (char*)ws, (hipStream_t)stream);
}

}  // extern "C"
