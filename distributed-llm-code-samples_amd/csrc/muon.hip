// Newton-Schulz orthogonalisation of 2-D updates and the Muon optimizer step.
//
// X0 = U / (|U|_F + eps) with the shorter side m as rows (m <= n), then `steps` times
//     A = X X^T,   X <- P X,   P = a I + b A + c A^2,   (a, b, c) = (3.4445, -4.7750, 2.0315)
// which pulls every singular value of X towards 1 and keeps the singular vectors.  All P are polynomials of one symmetric
// matrix, so they commute and stay symmetric, and the next A is P A P: up to three steps run on the m x m side alone,
//     Q = P_k ... P_1,   A <- (P A) P
// and X is multiplied by Q once at the end of such a segment.  Segments cost less (for n = 4 m, counting symmetric products
// half: 19 products of m x m x m for 3 + 2 steps, 32.5 for single steps) and lose digits: a Gram matrix's small eigenvalues
// are squares of small singular values, and its rounding is amplified as they are (12 a step).  Against 64 bits, errors of
// gradient-like matrices: single steps 0.5 to 1.1e-6, as an fp32 iteration; 3 + 2 steps 1 to 4e-6; five steps on one Gram
// matrix 2e-5.  So a result handed out in fp32 runs single steps; a bf16 result (half a step 2e-3) and a weight update
// (which scales the result by the learning rate before adding it) run segments of three.
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

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;
constexpr int SX = 15, SA = 15, SP = 14, SQ = 10;   // plane scales 2^s of X, A (and P A), P, products of P
constexpr int NS_SEGMENT = 3;                        // steps on one Gram matrix where the result allows it
constexpr int NS_PARTS = 256;                        // partial sums of squares per matrix

__device__ __forceinline__ void split16(float v, f16& h, f16& l) {
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
};

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

// momentum update and the partial sums of u^2 (64-bit: gradients of any magnitude, and a sum that does not depend on how it
// is cut).  grid (NS_PARTS, B)
template <int KIND>
__global__ __launch_bounds__(256) void muon_sumsq_kernel(MuonIn p, double* part) {
  __shared__ double red[4];
  const long n = (long)p.R * p.C, base = (long)blockIdx.y * n;
  double s = 0.0;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    if constexpr (KIND == NS_MUON)
      p.mom[base + i] = fmaf(p.beta, p.mom[base + i], p.gscale * ld_g(p, base + i));
    const double u = (double)muon_u<KIND>(p, base + i);
    s += u * u;
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) s += __shfl_down(s, d);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[(long)blockIdx.y * NS_PARTS + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// X0 planes in both orientations: same [Rp][Cp] and transposed [Cp][Rp], zeros outside [R][C].  64x64 tiles, grid
// (Cp / 64, Rp / 64, B)
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
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
  for (int k = t; k < 4096; k += 256) {
    const int r = r0 + (k >> 6), c = c0 + (k & 63);
    float v = 0.f;
    if (r < p.R && c < p.C) v = muon_u<KIND>(p, ((long)blockIdx.z * p.R + r) * p.C + c) * inv;
    tile[k >> 6][k & 63] = v;
    f16 h, l;
    split16(v, h, l);
    so[(long)r * Cp + c] = h;
    so[plane + (long)r * Cp + c] = l;
  }
  __syncthreads();
  for (int k = t; k < 4096; k += 256) {
    f16 h, l;
    split16(tile[k & 63][k >> 6], h, l);
    const long o = (long)(c0 + (k >> 6)) * Rp + r0 + (k & 63);
    to[o] = h;
    to[plane + o] = l;
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
  float* w; uint16_t* copy; int16_t* lo; float decay, rate;   // NS_STEP: fp32 master (+ bf16 copy), or split (lo, copy)
};

template <int EPI>
__device__ __forceinline__ void ns_epi4(const NsGemm& p, int z, int m, int n, f32x4_t v) {
  if constexpr (EPI == NS_PLANES || EPI == NS_PLANES_T || EPI == NS_POLY) {
    f16x4_t h, l;
    const long o = (long)z * p.bo + (long)m * p.ldo + n;
    f32x4_t a4 = {0.f, 0.f, 0.f, 0.f};
    if constexpr (EPI == NS_POLY) {
      const f16x4_t ah = *(const f16x4_t*)(p.aux + o), al = *(const f16x4_t*)(p.aux + p.po + o);
#pragma unroll
      for (int r = 0; r < 4; ++r) a4[r] = p.cb * ((float)ah[r] + (float)al[r]) + (m == n + r ? p.ca : 0.f);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      f16 hh, ll;
      split16(EPI == NS_POLY ? fmaf(p.cs, v[r], a4[r]) : p.cs * v[r], hh, ll);
      h[r] = hh;
      l[r] = ll;
    }
    *(f16x4_t*)(p.out + o) = h;
    *(f16x4_t*)(p.out + p.po + o) = l;
    if constexpr (EPI == NS_PLANES_T) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const long q = (long)z * p.bt + (long)(n + r) * p.ldt + m;
        p.outT[q] = h[r];
        p.outT[p.pt + q] = l[r];
      }
    }
  } else {
    if (m >= p.R) return;
    const long o = ((long)z * p.R + m) * p.Cc + n;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
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
}

// 128x128 tile, 4 waves of 64x64; K steps of 64 (one 128-byte line per row) over the three plane pairs (hi, lo), (lo, hi),
// (hi, hi).  LDS rows of 128 B with XOR-swizzled 16-B chunks (conflict-free ds_read_b128), filled by LDS-DMA.
template <int EPI>
__global__ __launch_bounds__(256, 2) void ns_gemm_128(NsGemm p) {
  constexpr int TB = 128 * 128;
  __shared__ __attribute__((aligned(16))) char smem[4 * TB];
  DLLM_LDS char* lds = (DLLM_LDS char*)smem;
  const int t = threadIdx.x, lane = t & 63, z = blockIdx.y;
  const int wid = __builtin_amdgcn_readfirstlane(t >> 6);
  const int tiles_n = p.N >> 7;
  const int bid = xcd_remap(blockIdx.x, gridDim.x);
  const int m0 = (bid / tiles_n) * 128, n0 = (bid % tiles_n) * 128;
  const int i15 = lane & 15, g = lane >> 4, wr = wid >> 1, wc = wid & 1;
  const f16 *ap[4], *bp[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int q = i * 4 + wid, row = 8 * q + (lane >> 3), c = ((lane & 7) ^ ((row >> 1) & 7)) * 8;
    ap[i] = p.A + (long)z * p.ba + (long)(m0 + row) * p.lda + c;
    bp[i] = p.B + (long)z * p.bb + (long)(n0 + row) * p.ldb + c;
  }
  const int nk = p.K >> 6;
  // the small products first: the accumulator is rounded at its final size a third as often
  auto stage = [&](int seg, int kt, int buf) {
    DLLM_LDS char* d = lds + buf * 2 * TB;
    const long oa = (long)kt * 64 + (seg == 1 ? p.pa : 0), ob = (long)kt * 64 + (seg == 0 ? p.pb : 0);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      __builtin_amdgcn_global_load_lds((const DLLM_GLB void*)(ap[i] + oa), (DLLM_LDS void*)(d + (i * 4 + wid) * 1024), 16, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      __builtin_amdgcn_global_load_lds((const DLLM_GLB void*)(bp[i] + ob), (DLLM_LDS void*)(d + TB + (i * 4 + wid) * 1024), 16, 0, 0);
  };
  auto frag = [&](const DLLM_LDS char* tile, int row, int chunk) {
    return *(const DLLM_LDS f16x8_t*)(tile + row * 128 + ((chunk ^ ((row >> 1) & 7)) << 4));
  };
  f32x4_t acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[i][k] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  stage(0, 0, 0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  int seg = 0, kt = 0;
  for (int it = 0; it < 3 * nk; ++it) {
    if (++kt == nk) { kt = 0; ++seg; }
    if (it + 1 < 3 * nk) stage(seg, kt, (it + 1) & 1);
    const DLLM_LDS char* As = lds + (it & 1) * 2 * TB;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      f16x8_t fa[4], fb[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        fa[i] = frag(As, wr * 64 + i * 16 + i15, 4 * s + g);
        fb[i] = frag(As + TB, wc * 64 + i * 16 + i15, 4 * s + g);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[i][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fb[k], fa[i], acc[i][k], 0, 0, 0);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) ns_epi4<EPI>(p, z, m0 + wr * 64 + i * 16 + i15, n0 + wc * 64 + k * 16 + 4 * g, acc[i][k]);
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

template <int EPI>
__global__ __launch_bounds__(512, 2) void ns_gemm_256(NsGemm p) {
  __shared__ __attribute__((aligned(16))) char smem[N8_LDS];
  DLLM_LDS char* lds = (DLLM_LDS char*)smem;
  const int t = threadIdx.x, lane = t & 63, z = blockIdx.y;
  const int wid = __builtin_amdgcn_readfirstlane(t >> 6);
  const int tiles_m = p.M >> 8, tiles_n = p.N >> 8;
  const int bid = xcd_remap(blockIdx.x, gridDim.x);
  const int width = 4 * tiles_n, first = bid / width * 4, gsz = min(tiles_m - first, 4);
  const int m0 = (first + bid % width % gsz) * 256, n0 = (bid % width / gsz) * 256;
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

#pragma unroll
  for (int qm = 0; qm < 2; ++qm)
#pragma unroll
    for (int qn = 0; qn < 2; ++qn) {
      const int n = n0 + n8_col(wid, lane, qn);
      f16x4_t th[8], tl[8];   // transposed planes: column n + e, rows of the four mt
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        const int m = m0 + n8_row(wid, lane, qm, mt);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = acc[qm][qn][mt][e & 1][e >> 1];
        if constexpr (EPI == NS_PLANES || EPI == NS_PLANES_T || EPI == NS_POLY) {
          ns_value8<EPI>(p, z, m, n, v);
          f16x8_t h, l;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            f16 hh, ll;
            split16(v[e], hh, ll);
            h[e] = hh;
            l[e] = ll;
            if constexpr (EPI == NS_PLANES_T) { th[e][mt] = hh; tl[e][mt] = ll; }
          }
          const long o = (long)z * p.bo + (long)m * p.ldo + n;
          *(f16x8_t*)(p.out + o) = h;
          *(f16x8_t*)(p.out + p.po + o) = l;
        } else {
          ns_epi4<EPI>(p, z, m, n, f32x4_t{v[0], v[1], v[2], v[3]});
          ns_epi4<EPI>(p, z, m, n + 4, f32x4_t{v[4], v[5], v[6], v[7]});
        }
      }
      if constexpr (EPI == NS_PLANES_T) {
        const int m = m0 + n8_row(wid, lane, qm, 0);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const long q = (long)z * p.bt + (long)(n + e) * p.ldt + m;
          *(f16x4_t*)(p.outT + q) = th[e];
          *(f16x4_t*)(p.outT + p.pt + q) = tl[e];
        }
      }
    }
}

template <int EPI>
static hipError_t ns_launch(const NsGemm& p, int B, hipStream_t s) {
  if (p.M % 256 == 0 && p.N % 256 == 0)
    hipLaunchKernelGGL((ns_gemm_256<EPI>), dim3((p.M / 256) * (p.N / 256), B), dim3(512), 0, s, p);
  else
    hipLaunchKernelGGL((ns_gemm_128<EPI>), dim3((p.M / 128) * (p.N / 128), B), dim3(256), 0, s, p);
  return hipGetLastError();
}

static long pad128(long n) { return (n + 127) / 128 * 128; }

// workspace: partial sums, X and X^T planes (a second X^T when X is rewritten), six m x m plane pairs
struct NsSpace {
  long mp, np, big, sq;
  double* part;
  f16 *X, *XT, *XT2, *S[6];
  size_t bytes;
};
static NsSpace ns_space(char* base, int B, int R, int C, bool again) {
  NsSpace w;
  w.mp = pad128(min(R, C));
  w.np = pad128(max(R, C));
  w.big = 2 * w.mp * w.np;
  w.sq = 2 * w.mp * w.mp;
  size_t o = 0;
  auto take = [&](size_t n) {
    char* p = base + o;
    o += (n + 255) / 256 * 256;
    return p;
  };
  w.part = (double*)take((size_t)B * NS_PARTS * 8);
  w.X = (f16*)take((size_t)B * w.big * 2);
  w.XT = (f16*)take((size_t)B * w.big * 2);
  w.XT2 = again ? (f16*)take((size_t)B * w.big * 2) : nullptr;
  for (int i = 0; i < 6; ++i) w.S[i] = (f16*)take((size_t)B * w.sq * 2);
  w.bytes = o;
  return w;
}

#define NS_TRY(e)                                 \
  do {                                            \
    const hipError_t err_ = (e);                  \
    if (err_ != hipSuccess) return (int)err_;     \
  } while (0)

// the whole iteration; `fin` carries the last product's outputs
template <int KIND, int LAST>
static int ns_run(const MuonIn& in, NsGemm fin, int B, int steps, int seg, float eps, char* ws, hipStream_t s) {
  const bool tall = in.R > in.C;
  NsSpace w = ns_space(ws, B, in.R, in.C, steps > seg);
  const int mp = (int)w.mp, np = (int)w.np;
  const int Rp = tall ? np : mp, Cp = tall ? mp : np;
  hipLaunchKernelGGL((muon_sumsq_kernel<KIND>), dim3(NS_PARTS, B), dim3(256), 0, s, in, w.part);
  NS_TRY(hipGetLastError());
  hipLaunchKernelGGL((ns_split_kernel<KIND>), dim3(Cp / 64, Rp / 64, B), dim3(256), 0, s, in, w.part, eps,
                     tall ? w.XT : w.X, tall ? w.X : w.XT, Rp, Cp);
  NS_TRY(hipGetLastError());

  const long psq = w.sq / 2, pbig = w.big / 2;
  auto square = [&](const f16* a, const f16* b, f16* out, float cs) {   // [mp, mp] from two [mp, mp]
    NsGemm p = {};
    p.A = a; p.lda = mp; p.pa = psq; p.ba = w.sq;
    p.B = b; p.ldb = mp; p.pb = psq; p.bb = w.sq;
    p.M = mp; p.N = mp; p.K = mp; p.cs = cs;
    p.out = out; p.ldo = mp; p.po = psq; p.bo = w.sq;
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
    gr.lda = gr.ldb = np; gr.pa = gr.pb = pbig; gr.ba = gr.bb = w.big; gr.K = np;
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
      ap.A = qa; ap.lda = mp; ap.pa = psq; ap.ba = w.sq;
      ap.B = xa; ap.ldb = mp; ap.pb = pbig; ap.bb = w.big;
      ap.M = mp; ap.N = np; ap.K = mp; ap.cs = e2(-sq);
      ap.out = w.X; ap.ldo = np; ap.po = pbig; ap.bo = w.big;
      ap.outT = XTn; ap.ldt = mp; ap.pt = pbig; ap.bt = w.big;
      NS_TRY(ns_launch<NS_PLANES_T>(ap, B, s));
      f16* x = XT; XT = XTn; XTn = x;
    } else {          // the result, in U's own orientation
      ap = fin;
      const f16 *a = tall ? xa : qa, *b = tall ? qa : xa;
      ap.A = a; ap.lda = mp; ap.pa = tall ? pbig : psq; ap.ba = tall ? w.big : w.sq;
      ap.B = b; ap.ldb = mp; ap.pb = tall ? psq : pbig; ap.bb = tall ? w.sq : w.big;
      ap.M = Rp; ap.N = Cp; ap.K = mp; ap.cs = e2(-sq - SX);
      ap.R = in.R; ap.Cc = in.C;
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
  return (long)ns_space(nullptr, B, R, C, steps > 1).bytes;
}

// out [B][R][C] = the orthogonalised x
int dllm_orthogonalize(const void* x, int xdt, void* out, int odt, int B, int R, int C, int steps, float eps, void* ws,
                       long ws_bytes, void* stream) {
  const long need = dllm_muon_workspace(B, R, C, steps);
  if (need == 0 || ws == nullptr || ws_bytes < need || (uintptr_t)ws % 256) return -1;
  if ((xdt != DT_BF16 && xdt != DT_F32) || (odt != DT_BF16 && odt != DT_F32) || !x || !out) return -1;
  MuonIn in{x, xdt, nullptr, 0.f, 1.f, 0, R, C};
  NsGemm fin = {};
  fin.C = out; fin.cdt = odt;
  return ns_run<NS_ORTH, NS_OUT>(in, fin, B, steps, odt == DT_F32 ? 1 : NS_SEGMENT, eps, (char*)ws, (hipStream_t)stream);
}

// momentum update, orthogonalisation and W <- decay W - rate O, on an fp32 master (w, optional bf16 copy) or a split one
// (lo, copy); gradient [B][R][C] bf16 / fp32, momentum fp32
int dllm_muon_step(const void* g, int gdt, float* mom, float* w, void* copy, void* lo, int B, int R, int C, int steps,
                   float eps, float beta, int nesterov, float gscale, float decay, float rate, void* ws, long ws_bytes,
                   void* stream) {
  const long need = dllm_muon_workspace(B, R, C, steps);
  if (need == 0 || ws == nullptr || ws_bytes < need || (uintptr_t)ws % 256) return -1;
  if ((gdt != DT_BF16 && gdt != DT_F32) || !g || !mom || (!w && !(lo && copy)) || (w && lo)) return -1;
  MuonIn in{g, gdt, mom, beta, gscale, nesterov, R, C};
  NsGemm fin = {};
  fin.w = w; fin.copy = (uint16_t*)copy; fin.lo = (int16_t*)lo; fin.decay = decay; fin.rate = rate;
  return ns_run<NS_MUON, NS_STEP>(in, fin, B, steps, NS_SEGMENT, eps, (char*)ws, (hipStream_t)stream);
}

}  // extern "C"
