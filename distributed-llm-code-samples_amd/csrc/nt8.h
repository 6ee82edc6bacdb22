// 256x256-tile main loop for two K-contiguous operands of 128-byte K steps (block-scaled 8-bit: 128 k, fp16 planes: 64 k).
//
// 512 threads, 8 waves as 2 (M) x 4 (N).  LDS holds two K steps of both operands as half-tiles of 128 rows x 128 B
// (8 x 16 KiB).  One loop iteration is two K steps in 8 phases; in a phase every wave computes a 64x32 piece of one
// quadrant of the tile, the next half-tile is fetched by LDS-DMA, and the fragments of the next phase are read.  Waves 4-7
// run one barrier interval behind waves 0-3 (their SIMD partners), so a SIMD alternates one wave's matrix instructions with
// the other's LDS reads.  Reads a phase: 8 / 4 / 8 / 4 fragments-halves (every K step's B-half 0 one phase early).
//
//   phase   reads (buffer)   fetches                      waits (own LDS-DMA, before the barrier)
//   P0      A0 (even)        A1 of step 2i+1
//   P1      B1 (even)        A0 of step 2i+2
//   P2      A1 (even)        B0 of step 2i+2              vmcnt(8): B0 of step 2i+1 has landed
//   P3      B0 (odd)         B1 of step 2i+2              vmcnt(6): all of step 2i+1 up to its A1
//   P4..P7  the same with the buffers exchanged
//
// A half-tile is overwritten at least one phase after its last read (every phase waits for its own reads before its
// barrier).  Fetches past the last K step re-load it into slots that are not read again.  vmcnt counts every memory
// operation in flight, so loads that a trait adds (scales) make the waits stricter, never looser.
//
// LDS rows are permuted: slot 16 mt + i of a 64-row group of A holds row 4 i + mt, slot 16 nt + i of a 32-row group of B
// holds row 2 i + nt.  A lane (i = lane % 16, g = lane / 16) then ends with rows 4 i .. 4 i + 3 (mt) and columns 8 g .. 8 g
// + 7 (2 r + nt) of its wave's piece: 16-byte bf16 / fp16 stores along a row, 8-byte stores along a column whose 16 lanes
// write 128 consecutive bytes of the transposed matrix, and one 32-bit word holds the scales of a lane's four A rows.
#pragma once
#include <type_traits>

#include "common.h"

namespace dllm {

constexpr int N8_HT = 16384;               // half-tile bytes
constexpr int N8_LDS = 8 * N8_HT;

typedef __attribute__((ext_vector_type(4))) int n8_i32x4;

#define N8_BARRIER()               \
  do {                             \
    asm volatile("" ::: "memory"); \
    __builtin_amdgcn_s_barrier();  \
    asm volatile("" ::: "memory"); \
  } while (0)
#define N8_LDS_WAIT()                                   \
  do {                                                  \
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  \
    __builtin_amdgcn_sched_barrier(0);                  \
  } while (0)

// fragment reads in inline asm: the compiler cannot tell them from the LDS-DMA in flight and would drain it before each.
// Every phase waits (N8_LDS_WAIT) before anything uses what it read.
template <int OFF>
__device__ __forceinline__ void n8_read(n8_i32x4& d, uint32_t addr) {
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(d) : "v"(addr), "i"(OFF));
}
// 16 bytes a lane from `src` (uniform) + `off` (a lane's own, below 2^31) to LDS, in the buffer form: the address is made
// from the descriptor's base and the 32-bit offset by the load itself, with no vector instruction or register pair
__device__ __forceinline__ void n8_dma(const char* src, uint32_t off, DLLM_LDS char* dst) {
  __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)src, 0, 0x7fffffff, 0x00027000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (DLLM_LDS void*)dst, 16, (int)off, 0, 0, 0);
}

// CUs of the device (256 where there is none: plans are made on the host)
static inline int cu_count() {
  static const int n = [] {
    int dev = 0, v = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || v <= 0) v = 256;
    return v;
  }();
  return n;
}

// dynamic LDS beyond 64 KiB is allowed per kernel, once
static inline hipError_t lds_opt_in(const void* kernel, int bytes) {
  return hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

struct N8Frag { n8_i32x4 lo, hi; };        // 32 bytes of a row: 16-B chunks g and 4 + g of the K step

// byte offsets (within the operand, from the tile's first row) of the two LDS-DMA pieces a wave fetches of a half-tile.
// `left`: rows from the tile's first row to the operand's last; rows behind it re-load the last one
template <bool IS_A>
__device__ __forceinline__ void n8_offsets(long ld, int half, int left, int wid, int lane, uint32_t (&off)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int s = 8 * (wid + 8 * i) + (lane >> 3);   // LDS slot
    const int row = 128 * half + (IS_A ? (s & 64) + 4 * (s & 15) + ((s >> 4) & 3) : (s & 96) + 2 * (s & 15) + ((s >> 4) & 1));
    const int c = (lane & 7) ^ ((s >> 1) & 7);
    off[i] = (uint32_t)((long)min(row, left) * ld + c * 16);
  }
}

// row / first column (within the tile) of accumulator group (qm, qn, mt); r, nt: column 2 r + nt of the 8
__device__ __forceinline__ int n8_row(int wid, int lane, int qm, int mt) {
  return 128 * qm + (wid >> 2) * 64 + 4 * (lane & 15) + mt;
}
__device__ __forceinline__ int n8_col(int wid, int lane, int qn) { return 128 * qn + (wid & 3) * 32 + 8 * (lane >> 4); }

// The loop.  T (the trait) supplies the operands and the matrix instruction:
//   t.advance(a, b, it)    moves the K-step pointers from pair `it` to the next one (from the last: nowhere) and returns the
//                          bytes from that pair's first step to its second
//   t.load(odd, it)        issued once per K step, after the phase's wait: per-step extras for the step two on
//   t.mma<QM, QN, ODD>(acc, fa, fb)
// `a0`, `b0`: K step 0 of the tile, `step`: bytes to step 1.  nk2: pairs of K steps.
template <class T>
__device__ __forceinline__ void n8_loop(T& t, DLLM_LDS char* lds, const char* a0, const char* b0, int step,
                                        const uint32_t (&ao)[2][2], const uint32_t (&bo)[2][2], int nk2, int wid, int lane,
                                        f32x4_t (&acc)[2][2][4][2]) {
  const int wr = wid >> 2, wc = wid & 3, i15 = lane & 15, g = lane >> 4;
  auto stage_a = [&](int hh, const char* src, int buf) {
    DLLM_LDS char* d = lds + (hh * 2 + buf) * N8_HT;
    n8_dma(src, ao[hh][0], d + wid * 1024);
    n8_dma(src, ao[hh][1], d + (wid + 8) * 1024);
  };
  auto stage_b = [&](int hh, const char* src, int buf) {
    DLLM_LDS char* d = lds + (4 + hh * 2 + buf) * N8_HT;
    n8_dma(src, bo[hh][0], d + wid * 1024);
    n8_dma(src, bo[hh][1], d + (wid + 8) * 1024);
  };
  const uint32_t lb = (uint32_t)(uintptr_t)lds;
  const int f = (i15 >> 1) & 7;
  const uint32_t abase[2] = {lb + (wr * 64 + i15) * 128 + ((g ^ f) << 4), lb + (wr * 64 + i15) * 128 + (((4 + g) ^ f) << 4)};
  const uint32_t bbase[2] = {lb + 4 * N8_HT + (wc * 32 + i15) * 128 + ((g ^ f) << 4),
                             lb + 4 * N8_HT + (wc * 32 + i15) * 128 + (((4 + g) ^ f) << 4)};
  N8Frag fa[4], fb0[2], fb1[2];
  auto read_a = [&](auto hh, auto buf) {
    constexpr int SO = (hh.value * 2 + buf.value) * N8_HT;
    n8_read<SO>(fa[0].lo, abase[0]); n8_read<SO>(fa[0].hi, abase[1]);
    n8_read<SO + 2048>(fa[1].lo, abase[0]); n8_read<SO + 2048>(fa[1].hi, abase[1]);
    n8_read<SO + 4096>(fa[2].lo, abase[0]); n8_read<SO + 4096>(fa[2].hi, abase[1]);
    n8_read<SO + 6144>(fa[3].lo, abase[0]); n8_read<SO + 6144>(fa[3].hi, abase[1]);
  };
  auto read_b = [&](auto hh, auto buf, N8Frag (&fb)[2]) {
    constexpr int SO = (hh.value * 2 + buf.value) * N8_HT;
    n8_read<SO>(fb[0].lo, bbase[0]); n8_read<SO>(fb[0].hi, bbase[1]);
    n8_read<SO + 2048>(fb[1].lo, bbase[0]); n8_read<SO + 2048>(fb[1].hi, bbase[1]);
  };
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  auto mma = [&](auto qm, auto qn, N8Frag (&fb)[2], auto odd) {
    __builtin_amdgcn_s_setprio(1);
    t.template mma<qm.value, qn.value, odd.value>(acc[qm.value][qn.value], fa, fb);
    __builtin_amdgcn_s_setprio(0);
  };

  // K step 0 -> even buffer, step 1 -> odd buffer but its A1 (fetched in P0)
  stage_a(0, a0, 0); stage_b(0, b0, 0); stage_b(1, b0, 0); stage_a(1, a0, 0);
  stage_a(0, a0 + step, 1); stage_b(0, b0 + step, 1); stage_b(1, b0 + step, 1);
  const char *aodd = a0 + step, *an = a0, *bn = b0;   // an, bn: the pair after the current one
  asm volatile("s_waitcnt vmcnt(6)" ::: "memory");
  N8_BARRIER();
  read_b(I0{}, I0{}, fb0);
  N8_LDS_WAIT();
  if (wr == 1) N8_BARRIER();

  for (int it = 0; it < nk2; ++it) {
    step = t.advance(an, bn, it);
    // even buffer; its B0 is in fb0
    read_a(I0{}, I0{});
    stage_a(1, aodd, 1);                       // P0
    N8_LDS_WAIT();
    N8_BARRIER();
    mma(I0{}, I0{}, fb0, I0{});
    N8_BARRIER();
    read_b(I1{}, I0{}, fb1);
    stage_a(0, an, 0);                         // P1
    N8_LDS_WAIT();
    N8_BARRIER();
    mma(I0{}, I1{}, fb1, I0{});
    N8_BARRIER();
    read_a(I1{}, I0{});
    stage_b(0, bn, 0);                         // P2
    asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    N8_LDS_WAIT();
    N8_BARRIER();
    mma(I1{}, I1{}, fb1, I0{});
    N8_BARRIER();
    read_b(I0{}, I1{}, fb1);                   // odd buffer's B0
    stage_b(1, bn, 0);                         // P3
    asm volatile("s_waitcnt vmcnt(6)" ::: "memory");
    N8_LDS_WAIT();
    N8_BARRIER();
    mma(I1{}, I0{}, fb0, I0{});
    t.load(I0{}, it);                          // extras of step 2 it + 2
    N8_BARRIER();
    // odd buffer; its B0 is in fb1
    read_a(I0{}, I1{});
    stage_a(1, an, 0);                         // P4
    N8_LDS_WAIT();
    N8_BARRIER();
    mma(I0{}, I0{}, fb1, I1{});
    N8_BARRIER();
    read_b(I1{}, I1{}, fb0);
    stage_a(0, an + step, 1);               // P5
    N8_LDS_WAIT();
    N8_BARRIER();
    mma(I0{}, I1{}, fb0, I1{});
    N8_BARRIER();
    read_a(I1{}, I1{});
    stage_b(0, bn + step, 1);               // P6
    asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    N8_LDS_WAIT();
    N8_BARRIER();
    mma(I1{}, I1{}, fb0, I1{});
    N8_BARRIER();
    read_b(I0{}, I0{}, fb0);                   // the next pair's B0
    stage_b(1, bn + step, 1);               // P7
    asm volatile("s_waitcnt vmcnt(6)" ::: "memory");
    N8_LDS_WAIT();
    N8_BARRIER();
    mma(I1{}, I0{}, fb1, I1{});
    t.load(I1{}, it);                          // extras of step 2 it + 3
    N8_BARRIER();
    aodd = an + step;
  }
  if (wr == 0) N8_BARRIER();
  // the last fetches land before the block can release its LDS
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

}  // namespace dllm
