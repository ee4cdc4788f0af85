// 16-bit (bf16 / fp16) products on CTA pairs, with the feed-forward epilogues.
//
//   D[m][n] = sum_k A[m][k] B[n][k]      fp32 sums in tensor memory
//
// Either operand may lie in memory with its rows contiguous (K-major) or with
// its contraction axis outermost (MN-major): the forward product reads both
// K-major, the gradient of the input reads the weight MN-major, the gradient
// of the weight reads both operands MN-major.  The matrix descriptors express
// the difference; no operand is transposed in memory.
//
// One pair of CTAs (cta_group::2) computes a 256 x tn tile: each CTA stages
// its own 128 rows of A and tn/2 rows of B, and the pair's MMA reads both
// halves of B, so an operand byte fetched from L2 is used twice as often as by
// single CTAs.  Roles: warps 0 and 3 TMA producers (A and B: one thread that
// issued all copies took longer for a stage than the 512 cycles of its MMAs),
// warp 1 of the leader MMA issuer, the warps from 4 on epilogue.  The two 256-column accumulators in TMEM let the
// epilogue of one tile overlap the products of the next.
//
// Epilogues (all arithmetic in fp32, one rounding when a value is stored; h, dg
// and du are stored in 16 bits because the next product's operands are: 2^-8 of
// a value in bf16, 2^-11 in fp16, where h past 65,504 becomes an infinity):
//   kEpiLinear    y = act(D + bias) + residual; optionally z = D + bias is
//                 kept for the backward pass (groups of 32 in 16 or 8 bits)
//   kEpiGated     B holds gate rows [0, n) and up rows [n, 2n); the tile takes
//                 tn/2 of each, so a thread has both factors of
//                 h = act(min(g, L)) * clamp(u, -L, L) in its registers
//   kEpiGatedBwd  D = dh; reads the kept g and u and writes
//                 dg = dh u' act'(g') [g <= L], du = dh act(g') [|u| <= L]
//                 (and h where it has to be formed again)
#pragma once

#include "common.cuh"
#include "feed_forward_kernels.cuh"

namespace dsv4 {

enum F16DeviceErr : int {
  kErrF16WaitEmpty = 0x201,
  kErrF16WaitFull = 0x202,
  kErrF16WaitAccFull = 0x203,
  kErrF16WaitAccEmpty = 0x204,
};

enum F16Epi : int { kEpiLinear = 0, kEpiGated = 1, kEpiGatedBwd = 2 };

// Epilogue warps and their 2-KB shared slices.  The forward epilogues fit 96
// registers and one slice: 16 warps (2048 x 2048 -> 7168 with bias, gelu,
// residual and z kept: 60 us, 63 with 12, 67 with 8; gated 4096 x 1024 -> 2 x
// 2048 with a limit and z kept: 37, 38 and 39).  The gate's backward pass turns
// two matrices over in place and is best with few warps and all of their
// registers (4096 x 1024 -> 2048: 43 us, 46 with 12, 50 with 16).
template <int EPI>
struct F16Roles {
  static constexpr int kEpiWarps = EPI == kEpiGatedBwd ? 8 : 16;
  static constexpr int kSlices = EPI == kEpiGatedBwd ? 2 : 1;
  static constexpr int kThreads = 128 + 32 * kEpiWarps;
  static constexpr int kEpiBytes = kEpiWarps * kSlices * 2048;
};
constexpr int kF16ABytes = 128 * 128;          // 128 rows x 64 elements of A per stage
constexpr int kF16StageSlice = 2048;           // 32 x 32 16-bit values
constexpr int kF16MaxStages = 12;
constexpr int kF16SmemMax = 232448;
constexpr int kF16BarBytes = 256;
static_assert((2 * kF16MaxStages + 4) * 8 + 8 <= kF16BarBytes, "barrier area");

// A row-major matrix that the epilogue reads or writes by 16-byte pieces where
// its address and row stride allow it.
struct F16Mat {
  void* p;
  int64_t ld;  // elements
  int vec;     // 16-byte aligned base and rows
};

struct F16GemmParams {
  CUtensorMap map_a, map_b;
  int m, n, k;            // n: columns of D (kEpiGated: of h)
  int tn;                 // B rows of a pair tile (kEpiGated: gate and up together)
  int stages, b_stage;    // ring depth, bytes of B per stage and CTA
  int a_mn, b_mn;         // 1: the operand is MN-major
  int a_wide, b_wide;     // MN-major in whole 64s of rows: one copy per stage
  int tiles_m, tiles_n, group_m;
  int up_row;             // kEpiGated: B row of up row 0
  int act;
  float limit;            // infinity where there is none
  const void* bias;
  F16Mat residual, out;   // out: y, h (kEpiGatedBwd: h, or null)
  F16Mat d0, d1;          // kEpiGatedBwd: dg and du
  void* zq;               // kept z, or g and u: codes of zbits [m][halves * n32] ...
  int zbits;              // 0 (none), 8 or 16
  float* zs;              // ... and scales [halves * n32 / 32][m]
  int64_t n32;            // n rounded up to the group
};

// ---- tcgen05 / TMA forms of the pair ----
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int c0,
                                                 int c1, uint32_t cl_bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(cl_bar)
      : "memory");
}

__device__ __forceinline__ void tma_load_3d_pair_plain(uint32_t dst, const CUtensorMap* map, int c0,
                                                       int c1, int c2, uint32_t cl_bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(cl_bar)
      : "memory");
}

// One CTA's `rows` rows of an operand at row `row`, 64 of k from `kk`.
__device__ __forceinline__ void load_operand(uint32_t dst, const CUtensorMap* map, int mn, int wide,
                                             int rows, int row, int kk, uint32_t cl_bar) {
  if (!mn) {
    tma_load_2d_pair(dst, map, kk, row, cl_bar);
  } else if (wide) {
    tma_load_3d_pair_plain(dst, map, 0, kk, row >> 6, cl_bar);
  } else {
    for (int j = 0; j < rows; j += 64) tma_load_2d_pair(dst + j * 128, map, row + j, kk, cl_bar);
  }
}

__device__ __forceinline__ void mma_f16_ss_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                                uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Arrive on the barrier at this shared-memory offset in both CTAs of the pair
// once all pair MMAs issued so far by this thread complete.
__device__ __forceinline__ void mma_commit_both(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
      " [%0], %1;" ::"r"(bar),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}

// MN-major operand, 128-byte swizzle: 64 elements of the row axis side by side
// (128 B), contraction steps 128 B apart.  Groups of 8 contraction steps are
// 1024 B apart (SBO), groups of 64 rows one box apart (LBO).
__device__ __forceinline__ uint64_t smem_desc_sw128_mn(uint32_t box_bytes) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>(box_bytes >> 4) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}

// Place in a ring of `stages`: slot and parity of its current use, stepped
// without divisions (one thread walks it: its latency is the loop's).
struct RingCursor {
  int slot = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void step(int stages) {
    if (++slot == stages) slot = 0, parity ^= 1;
  }
};

// Descriptor of an operand at shared address 0; desc_addr() is added to it.
// In a cluster a shared address carries the CTA's rank above its 18 bits of
// offset: without the mask they would run into the LBO field.
__device__ __forceinline__ uint32_t desc_addr(uint32_t saddr) { return (saddr & 0x3FFFFu) >> 4; }

__device__ __forceinline__ uint64_t operand_desc(int mn, uint32_t box_bytes) {
  return mn ? smem_desc_sw128_mn(box_bytes) : smem_desc_sw128(0);
}

// One lane of a warp that runs together.  The issuing roles run as whole warps
// and elect the lane only where an instruction is issued: descriptors, slots
// and counters then live in uniform registers.  (As a branch of lane 0 an MMA
// cost its issuer 71 cycles and a stage of four 587, more than the 512 of the
// tensor cores.)
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(p));
  return p != 0;
}

// kind::f16, fp32 accumulator; A and B of the same type.
__device__ __forceinline__ uint32_t idesc_f16(bool bf16, uint32_t m, uint32_t n, uint32_t a_mn,
                                              uint32_t b_mn) {
  const uint32_t t = bf16 ? 1u : 0u;
  return (1u << 4) | (t << 7) | (t << 10) | (a_mn << 15) | (b_mn << 16) | ((n >> 3) << 17) |
         ((m >> 4) << 24);
}

// ---- 32 x 32 chunks of 16-bit matrices: global <-> registers of a row ----
// Where rows are 16-byte aligned (mat.vec) and the chunk is whole, lane l moves
// the 16-byte pieces of rows 8i + l/4, columns 8 (l & 3): four lanes cover a
// row's 64 bytes, so accesses are whole sectors.  Otherwise a lane moves its
// column, row by row: 64 contiguous bytes an access.  The shared slice turns
// either into one row per lane; its 16-byte units are XORed with bits of the
// row, which leaves both sides free of bank conflicts.
__device__ __forceinline__ uint32_t slice_off(int row, int piece) {
  return static_cast<uint32_t>(row * 64 + ((piece ^ ((row >> 1) & 3)) << 4));
}

__device__ __forceinline__ uint32_t slice_elem(int row, int col) {
  return slice_off(row, col >> 3) + 2 * (col & 7);
}

__device__ __forceinline__ bool chunk_whole(const F16Mat& mat, int col0, int cols) {
  return mat.vec && col0 + 32 <= cols;
}

__device__ __forceinline__ void whole_chunk_fetch(uint4 (&r)[4], const uint16_t* base, int64_t ld,
                                                  int lane, int row0, int rows) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 8 * i + (lane >> 2);
    r[i] = make_uint4(0, 0, 0, 0);
    if (row0 + row < rows) r[i] = *reinterpret_cast<const uint4*>(base + row * ld + 8 * (lane & 3));
  }
}

// In the second form register word i holds rows 2i and 2i + 1 of the column.
__device__ __forceinline__ void chunk_fetch(uint4 (&r)[4], const F16Mat& mat, int lane, int row0,
                                            int rows, int col0, int cols) {
  const uint16_t* base = static_cast<const uint16_t*>(mat.p) + row0 * mat.ld + col0;
  if (chunk_whole(mat, col0, cols)) {
    whole_chunk_fetch(r, base, mat.ld, lane, row0, rows);
  } else {
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      w[i] = 0;
      if (col0 + lane < cols) {
        if (row0 + 2 * i < rows) w[i] = base[2 * i * mat.ld + lane];
        if (row0 + 2 * i + 1 < rows) w[i] |= static_cast<uint32_t>(base[(2 * i + 1) * mat.ld + lane]) << 16;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }
}

__device__ __forceinline__ void whole_chunk_to_slice(uint32_t slice, int lane, const uint4 (&r)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    st_shared_v4(slice + slice_off(8 * i + (lane >> 2), lane & 3), r[i]);
}

__device__ __forceinline__ void chunk_to_rows(uint32_t slice, int lane, const uint4 (&r)[4],
                                              bool whole, uint32_t (&w)[16]) {
  if (whole) {
    whole_chunk_to_slice(slice, lane, r);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        st_shared_u16(slice + slice_elem(8 * i + 2 * j, lane), v[j]);
        st_shared_u16(slice + slice_elem(8 * i + 2 * j + 1, lane), v[j] >> 16);
      }
    }
  }
  __syncwarp();
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint4 v = ld_shared_v4(slice + slice_off(lane, c));
    w[4 * c] = v.x, w[4 * c + 1] = v.y, w[4 * c + 2] = v.z, w[4 * c + 3] = v.w;
  }
  __syncwarp();
}

// A lane's row in the slice, from piece `c` on.
template <int N>
__device__ __forceinline__ void row_to_slice(uint32_t slice, int lane, int c, const uint32_t (&w)[N]) {
#pragma unroll
  for (int i = 0; i < N / 4; ++i)
    st_shared_v4(slice + slice_off(lane, c + i),
                 make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]));
}

__device__ __forceinline__ void slice_store(uint32_t slice, int lane, const F16Mat& mat, int row0,
                                            int rows, int col0, int cols) {
  __syncwarp();
  uint16_t* base = static_cast<uint16_t*>(mat.p) + row0 * mat.ld + col0;
  if (chunk_whole(mat, col0, cols)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 8 * i + (lane >> 2);
      const uint4 v = ld_shared_v4(slice + slice_off(row, lane & 3));
      if (row0 + row < rows) *reinterpret_cast<uint4*>(base + row * mat.ld + 8 * (lane & 3)) = v;
    }
  } else if (col0 + lane < cols) {
#pragma unroll 8
    for (int row = 0; row < 32; ++row)
      if (row0 + row < rows)
        base[row * mat.ld + lane] = static_cast<uint16_t>(ld_shared_u16(slice + slice_elem(row, lane)));
  }
  __syncwarp();
}

__device__ __forceinline__ void chunk_store(uint32_t slice, int lane, const uint32_t (&w)[16],
                                            const F16Mat& mat, int row0, int rows, int col0,
                                            int cols) {
  row_to_slice(slice, lane, 0, w);
  slice_store(slice, lane, mat, row0, rows, col0, cols);
}

// 8-bit codes of a 32 x 32 chunk (rows of 32 bytes, always whole: the code
// rows are padded to the group).
__device__ __forceinline__ void codes_store(uint32_t slice, int lane, const uint32_t (&q)[8],
                                            int8_t* base, int64_t ld, int row0, int rows,
                                            int64_t col0) {
  st_shared_v4(slice + lane * 32 + (((lane >> 2) & 1) << 4), make_uint4(q[0], q[1], q[2], q[3]));
  st_shared_v4(slice + lane * 32 + ((((lane >> 2) & 1) ^ 1) << 4),
               make_uint4(q[4], q[5], q[6], q[7]));
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 16 * i + (lane >> 1), half = lane & 1;
    const uint4 v = ld_shared_v4(slice + r * 32 + ((half ^ ((r >> 2) & 1)) << 4));
    if (row0 + r < rows)
      *reinterpret_cast<uint4*>(base + (row0 + r) * ld + col0 + 16 * half) = v;
  }
  __syncwarp();
}

__device__ __forceinline__ void codes_fetch(uint4 (&v)[4], const int8_t* base, int64_t ld,
                                            int lane, int row0, int rows, int64_t col0) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 16 * i + (lane >> 1);
    v[i] = make_uint4(0, 0, 0, 0);
    if (row0 + r < rows)
      v[i] = *reinterpret_cast<const uint4*>(base + (row0 + r) * ld + col0 + 16 * (lane & 1));
  }
}

__device__ __forceinline__ void codes_to_rows(uint32_t slice, int lane, const uint4& v0, const uint4& v1,
                                              uint32_t (&q)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 16 * i + (lane >> 1);
    st_shared_v4(slice + r * 32 + (((lane & 1) ^ ((r >> 2) & 1)) << 4), i ? v1 : v0);
  }
  __syncwarp();
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const uint4 c = ld_shared_v4(slice + lane * 32 + ((half ^ ((lane >> 2) & 1)) << 4));
    q[4 * half] = c.x, q[4 * half + 1] = c.y, q[4 * half + 2] = c.z, q[4 * half + 3] = c.w;
  }
  __syncwarp();
}

// A warp's 32 rows of one kept group, columns `at`.. of code rows of `ld`.
template <bool BF16>
__device__ __forceinline__ void keep_rows(const F16GemmParams& p, uint32_t slice, int lane,
                                          const float (&v)[32], int64_t ld, int row0, int at) {
  float s;
  if (p.zbits == 8) {
    uint32_t q[8];
    s = keep_group8(v, q);
    codes_store(slice, lane, q, static_cast<int8_t*>(p.zq), ld, row0, p.m, at);
  } else {
    uint32_t q[16];
    s = keep_group16<BF16>(v, p.limit, p.act == kActRelu, q);
    chunk_store(slice, lane, q, F16Mat{p.zq, ld, 1}, row0, p.m, at, static_cast<int>(ld));
  }
  if (row0 + lane < p.m) p.zs[static_cast<int64_t>(at >> 5) * p.m + row0 + lane] = s;
}

// The way back: a warp's 32 rows of a kept group as they lie in memory, and
// each row's scale.
__device__ __forceinline__ float kept_fetch(const F16GemmParams& p, uint4 (&r)[4], int lane, int64_t ld,
                                            int row0, int at) {
  if (p.zbits == 8) {
    codes_fetch(r, static_cast<const int8_t*>(p.zq), ld, lane, row0, p.m, at);
  } else {
    whole_chunk_fetch(r, static_cast<const uint16_t*>(p.zq) + row0 * ld + at, ld, lane, row0, p.m);
  }
  return row0 + lane < p.m ? p.zs[static_cast<int64_t>(at >> 5) * p.m + row0 + lane] : 0.f;
}

// 16 values of a lane's row: codes in the slice (16 bits) or in its registers.
template <bool BF16>
__device__ __forceinline__ void kept_half(const F16GemmParams& p, uint32_t slice, int lane, int half,
                                          const uint32_t (&q)[8], float scale, float (&v)[16]) {
  if (p.zbits == 8) {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = scale * code8_value(q[4 * half + (j >> 2)], j & 3);
  } else {
    const uint4 a = ld_shared_v4(slice + slice_off(lane, 2 * half));
    const uint4 b = ld_shared_v4(slice + slice_off(lane, 2 * half + 1));
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    kept16_values<BF16>(w, scale, v);
  }
}

template <int EPI, bool BF16>
__global__ void __launch_bounds__(F16Roles<EPI>::kThreads, 1)
    f16_pair_gemm_kernel(const __grid_constant__ F16GemmParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int stage_bytes = kF16ABytes + p.b_stage;
  const uint32_t epi_smem = smem + p.stages * stage_bytes;
  constexpr int kEpiWarps = F16Roles<EPI>::kEpiWarps, kSlices = F16Roles<EPI>::kSlices;
  const uint32_t bars = epi_smem + F16Roles<EPI>::kEpiBytes;
  const auto full = [&](int s) { return bars + 8u * s; };
  const auto empty = [&](int s) { return bars + 8u * (kF16MaxStages + s); };
  const auto acc_full = [&](int b) { return bars + 8u * (2 * kF16MaxStages + b); };
  const auto acc_empty = [&](int b) { return bars + 8u * (2 * kF16MaxStages + 2 + b); };
  const uint32_t tmem_slot = bars + 8u * (2 * kF16MaxStages + 4);

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full(b), 1);
      mbar_init(acc_empty(b), 2 * kEpiWarps);
    }
    mbar_fence_init();
    tma_prefetch_desc(&p.map_a);
    tma_prefetch_desc(&p.map_b);
  }
  if (warp == 2) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
    tc_fence_before();
  }
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = ld_shared_u32(tmem_slot);
  pdl_entry();

  const int kblocks = (p.k + 63) >> 6;
  const int tiles = p.tiles_m * p.tiles_n;
  const int half_n = p.tn >> 1;
  // tile -> (row tile, column tile): columns advance after group_m row tiles,
  // so the tiles in flight share both operands in L2
  const auto tile_at = [&](int t, int& tm, int& tc) {
    const int per = p.group_m * p.tiles_n;
    const int g = t / per, first = g * p.group_m;
    const int rows = min(p.group_m, p.tiles_m - first);
    const int r = t - g * per;
    tm = first + r % rows;
    tc = r / rows;
  };

  if (warp == 0 || warp == 3) {
    // ---- TMA producers: warp 0 this CTA's rows of A, warp 3 of B ----
    const bool first = warp == 0;
    RingCursor ring;
    uint32_t filled = 0;  // slots in use at the end, up to the ring's depth
    bool ok = true;
    const uint32_t leader = mapa_shared(bars, 0);
    for (int t = pair; t < tiles && ok; t += pairs) {
      int tm, tc;
      tile_at(t, tm, tc);
      const int row = tm * 256 + static_cast<int>(rank) * 128;
      const int brow = EPI == kEpiGated ? tc * half_n + (rank ? p.up_row : 0)
                                        : tc * p.tn + static_cast<int>(rank) * half_n;
      for (int kk = 0; kk < kblocks * 64; kk += 64) {
        const int s = ring.slot;
        if (filled == static_cast<uint32_t>(p.stages)) {
          if (!mbar_wait_cl(empty(s), ring.parity ^ 1, kErrF16WaitEmpty)) {
            ok = false;
            break;
          }
        } else {
          ++filled;
        }
        const uint32_t bar = leader + 8u * s, a = smem + s * stage_bytes;
        if (elect_one()) {
          if (first) {
            if (rank == 0) mbar_arrive_expect_tx(full(s), 2 * stage_bytes);
            load_operand(a, &p.map_a, p.a_mn, p.a_wide, 128, row, kk, bar);
          } else {
            load_operand(a + kF16ABytes, &p.map_b, p.b_mn, p.b_wide, half_n, brow, kk, bar);
          }
        }
        ring.step(p.stages);
      }
    }
    // the last commits arrive here before this CTA may exit: the slots in use,
    // oldest first
    if (filled < static_cast<uint32_t>(p.stages)) ring = RingCursor{};
    else ring.parity ^= 1;
    for (uint32_t i = 0; ok && i < filled; ++i) {
      ok = mbar_wait_cl(empty(ring.slot), ring.parity, kErrF16WaitEmpty);
      ring.step(p.stages);
    }
    if (!ok) {  // copies in flight land before shared memory is given up
      const unsigned long long t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 1000000ull) {
      }
    }
  } else if (warp == 1 && rank == 0) {
    // ---- MMA issuer of the pair ----
    const uint32_t idesc = idesc_f16(BF16, 256, p.tn, p.a_mn, p.b_mn);
    const uint32_t a_step = p.a_mn ? 128u : 2u, b_step = p.b_mn ? 128u : 2u;  // 16 of k, /16 bytes
    const uint64_t a_desc = operand_desc(p.a_mn, 8192), b_desc = operand_desc(p.b_mn, 8192);
    RingCursor ring;
    uint32_t nt = 0;
    bool ok = true;
    for (int t = pair; t < tiles && ok; t += pairs, ++nt) {
      const uint32_t buf = nt & 1, use = nt >> 1;
      if (use > 0 && !mbar_wait_cl(acc_empty(buf), (use - 1) & 1, kErrF16WaitAccEmpty)) break;
      tc_fence_after();
      const uint32_t d = tmem + buf * 256;
      for (int kb = 0; kb < kblocks; ++kb) {
        const int s = ring.slot;
        if (!mbar_wait_cl(full(s), ring.parity, kErrF16WaitFull)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t a = desc_addr(smem + s * stage_bytes);
        const uint64_t ad = a_desc + a, bd = b_desc + (a + (kF16ABytes >> 4));
        if (elect_one()) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mma_f16_ss_pair(d, ad + j * a_step, bd + j * b_step, idesc, (kb | j) != 0);
          mma_commit_both(empty(s));
        }
        ring.step(p.stages);
      }
      if (ok && elect_one()) mma_commit_both(acc_full(buf));
    }
  } else if (warp >= 4) {
    // ---- epilogue: warp w reads TMEM lanes 32 (w & 3).., its share of the chunks ----
    const int quarter = warp & 3, side = (warp - 4) >> 2;
    const uint32_t slice0 = epi_smem + (warp - 4) * kSlices * kF16StageSlice;
    const uint32_t slice1 = slice0 + (kSlices - 1) * kF16StageSlice;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    uint32_t nt = 0;
    for (int t = pair; t < tiles; t += pairs, ++nt) {
      int tm, tc;
      tile_at(t, tm, tc);
      const uint32_t buf = nt & 1, use = nt >> 1;
      const int row0 = tm * 256 + static_cast<int>(rank) * 128 + quarter * 32;
      const int width = EPI == kEpiGated ? half_n : p.tn;
      const int cbase = tc * width;
      // kEpiGatedBwd: the kept groups of the next chunk, on their way
      uint4 rg[4], ru[4];
      float next_sg = 0.f, next_su = 0.f;
      const auto fetch = [&](int col) {
        next_sg = kept_fetch(p, rg, lane, 2 * p.n32, row0, col);
        next_su = kept_fetch(p, ru, lane, 2 * p.n32, row0, static_cast<int>(p.n32) + col);
      };
      if (EPI == kEpiGatedBwd && cbase + side * 32 < p.n) fetch(cbase + side * 32);
      if (!mbar_wait_cl(acc_full(buf), use & 1, kErrF16WaitAccFull)) break;
      tc_fence_after();
      const uint32_t acc = tmem + buf * 256 + lanes;
      for (int c0 = side * 32; c0 < width; c0 += 8 * kEpiWarps) {
        const int col = cbase + c0;
        if (col >= p.n) break;
        if constexpr (EPI == kEpiLinear) {
          uint4 rres[4];
          if (p.residual.p) chunk_fetch(rres, p.residual, lane, row0, p.m, col, p.n);
          float v[32];
          tmem_ld_f32x32(acc + c0, v);
          if (p.bias) {
            const float bl = col + lane < p.n ? ld_16<BF16>(p.bias, col + lane) : 0.f;
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] += __shfl_sync(0xffffffffu, bl, j);
          }
          uint32_t w[16];
          if (p.zbits) {
            if (col + 32 > p.n) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (col + j >= p.n) v[j] = 0.f;
            }
            keep_rows<BF16>(p, slice0, lane, v, p.n32, row0, col);
          }
          act_row(p.act, v);
          if (p.residual.p) {
            chunk_to_rows(slice1, lane, rres, chunk_whole(p.residual, col, p.n), w);
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] += unpack_16<BF16>(w[j >> 1], j & 1);
          }
          pack_row<BF16>(v, w);
          chunk_store(slice0, lane, w, p.out, row0, p.m, col, p.n);
        } else if constexpr (EPI == kEpiGated) {
          float g[32], u[32];
          tmem_ld_f32x32(acc + c0, g);
          tmem_ld_f32x32(acc + half_n + c0, u);
          uint32_t w[16];
          if (p.zbits) {
            if (col + 32 > p.n) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (col + j >= p.n) g[j] = u[j] = 0.f;
            }
            keep_rows<BF16>(p, slice0, lane, g, 2 * p.n32, row0, col);
            keep_rows<BF16>(p, slice1, lane, u, 2 * p.n32, row0, static_cast<int>(p.n32) + col);
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            g[j] = clamp_top(g[j], p.limit);
            u[j] = clamp_both(u[j], p.limit);
          }
          act_row(p.act, g);
#pragma unroll
          for (int j = 0; j < 32; ++j) g[j] *= u[j];
          pack_row<BF16>(g, w);
          chunk_store(slice0, lane, w, p.out, row0, p.m, col, p.n);
        } else {
          const float sg = next_sg, su = next_su;
          uint32_t qg[8] = {}, qu[8] = {}, wh[16];
          if (p.zbits == 8) {
            codes_to_rows(slice0, lane, rg[0], rg[1], qg);
            codes_to_rows(slice1, lane, ru[0], ru[1], qu);
          } else {
            whole_chunk_to_slice(slice0, lane, rg);
            whole_chunk_to_slice(slice1, lane, ru);
            __syncwarp();
          }
          if (c0 + 8 * kEpiWarps < width && col + 8 * kEpiWarps < p.n) fetch(col + 8 * kEpiWarps);
          // half a group at a time: its results take its codes' place in the slices
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float v[16], g[16], u[16];
            tmem_ld_f32x16(acc + c0 + 16 * half, v);
            kept_half<BF16>(p, slice0, lane, half, qg, sg, g);
            kept_half<BF16>(p, slice1, lane, half, qu, su, u);
            uint32_t wg[8], wu[8], w[8];
            gated_backward_row<BF16>(p.act, p.limit, v, g, u, wg, wu, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) wh[8 * half + j] = w[j];
            row_to_slice(slice0, lane, 2 * half, wg);
            row_to_slice(slice1, lane, 2 * half, wu);
          }
          slice_store(slice0, lane, p.d0, row0, p.m, col, p.n);
          slice_store(slice1, lane, p.d1, row0, p.m, col, p.n);
          if (p.out.p) chunk_store(slice0, lane, wh, p.out, row0, p.m, col, p.n);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cl(mapa_shared(acc_empty(buf), 0));
    }
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync_all();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

}  // namespace dsv4
