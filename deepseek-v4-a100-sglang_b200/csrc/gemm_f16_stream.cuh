// 16-bit products for few tokens: the weights stream once through the SMs.
//
// For up to 128 tokens a product is bound by reading its weights, so the roles
// are swapped: 128 weight rows are the MMA's M, the tokens (padded to 16) its
// N, and the contraction is split over the CTAs of a cluster so that the
// weight stream runs on most SMs however few row tiles there are.  Each CTA
// keeps its ring of TMA boxes full (16 KB of weights per 64 of k) and sums its
// part in tensor memory; the parts meet in distributed shared memory, where
// every CTA of the cluster adds and finishes an equal share of the results in
// a fixed order.  One launch, no workspace, no atomics.
#pragma once

#include "gemm_f16.cuh"

namespace dsv4 {

enum F16StreamErr : int {
  kErrStreamWaitEmpty = 0x211,
  kErrStreamWaitFull = 0x212,
  kErrStreamWaitAcc = 0x213,
};

constexpr int kStreamThreads = 256;
constexpr int kStreamMaxTokens = 128;
constexpr int kStreamMaxStages = 12;
constexpr int kStreamBarBytes = 256;
static_assert((2 * kStreamMaxStages + 1) * 8 + 8 <= kStreamBarBytes, "barrier area");

struct F16StreamParams {
  CUtensorMap map_w, map_x;
  int m, n, k;          // tokens, result columns, contraction
  int tn;               // tokens of a tile, a multiple of 16
  int tmem_cols;
  int stages, x_stage;  // ring depth, bytes of tokens per stage
  int w_mn, x_mn;
  int row_tiles, cluster;
  int up_row;           // kEpiGated: weight row of up row 0
  int act;
  float limit;
  const void* bias;
  F16Mat residual, out;
};

__device__ __forceinline__ void mma_f16_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                           uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tma_load_2d_plain(uint32_t dst, const CUtensorMap* map, int c0,
                                                  int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}

// Sum over the cluster, in rank order, of 4 fp32 at the same offset.
__device__ __forceinline__ void sum_parts(uint32_t at, int cluster, float (&v)[4]) {
  float q[8][4];
#pragma unroll
  for (int r = 0; r < 8; ++r)
    if (r < cluster)
      asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                   : "=f"(q[r][0]), "=f"(q[r][1]), "=f"(q[r][2]), "=f"(q[r][3])
                   : "r"(mapa_shared(at, r))
                   : "memory");
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = q[0][j];
#pragma unroll
  for (int r = 1; r < 8; ++r)
    if (r < cluster) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += q[r][j];
    }
}

template <int EPI, bool BF16>
__global__ void __launch_bounds__(kStreamThreads)
    f16_stream_gemm_kernel(const __grid_constant__ F16StreamParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int tile = blockIdx.x / p.cluster;
  const int row_tile = tile % p.row_tiles, token0 = tile / p.row_tiles * p.tn;
  const int stage_bytes = kF16ABytes + p.x_stage;
  const uint32_t bars = smem + p.stages * stage_bytes;
  const auto full = [&](int s) { return bars + 8u * s; };
  const auto empty = [&](int s) { return bars + 8u * (kStreamMaxStages + s); };
  const uint32_t acc_full = bars + 8u * (2 * kStreamMaxStages);
  const uint32_t tmem_slot = acc_full + 8u;

  // this CTA's share of the contraction, in blocks of 64
  const int kblocks = (p.k + 63) >> 6;
  const int per = kblocks / p.cluster, more = kblocks % p.cluster;
  const int kb0 = rank * per + min(rank, more), nkb = per + (rank < more ? 1 : 0);

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    mbar_init(acc_full, 1);
    mbar_fence_init();
    tma_prefetch_desc(&p.map_w);
    tma_prefetch_desc(&p.map_x);
  }
  if (warp == 2) {
    tmem_alloc(tmem_slot, p.tmem_cols);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ld_shared_u32(tmem_slot);
  pdl_entry();

  if (warp == 0 && lane == 0) {
    const int row = EPI == kEpiGated ? row_tile * 64 : row_tile * 128;
    const int x_boxes = p.x_mn ? (p.tn + 63) >> 6 : 1;
    RingCursor ring;
    bool ok = true;
    for (int i = 0; i < nkb; ++i) {
      const int s = ring.slot;
      if (i >= p.stages && !mbar_wait(empty(s), ring.parity ^ 1, kErrStreamWaitEmpty)) {
        ok = false;
        break;
      }
      ring.step(p.stages);
      const uint32_t w = smem + s * stage_bytes, x = w + kF16ABytes, bar = full(s);
      const int kk = (kb0 + i) * 64;
      mbar_arrive_expect_tx(bar, stage_bytes);
      if (EPI == kEpiGated) {  // boxes of 64 rows (or 64 x 64, MN-major)
        if (p.w_mn) {
          tma_load_2d_plain(w, &p.map_w, row, kk, bar);
          tma_load_2d_plain(w + 8192, &p.map_w, p.up_row + row, kk, bar);
        } else {
          tma_load_2d_plain(w, &p.map_w, kk, row, bar);
          tma_load_2d_plain(w + 8192, &p.map_w, kk, p.up_row + row, bar);
        }
      } else if (p.w_mn) {
        tma_load_2d_plain(w, &p.map_w, row, kk, bar);
        tma_load_2d_plain(w + 8192, &p.map_w, row + 64, kk, bar);
      } else {
        tma_load_2d_plain(w, &p.map_w, kk, row, bar);
      }
      if (p.x_mn) {
        for (int j = 0; j < x_boxes; ++j)
          tma_load_2d_plain(x + j * 8192, &p.map_x, token0 + j * 64, kk, bar);
      } else {
        tma_load_2d_plain(x, &p.map_x, kk, token0, bar);
      }
    }
    if (!ok) {  // copies in flight land before shared memory is used again
      const unsigned long long t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 1000000ull) {
      }
    }
  } else if (warp == 1 && lane == 0) {
    const uint32_t idesc = idesc_f16(BF16, 128, p.tn, p.w_mn, p.x_mn);
    const uint32_t w_step = p.w_mn ? 128u : 2u, x_step = p.x_mn ? 128u : 2u;
    const uint64_t w_desc = operand_desc(p.w_mn), x_desc = operand_desc(p.x_mn);
    RingCursor ring;
    uint32_t accumulate = 0;
    bool ok = true;
    for (int i = 0; i < nkb; ++i) {
      const int s = ring.slot;
      if (!mbar_wait(full(s), ring.parity, kErrStreamWaitFull)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t w = desc_addr(smem + s * stage_bytes);
      uint64_t wd = w_desc + w, xd = x_desc + (w + (kF16ABytes >> 4));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        mma_f16_ss(tmem, wd, xd, idesc, accumulate);
        accumulate = 1;
        wd += w_step, xd += x_step;
      }
      mma_commit(empty(s));
      ring.step(p.stages);
    }
    if (ok) mma_commit(acc_full);
  }
  __syncwarp();

  // this CTA's part: fp32 [token][128 weight rows], over the ring that the
  // MMAs have finished reading
  const int tokens = min(p.tn, p.m - token0);
  if (warp >= 4) {
    mbar_wait(acc_full, 0, kErrStreamWaitAcc);
    tc_fence_after();
    const int quarter = warp & 3;
    const uint32_t acc = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    for (int t0 = 0; t0 < tokens; t0 += 16) {
      int32_t v[16];
      tmem_ld_x16(acc + t0, v);
      tmem_ld_wait_regs(v);
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (t0 + j < tokens)
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(smem + (t0 + j) * 512 + quarter * 128 +
                                                        lane * 4),
                       "r"(v[j])
                       : "memory");
    }
    tc_fence_before();
  }
  cluster_sync_all();

  // every CTA adds the parts of its share of the results, in rank order; a
  // thread takes 4 columns of a token, all parts in flight at once
  constexpr int kCols = EPI == kEpiGated ? 64 : 128, kPieces = kCols / 4;
  const int col0 = row_tile * kCols;
  for (int e = rank * kStreamThreads + threadIdx.x; e < tokens * kPieces;
       e += p.cluster * kStreamThreads) {
    const int t = e / kPieces, c = e % kPieces * 4;
    const int col = col0 + c;
    if (col >= p.n) continue;
    const uint32_t at = smem + t * 512 + c * 4;
    const int64_t row = token0 + t;
    float v[4], u[4];
    sum_parts(at, p.cluster, v);
    if constexpr (EPI == kEpiGated) sum_parts(at + 256, p.cluster, u);
    const bool whole = col + 4 <= p.n;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (EPI == kEpiGated) v[j] = clamp_top(v[j], p.limit);
      if (EPI == kEpiLinear && p.bias && (whole || col + j < p.n)) v[j] += ld_16<BF16>(p.bias, col + j);
    }
    act_dispatch(p.act, [&](auto kind) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = act_value<decltype(kind)::value>(v[j]);
    });
    if constexpr (EPI == kEpiGated) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] *= clamp_both(u[j], p.limit);
    }
    if (EPI == kEpiLinear && p.residual.p) {
      const uint16_t* r = static_cast<const uint16_t*>(p.residual.p) + row * p.residual.ld + col;
      if (whole && p.residual.vec) {
        const uint2 w = *reinterpret_cast<const uint2*>(r);
        v[0] += unpack_16<BF16>(w.x, 0), v[1] += unpack_16<BF16>(w.x, 1);
        v[2] += unpack_16<BF16>(w.y, 0), v[3] += unpack_16<BF16>(w.y, 1);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (col + j < p.n) v[j] += unpack_16<BF16>(r[j], 0);
      }
    }
    uint16_t* o = static_cast<uint16_t*>(p.out.p) + row * p.out.ld + col;
    const uint2 w = make_uint2(pack_16<BF16>(v[0], v[1]), pack_16<BF16>(v[2], v[3]));
    if (whole && p.out.vec) {
      *reinterpret_cast<uint2*>(o) = w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col + j < p.n) o[j] = static_cast<uint16_t>((j < 2 ? w.x : w.y) >> (16 * (j & 1)));
    }
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync_all();  // no CTA leaves while its part may be read
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, p.tmem_cols);
  }
}

}  // namespace dsv4
