// 16-bit products for few tokens: the weights stream once through the SMs.
//
// For up to 128 tokens a product is bound by reading its weights.  The tokens
// (up to 128) are the MMA's M and a tile of weight rows its N, so the
// accumulator holds one token per lane; the contraction is split over the CTAs
// of a cluster so that the weight stream runs on all SMs however few row tiles
// there are.  Each CTA keeps its ring of TMA boxes full and sums its part in
// tensor memory; the parts meet in distributed shared memory, where every CTA
// of the cluster adds and finishes an equal share of the results in a fixed
// order.  One launch, no workspace, no atomics.
//
// A stage costs its two single threads (TMA producer, MMA issuer) ~0.3 us
// however few bytes it brings, more than its share of HBM bandwidth: so a
// stage holds `atoms` blocks of 64 of k, fetched by one copy per operand.
// Weights as M and tokens as N would cost 128 cycles an MMA however few tokens
// there are; this way round it is 64.  Two CTAs fit an SM: under programmatic
// dependent launch the next product's CTAs come up while this one drains, and
// ask for their first weights in L2 before they wait for it (those are only
// brought nearer, not read: weights that the kernel before still writes are
// safe).  4096 x 7168, one token, back to back: 13.1 us without, 12.2 with.
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
constexpr int kStreamSmem = 112 * 1024;       // two CTAs per SM
constexpr int kStreamSmemAlone = 200 * 1024;  // one
static_assert((2 * kStreamMaxStages + 1) * 8 + 8 <= kStreamBarBytes, "barrier area");

// An MMA reads 128 token rows (16 KB) from where a block's tokens begin,
// however few of them there are; behind the last stage a pad takes that.
__host__ __device__ constexpr int stream_ring_bytes(int stages, int stage, int atoms, int x_atom) {
  const int reach = (atoms - 1) * x_atom + kF16ABytes;
  return stages * stage + (stage < reach ? reach - stage : 0);
}

struct F16StreamParams {
  CUtensorMap map_w, map_x;
  int m, n, k;          // tokens, result columns, contraction
  int tn;               // tokens of a tile, a multiple of 16
  int rows;             // weight rows of a tile, a multiple of 16 up to 128
                        // (kEpiGated: half gate, half up; a multiple of 32)
  int atoms;            // blocks of 64 of k in a stage
  int stages, x_atom, w_atom;  // ring depth, bytes of a block (MN-major: of 64 rows x 64)
  int x_stage, w_stage;
  int x_wide, w_wide;   // K-major, k in whole blocks: one copy brings all blocks of a stage
  int ring_bytes;       // the stages and what the MMA reads behind the last (stream_ring_bytes)
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

__device__ __forceinline__ void tma_load_3d_plain(uint32_t dst, const CUtensorMap* map, int c0,
                                                  int c1, int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void tma_load_4d_plain(uint32_t dst, const CUtensorMap* map, int c0,
                                                  int c1, int c2, int c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void tma_prefetch_3d(const CUtensorMap* map, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}

__device__ __forceinline__ void tma_prefetch_4d(const CUtensorMap* map, int c0, int c1, int c2,
                                                int c3) {
  asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}

// Part sums: fp32 [token][128], the 16-byte pieces of a row XORed with the
// token so that lanes writing the same piece of 32 tokens meet no conflicts.
__device__ __forceinline__ uint32_t part_off(int token, int piece) {
  return static_cast<uint32_t>(token * 512 + ((piece ^ (token & 31)) << 4));
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

// The copies of one stage.  MN-major boxes hold all of the stage's k for 64
// rows; K-major ones all blocks (x_wide, w_wide), or one block each.
template <int EPI>
__device__ __forceinline__ void load_stage(const F16StreamParams& p, uint32_t x, uint32_t w,
                                           uint32_t bar, int token0, int row, int kk) {
  if (p.w_mn) {
    tma_load_2d_plain(w, &p.map_w, row, kk, bar);
    tma_load_2d_plain(w + (p.w_stage >> 1), &p.map_w, EPI == kEpiGated ? p.up_row + row : row + 64,
                      kk, bar);
  } else if (p.w_wide) {
    if (EPI == kEpiGated) {
      tma_load_4d_plain(w, &p.map_w, 0, row, 0, kk >> 6, bar);
    } else {
      tma_load_3d_plain(w, &p.map_w, 0, row, kk >> 6, bar);
    }
  } else {
    for (int a = 0; a < p.atoms; ++a) {
      tma_load_2d_plain(w + a * p.w_atom, &p.map_w, kk + a * 64, row, bar);
      if (EPI == kEpiGated)
        tma_load_2d_plain(w + a * p.w_atom + (p.w_atom >> 1), &p.map_w, kk + a * 64,
                          p.up_row + row, bar);
    }
  }
  if (p.x_mn) {
    for (int j = 0; j * 64 < p.tn; ++j)
      tma_load_2d_plain(x + j * p.x_atom * p.atoms, &p.map_x, token0 + j * 64, kk, bar);
  } else if (p.x_wide) {
    tma_load_3d_plain(x, &p.map_x, 0, token0, kk >> 6, bar);
  } else {
    for (int a = 0; a < p.atoms; ++a)
      tma_load_2d_plain(x + a * p.x_atom, &p.map_x, kk + a * 64, token0, bar);
  }
}

template <int EPI, bool BF16>
__global__ void __launch_bounds__(kStreamThreads)
    f16_stream_gemm_kernel(const __grid_constant__ F16StreamParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int tile = blockIdx.x / p.cluster;
  const int row_tile = tile % p.row_tiles, token0 = tile / p.row_tiles * p.tn;
  const int cols = EPI == kEpiGated ? p.rows >> 1 : p.rows;  // result columns of a tile
  const int col0 = row_tile * cols;
  const int stage_bytes = p.x_stage + p.w_stage;
  const uint32_t bars = smem + p.ring_bytes;
  const auto full = [&](int s) { return bars + 8u * s; };
  const auto empty = [&](int s) { return bars + 8u * (kStreamMaxStages + s); };
  const uint32_t acc_full = bars + 8u * (2 * kStreamMaxStages);
  const uint32_t tmem_slot = acc_full + 8u;

  // this CTA's share of the contraction, in stages
  const int kspan = p.atoms * 64, kblocks = (p.k + kspan - 1) / kspan;
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
  if (threadIdx.x == 96 && p.w_wide) {
    for (int i = 0; i < min(nkb, p.stages); ++i) {
      const int block = (kb0 + i) * p.atoms;
      if (EPI == kEpiGated) {
        tma_prefetch_4d(&p.map_w, 0, col0, 0, block);
      } else {
        tma_prefetch_3d(&p.map_w, 0, col0, block);
      }
    }
  }
  if (warp == 2) {
    tmem_alloc(tmem_slot, 128);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ld_shared_u32(tmem_slot);
  pdl_entry();

  if (warp == 0) {
    RingCursor ring;
    bool ok = true;
    for (int i = 0; i < nkb; ++i) {
      const int s = ring.slot;
      if (i >= p.stages && !mbar_wait(empty(s), ring.parity ^ 1, kErrStreamWaitEmpty)) {
        ok = false;
        break;
      }
      ring.step(p.stages);
      const uint32_t x = smem + s * stage_bytes;
      if (elect_one()) {
        mbar_arrive_expect_tx(full(s), stage_bytes);
        load_stage<EPI>(p, x, x + p.x_stage, full(s), token0, col0, (kb0 + i) * kspan);
      }
    }
    if (!ok) {  // copies in flight land before shared memory is used again
      const unsigned long long t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 1000000ull) {
      }
    }
  } else if (warp == 1) {
    // M = 128 whatever the tokens: the rows behind them are other bytes of the
    // ring, and only fill lanes that nobody reads
    const uint32_t idesc = idesc_f16(BF16, 128, p.rows, p.x_mn, p.w_mn);
    const uint32_t w_step = p.w_mn ? 128u : 2u, x_step = p.x_mn ? 128u : 2u;
    const uint64_t w_desc = operand_desc(p.w_mn, p.w_atom * p.atoms);
    const uint64_t x_desc = operand_desc(p.x_mn, p.x_atom * p.atoms);
    // from one block to the next (MN-major: k just goes on)
    const uint32_t w_next = p.w_mn ? 512u : p.w_atom >> 4, x_next = p.x_mn ? 512u : p.x_atom >> 4;
    RingCursor ring;
    bool ok = true;
    for (int i = 0; i < nkb; ++i) {
      const int s = ring.slot;
      if (!mbar_wait(full(s), ring.parity, kErrStreamWaitFull)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t at = smem + s * stage_bytes;
      uint64_t xd = x_desc + desc_addr(at), wd = w_desc + desc_addr(at + p.x_stage);
      if (elect_one()) {
        for (int a = 0; a < p.atoms; ++a) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mma_f16_ss(tmem, xd + j * x_step, wd + j * w_step, idesc, (i | a | j) != 0);
          wd += w_next, xd += x_next;
        }
        mma_commit(empty(s));
      }
      ring.step(p.stages);
    }
    if (ok && elect_one()) mma_commit(acc_full);
  }
  __syncwarp();

  // this CTA's part, over the ring that the MMAs have finished reading
  const int tokens = min(p.tn, p.m - token0);
  if (warp >= 4) {
    mbar_wait(acc_full, 0, kErrStreamWaitAcc);
    tc_fence_after();
    const int t = (warp & 3) * 32 + lane;
    if ((warp & 3) * 32 < tokens) {
      const uint32_t acc = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
      for (int c = 0; c < p.rows; c += 16) {
        int32_t v[16];
        tmem_ld_x16(acc + c, v);
        tmem_ld_wait_regs(v);
        if (t < tokens) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            st_shared_v4(smem + part_off(t, (c >> 2) + j),
                         make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]));
        }
        __syncwarp();
      }
    }
    tc_fence_before();
  }
  cluster_sync_all();

  // every CTA adds the parts of its share of the results, in rank order; a
  // thread takes 4 columns of a token, all parts in flight at once
  const int pieces = cols >> 2;
  for (int e = rank * kStreamThreads + threadIdx.x; e < tokens * pieces;
       e += p.cluster * kStreamThreads) {
    const int t = e / pieces, piece = e - t * pieces;
    const int col = col0 + 4 * piece;
    if (col >= p.n) continue;
    const int64_t row = token0 + t;
    float v[4], u[4];
    sum_parts(smem + part_off(t, piece), p.cluster, v);
    if constexpr (EPI == kEpiGated) sum_parts(smem + part_off(t, pieces + piece), p.cluster, u);
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
    tmem_dealloc(tmem, 128);
  }
}

}  // namespace dsv4
