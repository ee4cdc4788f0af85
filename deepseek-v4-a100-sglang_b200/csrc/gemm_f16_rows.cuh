// 16-bit products for up to 8 tokens: weights from global memory straight into
// registers.
//
// With so few tokens the products cost nothing next to reading the weights
// once, and what a launch spends before its first load and after its last one
// counts as much as bandwidth: no tensor memory, no barriers, no cluster.  A
// block takes 16 weight rows and its 16 warps split the contraction in
// blocks of 64; a thread loads 16 bytes of a row (8 of k) at a time, all loads
// of two blocks in flight together, and feeds mma.sync with them as they come.
// The order of k inside an MMA is free as long as both operands keep it: a
// thread's 8 consecutive k serve two MMAs, so no shuffle or shared memory lies
// between memory and the tensor cores.  The warps' parts meet in shared memory
// and are added in warp order.  64 registers, so that two blocks fit an SM.
// Rows of more than 2048 keep their loads in flight without a break (4096 x
// 7168: 11.7 us instead of 13.2); the gated product does not gain by it (7168
// -> 2 x 2048: 0.8 us more).
//
// Rows at any even address (an odd k, a view): the two aligned 16-byte pieces
// around 8 values are loaded and shifted together.  That reads a few bytes of
// the rows beside it, never outside the matrix.
//
// kEpiGated: rows 0-7 of the MMA are gate rows, 8-15 the same up rows, so that
// a thread's sums hold both factors.
#pragma once

#include "gemm_f16.cuh"

namespace dsv4 {

constexpr int kRowsThreads = 512;
constexpr int kRowsWarps = kRowsThreads / 32;
constexpr int kRowsMaxTokens = 8;

struct F16RowsParams {
  const uint16_t* x;
  const uint16_t* w;
  int64_t ldx, ldw;
  int m, n, k;
  int up_row;  // kEpiGated
  int act;
  float limit;
  const void* bias;
  F16Mat residual, out;
};

template <bool BF16>
__device__ __forceinline__ void mma_m16n8k16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                             uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (BF16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

// 8 consecutive k of a row; zeros past the `left` that there are.
__device__ __forceinline__ uint4 load_k8(const uint16_t* p, int left) {
  if (left >= 8) return *reinterpret_cast<const uint4*>(p);
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < left) w[j >> 1] |= static_cast<uint32_t>(p[j]) << (16 * (j & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int EPI, bool BF16, bool ALIGNED>
__global__ void __launch_bounds__(kRowsThreads, ALIGNED ? 2 : 1)
    f16_rows_gemm_kernel(const F16RowsParams p) {
  constexpr int kRowsAhead = 2;  // blocks of 64 of k in flight
  __shared__ float s_part[kRowsWarps][128];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, q = lane & 3;
  constexpr int kCols = EPI == kEpiGated ? 8 : 16;  // result columns of a block
  const int col0 = blockIdx.x * kCols;
  const int kblocks = (p.k + 63) >> 6;

  // the two rows of the MMA that a thread reads (past the end, the last again)
  const int ca = min(col0 + g, p.n - 1), cb = EPI == kEpiGated ? ca + p.up_row : min(col0 + 8 + g, p.n - 1);
  const uint16_t* const row_a = p.w + ca * p.ldw;
  const uint16_t* const row_b = p.w + cb * p.ldw;
  // the first weights are asked for in L2 while the kernel before still runs
  // (brought nearer, not read)
#pragma unroll
  for (int u = 0; u < kRowsAhead; ++u) {
    const int k0 = (warp + u * kRowsWarps) * 64 + q * 16;
    if (k0 < p.k) {
      asm volatile("prefetch.global.L2 [%0];" ::"l"(row_a + k0));
      asm volatile("prefetch.global.L2 [%0];" ::"l"(row_b + k0));
    }
  }
  pdl_entry();

  float acc[4] = {};
  const bool live = g < p.m;
  const uint16_t* const token = p.x + (live ? g : 0) * p.ldx;
  if constexpr (!ALIGNED) {
    const Extent we = extent_of(p.w, EPI == kEpiGated ? 2 * p.up_row : p.n, p.ldw, p.k);
    const Extent xe = extent_of(p.x, p.m, p.ldx, p.k);
    // rows are apart by any number of elements, k by whole pieces: a row's shift stays
    const int sa = static_cast<int>(reinterpret_cast<uint64_t>(row_a) & 15);
    const int sb = static_cast<int>(reinterpret_cast<uint64_t>(row_b) & 15);
    const int sx = static_cast<int>(reinterpret_cast<uint64_t>(token) & 15);
    for (int kb = warp; kb < kblocks; kb += kRowsWarps) {
      Window a[2], b[2], x[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k0 = kb * 64 + h * 32 + q * 8, left = p.k - k0;
        a[h].a = a[h].b = b[h].a = b[h].b = x[h].a = x[h].b = make_uint4(0, 0, 0, 0);
        if (left > 0) {
          a[h] = load_window(row_a + k0, left, we);
          b[h] = load_window(row_b + k0, left, we);
          if (live) x[h] = load_window(token + k0, left, xe);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 va = shift_window(a[h], sa), vb = shift_window(b[h], sb), vx = shift_window(x[h], sx);
        mma_m16n8k16<BF16>(acc, va.x, vb.x, va.y, vb.y, vx.x, vx.y);
        mma_m16n8k16<BF16>(acc, va.z, vb.z, va.w, vb.w, vx.z, vx.w);
      }
    }
  }
  if constexpr (ALIGNED) {
    uint4 a[kRowsAhead][2], b[kRowsAhead][2];
    const auto load_weights = [&](int u, int kb) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k0 = kb * 64 + h * 32 + q * 8, left = p.k - k0;
        a[u][h] = b[u][h] = make_uint4(0, 0, 0, 0);
        if (left > 0) {
          a[u][h] = load_k8(row_a + k0, left);
          b[u][h] = load_k8(row_b + k0, left);
        }
      }
    };
    const auto load_tokens = [&](uint4 (&x)[2], int kb) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k0 = kb * 64 + h * 32 + q * 8, left = p.k - k0;
        x[h] = make_uint4(0, 0, 0, 0);
        if (live && left > 0) x[h] = load_k8(token + k0, left);
      }
    };
    const auto multiply = [&](int u, const uint4 (&x)[2]) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mma_m16n8k16<BF16>(acc, a[u][h].x, b[u][h].x, a[u][h].y, b[u][h].y, x[h].x, x[h].y);
        mma_m16n8k16<BF16>(acc, a[u][h].z, b[u][h].z, a[u][h].w, b[u][h].w, x[h].z, x[h].w);
      }
    };
    if (EPI == kEpiLinear && kblocks > kRowsAhead * kRowsWarps) {
      // long rows: a block's registers are filled again as soon as it is done,
      // which leaves none for its tokens (those come from L2 when it is due)
#pragma unroll
      for (int u = 0; u < kRowsAhead; ++u) load_weights(u, warp + u * kRowsWarps);
      for (int kb = warp; kb < kblocks; kb += kRowsAhead * kRowsWarps) {
#pragma unroll
        for (int u = 0; u < kRowsAhead; ++u) {
          uint4 x[2];
          load_tokens(x, kb + u * kRowsWarps);
          multiply(u, x);
          load_weights(u, kb + (u + kRowsAhead) * kRowsWarps);
        }
      }
    } else {
      for (int kb = warp; kb < kblocks; kb += kRowsAhead * kRowsWarps) {
        uint4 x[kRowsAhead][2];
#pragma unroll
        for (int u = 0; u < kRowsAhead; ++u) {
          load_weights(u, kb + u * kRowsWarps);
          load_tokens(x[u], kb + u * kRowsWarps);
        }
#pragma unroll
        for (int u = 0; u < kRowsAhead; ++u) multiply(u, x[u]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) s_part[warp][j * 32 + lane] = acc[j];
  __syncthreads();

  // the sum of MMA row `row` and a token: lane (row % 8) * 4 + token / 2,
  // register row / 8 * 2 + token % 2
  const auto sum = [&](int row, int token) {
    const int at = ((row >> 3) * 2 + (token & 1)) * 32 + (row & 7) * 4 + (token >> 1);
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < kRowsWarps; ++i) v += s_part[i][at];
    return v;
  };
  if (threadIdx.x >= 16 * p.m) return;
  const int t = threadIdx.x >> 4, c = threadIdx.x & 15, col = col0 + c;
  if (c >= kCols || col >= p.n) return;
  float v = sum(c, t);
  if constexpr (EPI == kEpiGated) {
    v = clamp_top(v, p.limit);
  } else if (p.bias) {
    v += ld_16<BF16>(p.bias, col);
  }
  act_dispatch(p.act, [&](auto kind) { v = act_value<decltype(kind)::value>(v); });
  if constexpr (EPI == kEpiGated) v *= clamp_both(sum(c + 8, t), p.limit);
  if (EPI == kEpiLinear && p.residual.p) v += ld_16<BF16>(p.residual.p, t * p.residual.ld + col);
  static_cast<uint16_t*>(p.out.p)[t * p.out.ld + col] =
      static_cast<uint16_t>(pack_16<BF16>(v, 0.f) & 0xffffu);
}

}  // namespace dsv4
