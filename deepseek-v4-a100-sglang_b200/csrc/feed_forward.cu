// C ABI of the 16-bit feed-forward operators (declared in include/dsv4_b200.h):
// products with bias, activation and residual, the gated block with its
// backward pass, and activation checkpoints in 8 bits.

#include <limits>

#include "host_common.h"

#include "feed_forward_kernels.cuh"
#include "gemm_f16.cuh"
#include "gemm_f16_rows.cuh"
#include "gemm_f16_stream.cuh"

namespace dsv4 {

namespace {

template <int EPI>
cudaError_t pair_attrs() {
  cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<void*>(&f16_pair_gemm_kernel<EPI, true>),
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, kF16SmemMax);
  if (e != cudaSuccess) return e;
  return cudaFuncSetAttribute(reinterpret_cast<void*>(&f16_pair_gemm_kernel<EPI, false>),
                              cudaFuncAttributeMaxDynamicSharedMemorySize, kF16SmemMax);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// To whole elements, as every pointer to them has to be.
bool aligned_to(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

F16Mat mat16(const void* p, int64_t ld) {
  return {const_cast<void*>(p), ld, aligned16(p) && ld % 8 == 0};
}

int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// 2-D operand of `rows` x `k` 16-bit elements, 128-byte swizzled boxes: K-major
// {64 of k, box_rows}, MN-major {64 rows, box_k of k}.
int encode_operand(CUtensorMap* map, const char* what, const void* p, int64_t rows, int64_t k,
                   int64_t ld, int mn, int box_rows, bool bf16, int box_k = 64) {
  if (tensor_map_encoder() == nullptr) return fail(DSV4_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const int64_t inner = mn ? rows : k, outer = mn ? k : rows;
  DSV4_REQUIRE(aligned16(p) && ld % 8 == 0 && ld >= inner,
               "%s must be 16-byte aligned with a row stride of at least its row and a multiple of "
               "8 elements (row stride %lld, row %lld)", what, (long long)ld, (long long)inner);
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * 2};
  cuuint32_t box[2] = {64, static_cast<cuuint32_t>(mn ? box_k : box_rows)};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = tensor_map_encoder()(
      map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
      const_cast<void*>(p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(DSV4_ERR_CUDA, "tensor map (%s) encode failed: %d", what, (int)r);
  return DSV4_OK;
}

// K-major operand whose k is a whole number of 64s, as {64, rows, k / 64} (or,
// for gate and up, {64, rows of a half, 2, k / 64}): one box holds several
// blocks of k, each laid out as encode_operand's.
int encode_wide(CUtensorMap* map, const char* what, const void* p, int64_t rows, int64_t k,
                int64_t ld, int box_rows, int atoms, bool gated, bool bf16) {
  if (tensor_map_encoder() == nullptr) return fail(DSV4_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  DSV4_REQUIRE(aligned16(p) && ld % 8 == 0 && ld >= k,
               "%s must be 16-byte aligned with a row stride of at least its row and a multiple of "
               "8 elements (row stride %lld, row %lld)", what, (long long)ld, (long long)k);
  const cuuint64_t row = static_cast<cuuint64_t>(ld) * 2, blocks = static_cast<cuuint64_t>(k / 64);
  const cuuint64_t half = static_cast<cuuint64_t>(rows / 2);
  const cuuint32_t br = static_cast<cuuint32_t>(box_rows), ba = static_cast<cuuint32_t>(atoms);
  const cuuint64_t dims3[3] = {64, static_cast<cuuint64_t>(rows), blocks}, str3[2] = {row, 128};
  const cuuint64_t dims4[4] = {64, half, 2, blocks}, str4[3] = {row, row * half, 128};
  const cuuint32_t box3[3] = {64, br, ba}, box4[4] = {64, br, 2, ba}, one[4] = {1, 1, 1, 1};
  const CUresult r = tensor_map_encoder()(
      map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, gated ? 4 : 3,
      const_cast<void*>(p), gated ? dims4 : dims3, gated ? str4 : str3, gated ? box4 : box3, one,
      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(DSV4_ERR_CUDA, "tensor map (%s) encode failed: %d", what, (int)r);
  return DSV4_OK;
}

// MN-major operand with a whole number of 64s of rows, as {64, k, rows / 64}:
// one box holds all of a CTA's rows, laid out as encode_operand's boxes.
int encode_wide_mn(CUtensorMap* map, const char* what, const void* p, int64_t rows, int64_t k,
                   int64_t ld, int box_rows, bool bf16) {
  if (tensor_map_encoder() == nullptr) return fail(DSV4_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  DSV4_REQUIRE(aligned16(p) && ld % 8 == 0 && ld >= rows,
               "%s must be 16-byte aligned with a row stride of at least its row and a multiple of "
               "8 elements (row stride %lld, row %lld)", what, (long long)ld, (long long)rows);
  const cuuint64_t dims[3] = {64, static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows / 64)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld) * 2, 128};
  const cuuint32_t box[3] = {64, 64, static_cast<cuuint32_t>(box_rows / 64)}, one[3] = {1, 1, 1};
  const CUresult r = tensor_map_encoder()(
      map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
      const_cast<void*>(p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(DSV4_ERR_CUDA, "tensor map (%s) encode failed: %d", what, (int)r);
  return DSV4_OK;
}

// Columns of a pair tile, and the microseconds that the pair product takes with
// them.  64 of k cost a tile 0.11 us and 1.04 ns a column (measured at 64, 128
// and 256 columns: 173, 229 and 377 ns, the last under the power cap); the tile
// that needs the least over all waves wins, the wider one on a tie.  3 us are
// set-up and the last tile's epilogue.
int pick_tn(int m, int n, int k, bool gated, double* us) {
  const int pairs = sm_count() / 2, tiles_m = (m + 255) / 256;
  const int step = gated ? 64 : 32;
  int best = 0;
  for (int tn = 256; tn >= 64; tn -= step) {
    const int width = gated ? tn / 2 : tn;
    const int64_t tiles = static_cast<int64_t>(tiles_m) * ((n + width - 1) / width);
    const double cost = static_cast<double>((tiles + pairs - 1) / pairs) * ((k + 63) / 64) * (0.11 + 0.00104 * tn) + 3.0;
    if (best == 0 || cost < 0.99 * *us) best = tn, *us = cost;
  }
  return best;
}

template <int EPI>
int launch_pair_gemm(F16GemmParams& p, const void* a, int64_t lda, int a_mn, const void* b,
                     int64_t b_rows, int64_t ldb, int b_mn, bool bf16, cudaStream_t st) {
  p.a_mn = a_mn != 0;
  p.b_mn = b_mn != 0;
  double us = 0;
  p.tn = pick_tn(p.m, p.n, p.k, EPI == kEpiGated, &us);
  const int half = p.tn / 2, width = EPI == kEpiGated ? half : p.tn;
  p.b_stage = p.b_mn ? (half + 63) / 64 * 8192 : half * 128;
  const int stage = kF16ABytes + p.b_stage;
  const int fixed = 1024 + F16Roles<EPI>::kEpiBytes + kF16BarBytes;
  p.stages = (kF16SmemMax - fixed) / stage;
  if (p.stages > kF16MaxStages) p.stages = kF16MaxStages;
  p.tiles_m = (p.m + 255) / 256;
  p.tiles_n = (p.n + width - 1) / width;
  p.group_m = 8;
  DSV4_REQUIRE(static_cast<int64_t>(p.tiles_m) * p.tiles_n < (1ll << 30), "product too large");
  p.a_wide = p.a_mn && p.m % 64 == 0;
  p.b_wide = p.b_mn && b_rows % 64 == 0 && half % 64 == 0 && p.up_row % 64 == 0;
  if (int r = p.a_wide ? encode_wide_mn(&p.map_a, "a", a, p.m, p.k, lda, 128, bf16)
                       : encode_operand(&p.map_a, "a", a, p.m, p.k, lda, p.a_mn, 128, bf16))
    return r;
  if (int r = p.b_wide ? encode_wide_mn(&p.map_b, "b", b, b_rows, p.k, ldb, half, bf16)
                       : encode_operand(&p.map_b, "b", b, b_rows, p.k, ldb, p.b_mn, half, bf16))
    return r;
  int64_t pairs = sm_count() / 2;
  const int64_t tiles = static_cast<int64_t>(p.tiles_m) * p.tiles_n;
  if (tiles < pairs) pairs = tiles;
  const dim3 grid(static_cast<unsigned>(2 * pairs));
  const size_t smem = fixed + static_cast<size_t>(p.stages) * stage;
  if (bf16) {
    launch_cluster(&f16_pair_gemm_kernel<EPI, true>, grid, dim3(F16Roles<EPI>::kThreads), smem, st, 2, p);
  } else {
    launch_cluster(&f16_pair_gemm_kernel<EPI, false>, grid, dim3(F16Roles<EPI>::kThreads), smem, st, 2, p);
  }
  return check_launch("f16_pair_gemm_kernel");
}

// Clusters that run at once, by [two CTAs per SM][log2 of the cluster size]
// (a cluster does not cross a GPC, so this is less than SMs / size).
constexpr int kMaxDevices = 64;
int g_stream_room[kMaxDevices][2][4];

const int (*stream_room())[4] {
  int dev = 0;
  cudaGetDevice(&dev);
  return g_stream_room[dev >= 0 && dev < kMaxDevices ? dev : 0];
}

cudaError_t query_stream_room() {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || dev < 0 || dev >= kMaxDevices) return e;
  for (int two = 0; two < 2; ++two)
    for (int log2 = 0; log2 < 4; ++log2) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(1024);
      cfg.blockDim = dim3(kStreamThreads);
      cfg.dynamicSmemBytes = two ? kStreamSmem : kStreamSmemAlone;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 1u << log2;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int n = 0;
      e = cudaOccupancyMaxActiveClusters(&n, &f16_stream_gemm_kernel<kEpiLinear, true>, &cfg);
      if (e != cudaSuccess) return e;
      g_stream_room[dev][two][log2] = n > 0 ? n : 1;
    }
  return cudaSuccess;
}

// Tokens of a tile: all of them up to 128, else tiles of equal height.
int stream_tokens(int64_t m) {
  const int64_t tiles = (m + kStreamMaxTokens - 1) / kStreamMaxTokens;
  return static_cast<int>(round_up((m + tiles - 1) / tiles, 16));
}

// Few tokens: the weight-streaming kernel.  A launch takes as long as its
// busiest SM, whose work is counted in weight rows x blocks of k: a block of a
// CTA costs its weight rows and, from L2, a third as much for its tokens; the
// part sums of a tile count as tokens x rows / 32.  One CTA per SM with all of
// the shared memory is 8 % slower than the same work in two halves; two need
// at least 8 blocks each.  Doubling the cluster costs 2 %.  The least of all
// tile heights and cluster sizes is taken.  (Fitted to 6 shapes, 512 x 1024 to
// 14336 x 1024 and 4096 x 7168, at 1 to 128 tokens: the choice is on average
// 2 %, at most 10 % slower than the best of all measured; the same count is used
// up to 1,024 tokens, where only the cases beside takes_stream were measured.)  A
// unit of this count is 2.35 ns, on top of 3.2 us.
double pick_stream(const F16GemmParams& q, bool gated, F16StreamParams& p, bool* two_per_sm) {
  const int kblocks = (q.k + 63) / 64, step = gated ? 32 : 16;
  const int token_tiles = (q.m + p.tn - 1) / p.tn;
  const int (*room)[4] = stream_room();
  double best = 0;
  p.rows = 0;
  for (int rows = 128; rows >= (p.w_mn ? 128 : 64); rows -= step) {
    const int cols = gated ? rows / 2 : rows;
    const int tiles = (q.n + cols - 1) / cols * token_tiles;
    for (int log2 = 0; log2 < 4 && (log2 == 0 || kblocks >= 2 << log2); ++log2) {
      const int blocks = (kblocks + (1 << log2) - 1) >> log2;
      const bool two = tiles > room[0][log2];
      if (two && log2 > 0 && blocks < 8) continue;
      const double waves = two ? 2 * ((tiles + room[1][log2] - 1) / room[1][log2]) : 1.08;
      const double cost = ((rows + p.tn / 3.0) * blocks + p.tn * rows / 32.0) * waves * (1 + 0.02 * log2);
      if (p.rows == 0 || cost < best) best = cost, p.rows = rows, p.cluster = 1 << log2, *two_per_sm = two;
    }
  }
  return 3.2 + 0.00235 * best;
}

template <int EPI>
int launch_stream_gemm(const F16GemmParams& q, F16StreamParams& p, bool two, const void* x, int64_t ldx, int x_mn, const void* w,
                       int64_t w_rows, int64_t ldw, int w_mn, bool bf16, cudaStream_t st) {
  constexpr bool gated = EPI == kEpiGated;
  p.m = q.m, p.n = q.n, p.k = q.k;
  p.x_mn = x_mn != 0;
  p.up_row = q.up_row, p.act = q.act, p.limit = q.limit, p.bias = q.bias;
  p.residual = q.residual, p.out = q.out;
  const int room = two ? kStreamSmem : kStreamSmemAlone;
  const int kblocks = (p.k + 63) / 64;
  const int width = gated ? p.rows / 2 : p.rows;
  p.row_tiles = (q.n + width - 1) / width;
  const int64_t ctas = static_cast<int64_t>(p.row_tiles) * ((q.m + p.tn - 1) / p.tn) * p.cluster;
  DSV4_REQUIRE(ctas < (1ll << 31), "product too large");
  const int x_groups = p.x_mn ? (p.tn + 63) / 64 : 1, w_groups = p.w_mn ? 2 : 1;
  p.x_atom = p.x_mn ? 8192 : p.tn * 128;
  p.w_atom = p.w_mn ? 8192 : p.rows * 128;
  const int block = p.x_atom * x_groups + p.w_atom * w_groups, fixed = 1024 + kStreamBarBytes;
  // two blocks a stage where three such stages fit
  p.atoms = kblocks >= 2 * p.cluster && 6 * block <= room - fixed ? 2 : 1;
  const int stage = p.atoms * block;
  p.x_stage = p.x_atom * x_groups * p.atoms;
  p.w_stage = p.w_atom * w_groups * p.atoms;
  p.stages = (room - fixed) / stage;
  if (p.stages > kStreamMaxStages) p.stages = kStreamMaxStages;
  while (fixed + stream_ring_bytes(p.stages, stage, p.atoms, p.x_atom) > room) --p.stages;
  p.ring_bytes = stream_ring_bytes(p.stages, stage, p.atoms, p.x_atom);
  const bool whole = p.k % 64 == 0;
  p.w_wide = !p.w_mn && whole, p.x_wide = !p.x_mn && whole;
  if (p.w_wide) {
    if (int r = encode_wide(&p.map_w, "b", w, w_rows, p.k, ldw, width, p.atoms, gated, bf16)) return r;
  } else {
    if (int r = encode_operand(&p.map_w, "b", w, w_rows, p.k, ldw, p.w_mn, width, bf16, 64 * p.atoms))
      return r;
  }
  if (p.x_wide) {
    if (int r = encode_wide(&p.map_x, "a", x, p.m, p.k, ldx, p.tn, p.atoms, false, bf16)) return r;
  } else {
    if (int r = encode_operand(&p.map_x, "a", x, p.m, p.k, ldx, p.x_mn, p.tn, bf16, 64 * p.atoms))
      return r;
  }
  const size_t smem = fixed + static_cast<size_t>(p.ring_bytes);
  const dim3 grid(static_cast<unsigned>(ctas));
  const unsigned cl = static_cast<unsigned>(p.cluster);
  if (bf16) {
    launch_cluster(&f16_stream_gemm_kernel<EPI, true>, grid, dim3(kStreamThreads), smem, st, cl, p);
  } else {
    launch_cluster(&f16_stream_gemm_kernel<EPI, false>, grid, dim3(kStreamThreads), smem, st, cl, p);
  }
  return check_launch("f16_stream_gemm_kernel");
}

// 32 KB of shared memory for two blocks; the rest of the SM's memory is L1, which
// holds the loads in flight (a block of 7168 -> 2048 -> 7168: 18.4 us, with all of it
// shared 30.7).
template <int EPI>
cudaError_t rows_attrs() {
  void* const fns[4] = {reinterpret_cast<void*>(&f16_rows_gemm_kernel<EPI, true, true>),
                        reinterpret_cast<void*>(&f16_rows_gemm_kernel<EPI, false, true>),
                        reinterpret_cast<void*>(&f16_rows_gemm_kernel<EPI, true, false>),
                        reinterpret_cast<void*>(&f16_rows_gemm_kernel<EPI, false, false>)};
  for (void* fn : fns) {
    const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributePreferredSharedMemoryCarveout, 14);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <int EPI>
cudaError_t stream_attrs() {
  void* const fns[2] = {reinterpret_cast<void*>(&f16_stream_gemm_kernel<EPI, true>),
                        reinterpret_cast<void*>(&f16_stream_gemm_kernel<EPI, false>)};
  for (void* fn : fns) {
    cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         kStreamSmemAlone);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(fn, cudaFuncAttributePreferredSharedMemoryCarveout,
                               cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

// The faster of the two products by the counts above (values before the
// activation are kept by the pair product only).  Up to 128 tokens stream nearly
// always; beyond that it is long contractions of few columns: 256 tokens 4096
// -> 1024 take 8.0 us streamed and 13.7 in pairs, 512 tokens 7168 -> 4096 37
// and 27.  (Fewest tokens: takes_rows.)
bool takes_stream(const F16GemmParams& q, bool gated, int w_mn, F16StreamParams& p, bool* two) {
  if (q.zbits != 0 || q.m > 1024) return false;
  p.tn = stream_tokens(q.m);
  p.w_mn = w_mn != 0;
  double pair_us = 0;
  pick_tn(q.m, q.n, q.k, gated, &pair_us);
  return pick_stream(q, gated, p, two) < pair_us;
}

bool aligned_rows(const void* x, int64_t ldx, const void* w, int64_t ldw) {
  return aligned16(x) && ldx % 8 == 0 && aligned16(w) && ldw % 8 == 0;
}

// Up to 8 tokens, both operands by rows: for one token 2048 x 2048 takes 3.3 us
// here and 5.1 streamed, 7168 x 2048 7.4 and 9.1, 4096 x 7168 11.7 and 12.8, a
// block of 7168 -> 2048 -> 7168 back to back 18.4 and 22.1.  Long rows of few
// columns leave most SMs without a block, so those are streamed (1000 x 4096,
// 63 blocks: 5.5 and 5.2; 256 x 7168, 16 blocks: 8.1 and 5.1) unless their
// alignment needs this product.
bool takes_rows(const F16GemmParams& q, bool gated, int x_mn, int w_mn, bool aligned) {
  if (q.m > kRowsMaxTokens || q.zbits != 0 || x_mn || w_mn) return false;
  const int64_t blocks = (static_cast<int64_t>(q.n) + (gated ? 7 : 15)) / (gated ? 8 : 16);
  return !aligned || q.k <= 2048 || 2 * blocks >= sm_count();
}

template <int EPI>
int launch_rows_gemm(const F16GemmParams& q, const void* x, int64_t ldx, const void* w, int64_t ldw,
                     bool bf16, cudaStream_t st) {
  DSV4_REQUIRE(aligned_to(x, 2) && aligned_to(w, 2), "a and b must be aligned to their elements");
  DSV4_REQUIRE(ldx >= q.k && ldw >= q.k, "row stride below k (%lld and %lld, k %d)",
               (long long)ldx, (long long)ldw, q.k);
  F16RowsParams p = {static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(w), ldx, ldw, q.m, q.n,
                     q.k, q.up_row, q.act, q.limit, q.bias, q.residual, q.out};
  constexpr int kCols = EPI == kEpiGated ? 8 : 16;
  const dim3 grid(static_cast<unsigned>((q.n + kCols - 1) / kCols));
  const bool aligned = aligned_rows(x, ldx, w, ldw);
  const auto go = [&](auto kernel) { launch_pdl(kernel, grid, dim3(kRowsThreads), 0, st, p); };
  if (aligned) bf16 ? go(&f16_rows_gemm_kernel<EPI, true, true>) : go(&f16_rows_gemm_kernel<EPI, false, true>);
  else bf16 ? go(&f16_rows_gemm_kernel<EPI, true, false>) : go(&f16_rows_gemm_kernel<EPI, false, false>);
  return check_launch("f16_rows_gemm_kernel");
}

constexpr int64_t kMaxDim = 1ll << 30;
constexpr float kNoLimit = std::numeric_limits<float>::infinity();

int check_common(int64_t m, int64_t n, int64_t k, int dtype, int act) {
  DSV4_REQUIRE(dtype == DSV4_BF16 || dtype == DSV4_F16, "dtype must be fp16 or bf16 (got %d)", dtype);
  DSV4_REQUIRE(m >= 0 && n >= 1 && k >= 1 && m < kMaxDim && n < kMaxDim && k < kMaxDim,
               "bad shape m=%lld n=%lld k=%lld", (long long)m, (long long)n, (long long)k);
  DSV4_REQUIRE(act >= kActNone && act <= kActGeluTanh, "unknown activation %d", act);
  return DSV4_OK;
}

int check_limit(int has_limit, float limit, float* out) {
  *out = kNoLimit;
  if (!has_limit) return DSV4_OK;
  DSV4_REQUIRE(limit > 0.f && limit < kNoLimit, "the clamp limit must be positive and finite");
  *out = limit;
  return DSV4_OK;
}

// kept values are moved by 16-byte pieces
int check_kept(const void* codes, int bits, const float* scales) {
  DSV4_REQUIRE(bits == 0 || bits == 8 || bits == 16, "z_bits must be 0, 8 or 16 (got %d)", bits);
  DSV4_REQUIRE((codes != nullptr) == (bits != 0) && (scales != nullptr) == (bits != 0),
               "z_codes, z_bits and z_scales go together");
  DSV4_REQUIRE(aligned16(codes), "codes must be 16-byte aligned");
  return DSV4_OK;
}

}  // namespace

// Loads the kernels that need no attribute, so that a first launch inside a
// stream capture finds all of them.
template <typename... Fns>
cudaError_t load_kernels(Fns... fns) {
  cudaError_t e = cudaSuccess;
  cudaFuncAttributes a;
  const auto one = [&](auto fn) {
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, reinterpret_cast<const void*>(fn));
  };
  (one(fns), ...);
  return e;
}

int feed_forward_init() {
  cudaError_t e = pair_attrs<kEpiLinear>();
  if (e == cudaSuccess) e = pair_attrs<kEpiGated>();
  if (e == cudaSuccess) e = pair_attrs<kEpiGatedBwd>();
  if (e == cudaSuccess) e = stream_attrs<kEpiLinear>();
  if (e == cudaSuccess) e = stream_attrs<kEpiGated>();
  if (e == cudaSuccess) e = query_stream_room();
  if (e == cudaSuccess) e = rows_attrs<kEpiLinear>();
  if (e == cudaSuccess) e = rows_attrs<kEpiGated>();
  if (e == cudaSuccess)
    e = load_kernels(&checkpoint_kernel<DSV4_F32, true>, &checkpoint_kernel<DSV4_F32, false>,
                     &checkpoint_kernel<DSV4_F16, true>, &checkpoint_kernel<DSV4_F16, false>,
                     &checkpoint_kernel<DSV4_BF16, true>, &checkpoint_kernel<DSV4_BF16, false>,
                     &restore_kernel<DSV4_F32, true>, &restore_kernel<DSV4_F32, false>,
                     &restore_kernel<DSV4_F16, true>, &restore_kernel<DSV4_F16, false>,
                     &restore_kernel<DSV4_BF16, true>, &restore_kernel<DSV4_BF16, false>,
                     &act_backward_kernel<true>, &act_backward_kernel<false>,
                     &column_sum_kernel<true>, &column_sum_kernel<false>, &pack_rows_kernel,
                     &pack_windows_kernel);
  if (e != cudaSuccess)
    return fail(DSV4_ERR_CUDA, "feed-forward kernels: %s", cudaGetErrorString(e));
  return DSV4_OK;
}

int feed_forward_status(int* status, int reset) {
  cudaError_t e = cudaMemcpyFromSymbol(status, g_device_status, sizeof(int));
  if (e != cudaSuccess) return fail(DSV4_ERR_CUDA, "read status: %s", cudaGetErrorString(e));
  if (reset && *status != 0) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_device_status, &zero, sizeof(int));
    if (e != cudaSuccess) return fail(DSV4_ERR_CUDA, "reset status: %s", cudaGetErrorString(e));
  }
  return DSV4_OK;
}

}  // namespace dsv4

using namespace dsv4;

extern "C" {

int dsv4_b200_dense_gemm(const void* a, int64_t lda, int a_mn, const void* b, int64_t ldb, int b_mn,
                         int64_t m, int64_t n, int64_t k, int dtype, const void* bias,
                         int activation, const void* residual, int64_t ldr, void* out, int64_t ldo,
                         void* z_codes, int z_bits, float* z_scales, void* stream) {
  if (int r = ensure_init()) return r;
  if (int r = check_common(m, n, k, dtype, activation)) return r;
  if (int r = check_kept(z_codes, z_bits, z_scales)) return r;
  if (m == 0) return DSV4_OK;
  DSV4_REQUIRE(a && b && out, "null pointer argument");
  DSV4_REQUIRE(aligned_to(bias, 2) && aligned_to(residual, 2) && aligned_to(out, 2) && aligned_to(z_scales, 4),
               "bias, residual, out and z_scales must be aligned to their elements");
  DSV4_REQUIRE(ldo >= n && (!residual || ldr >= n || ldr == 0), "row stride below n");
  F16GemmParams p = {};
  p.m = static_cast<int>(m), p.n = static_cast<int>(n), p.k = static_cast<int>(k);
  p.act = activation;
  p.limit = kNoLimit;
  p.bias = bias;
  p.residual = mat16(residual, ldr);
  p.out = mat16(out, ldo);
  p.zq = z_codes, p.zbits = z_bits, p.zs = z_scales, p.n32 = round_up(n, kGroup);
  if (takes_rows(p, false, a_mn, b_mn, aligned_rows(a, lda, b, ldb)))
    return launch_rows_gemm<kEpiLinear>(p, a, lda, b, ldb, dtype == DSV4_BF16, as_stream(stream));
  F16StreamParams few = {};
  bool two = false;
  if (takes_stream(p, false, b_mn, few, &two))
    return launch_stream_gemm<kEpiLinear>(p, few, two, a, lda, a_mn, b, n, ldb, b_mn, dtype == DSV4_BF16,
                                          as_stream(stream));
  return launch_pair_gemm<kEpiLinear>(p, a, lda, a_mn, b, n, ldb, b_mn, dtype == DSV4_BF16,
                                      as_stream(stream));
}

int dsv4_b200_gated_gemm(const void* x, int64_t ldx, int x_mn, const void* w13, int64_t ldw, int w_mn,
                         int64_t m, int64_t intermediate, int64_t k, int dtype, int activation,
                         int has_clamp, float clamp_limit, void* h, int64_t ldh, void* z_codes, int z_bits,
                         float* z_scales, void* stream) {
  if (int r = ensure_init()) return r;
  if (int r = check_common(m, 2 * intermediate, k, dtype, activation)) return r;
  if (int r = check_kept(z_codes, z_bits, z_scales)) return r;
  F16GemmParams p = {};
  if (int r = check_limit(has_clamp, clamp_limit, &p.limit)) return r;
  if (m == 0) return DSV4_OK;
  DSV4_REQUIRE(x && w13 && h, "null pointer argument");
  DSV4_REQUIRE(aligned_to(h, 2) && aligned_to(z_scales, 4), "h and z_scales must be aligned to their elements");
  DSV4_REQUIRE(ldh >= intermediate, "row stride below the row");
  // a TMA box starts at a multiple of 16 bytes
  DSV4_REQUIRE(!w_mn || intermediate % 8 == 0,
               "w13 stored by columns needs intermediate to be a multiple of 8 (got %lld)",
               (long long)intermediate);
  p.m = static_cast<int>(m), p.n = static_cast<int>(intermediate), p.k = static_cast<int>(k);
  p.act = activation;
  p.up_row = p.n;
  p.out = mat16(h, ldh);
  p.zq = z_codes, p.zbits = z_bits, p.zs = z_scales, p.n32 = round_up(intermediate, kGroup);
  if (takes_rows(p, true, x_mn, w_mn, aligned_rows(x, ldx, w13, ldw)))
    return launch_rows_gemm<kEpiGated>(p, x, ldx, w13, ldw, dtype == DSV4_BF16, as_stream(stream));
  F16StreamParams few = {};
  bool two = false;
  if (takes_stream(p, true, w_mn, few, &two))
    return launch_stream_gemm<kEpiGated>(p, few, two, x, ldx, x_mn, w13, 2 * intermediate, ldw, w_mn,
                                         dtype == DSV4_BF16, as_stream(stream));
  return launch_pair_gemm<kEpiGated>(p, x, ldx, x_mn, w13, 2 * intermediate, ldw, w_mn,
                                     dtype == DSV4_BF16, as_stream(stream));
}

int dsv4_b200_gated_feed_forward(const void* x, int64_t ldx, int x_mn, const void* w13, int64_t ldw13,
                                 int w13_mn, const void* w2, int64_t ldw2, int w2_mn, int64_t m,
                                 int64_t hidden, int64_t intermediate, int64_t out_cols, int dtype,
                                 int activation, int has_clamp, float clamp_limit,
                                 const void* residual, int64_t ldr, void* h, int64_t ldh, void* out,
                                 int64_t ldo, void* z_codes, int z_bits, float* z_scales,
                                 int8_t* x_codes, float* x_scales, void* stream) {
  if (x_codes != nullptr) {
    DSV4_REQUIRE(!x_mn, "x is kept in 8 bits by rows");
    if (int r = dsv4_b200_checkpoint_int8(x, dtype, m, hidden, ldx, x_codes, x_scales, stream)) return r;
  }
  if (int r = dsv4_b200_gated_gemm(x, ldx, x_mn, w13, ldw13, w13_mn, m, intermediate, hidden, dtype,
                                   activation, has_clamp, clamp_limit, h, ldh, z_codes, z_bits,
                                   z_scales, stream))
    return r;
  return dsv4_b200_dense_gemm(h, ldh, 0, w2, ldw2, w2_mn, m, out_cols, intermediate, dtype, nullptr,
                              DSV4_ACT_NONE, residual, ldr, out, ldo, nullptr, 0, nullptr, stream);
}

int dsv4_b200_gated_backward_gemm(const void* dy, int64_t lddy, int dy_mn, const void* w2,
                                  int64_t ldw, int w_mn, int64_t m, int64_t intermediate, int64_t k,
                                  int dtype, int activation, int has_clamp, float clamp_limit,
                                  const void* z_codes, int z_bits, const float* z_scales, void* dz, int64_t lddz, void* h, int64_t ldh,
                                  void* stream) {
  if (int r = ensure_init()) return r;
  if (int r = check_common(m, 2 * intermediate, k, dtype, activation)) return r;
  if (int r = check_kept(z_codes, z_bits, z_scales)) return r;
  F16GemmParams p = {};
  if (int r = check_limit(has_clamp, clamp_limit, &p.limit)) return r;
  if (m == 0) return DSV4_OK;
  DSV4_REQUIRE(dy && w2 && dz, "null pointer argument");
  DSV4_REQUIRE(aligned_to(dz, 2) && aligned_to(h, 2) && aligned_to(z_scales, 4),
               "dz, h and z_scales must be aligned to their elements");
  DSV4_REQUIRE(z_bits != 0, "the kept g and u are needed");
  DSV4_REQUIRE(lddz >= 2 * intermediate && (!h || ldh >= intermediate), "row stride below the row");
  p.m = static_cast<int>(m), p.n = static_cast<int>(intermediate), p.k = static_cast<int>(k);
  p.act = activation;
  p.out = mat16(h, ldh);
  p.d0 = mat16(dz, lddz), p.d1 = mat16(static_cast<const uint16_t*>(dz) + intermediate, lddz);
  p.zq = const_cast<void*>(z_codes), p.zbits = z_bits, p.zs = const_cast<float*>(z_scales);
  p.n32 = round_up(intermediate, kGroup);
  return launch_pair_gemm<kEpiGatedBwd>(p, dy, lddy, dy_mn, w2, intermediate, ldw, w_mn,
                                        dtype == DSV4_BF16, as_stream(stream));
}

int dsv4_b200_checkpoint_int8(const void* x, int dtype, int64_t m, int64_t k, int64_t ldx,
                              int8_t* codes, float* scales, void* stream) {
  if (int r = ensure_init()) return r;
  DSV4_REQUIRE(dtype == DSV4_F32 || dtype == DSV4_F16 || dtype == DSV4_BF16, "unknown dtype %d", dtype);
  DSV4_REQUIRE(m >= 0 && k >= 1 && m < kMaxDim && k < kMaxDim && (ldx >= k || m <= 1),
               "bad shape m=%lld k=%lld ldx=%lld", (long long)m, (long long)k, (long long)ldx);
  if (m == 0) return DSV4_OK;
  DSV4_REQUIRE(x && codes && scales, "null pointer argument");
  DSV4_REQUIRE(aligned16(codes), "codes must be 16-byte aligned");
  DSV4_REQUIRE(aligned_to(x, dtype == DSV4_F32 ? 4 : 2) && aligned_to(scales, 4),
               "x and scales must be aligned to their elements");
  const int64_t k32 = round_up(k, kGroup), cb = (k32 + 255) / 256, blocks = (m + 31) / 32 * cb;
  DSV4_REQUIRE(blocks < (1ll << 31), "checkpoint too large");
  const int per = dtype == DSV4_F32 ? 4 : 8;
  const bool vec = aligned16(x) && ldx % per == 0;
  const dim3 grid(static_cast<unsigned>(blocks));
  cudaStream_t st = as_stream(stream);
  const auto go = [&](auto kernel) {
    launch_pdl(kernel, grid, dim3(256), 0, st, x, ldx, m, k, k32, static_cast<uint32_t>(cb), codes,
               scales);
  };
  if (dtype == DSV4_F32) vec ? go(&checkpoint_kernel<DSV4_F32, true>) : go(&checkpoint_kernel<DSV4_F32, false>);
  else if (dtype == DSV4_F16) vec ? go(&checkpoint_kernel<DSV4_F16, true>) : go(&checkpoint_kernel<DSV4_F16, false>);
  else vec ? go(&checkpoint_kernel<DSV4_BF16, true>) : go(&checkpoint_kernel<DSV4_BF16, false>);
  return check_launch("checkpoint_kernel");
}

int dsv4_b200_restore_int8(const int8_t* codes, const float* scales, int64_t m, int64_t k, void* out,
                           int dtype, int64_t ldo, void* stream) {
  if (int r = ensure_init()) return r;
  DSV4_REQUIRE(dtype == DSV4_F32 || dtype == DSV4_F16 || dtype == DSV4_BF16, "unknown dtype %d", dtype);
  DSV4_REQUIRE(m >= 0 && k >= 1 && m < kMaxDim && k < kMaxDim && ldo >= k,
               "bad shape m=%lld k=%lld ldo=%lld", (long long)m, (long long)k, (long long)ldo);
  if (m == 0) return DSV4_OK;
  DSV4_REQUIRE(out && codes && scales, "null pointer argument");
  DSV4_REQUIRE(aligned16(codes), "codes must be 16-byte aligned");
  DSV4_REQUIRE(aligned_to(out, dtype == DSV4_F32 ? 4 : 2) && aligned_to(scales, 4),
               "out and scales must be aligned to their elements");
  const int64_t k32 = round_up(k, kGroup), cb = (k32 + 255) / 256, blocks = (m + 31) / 32 * cb;
  DSV4_REQUIRE(blocks < (1ll << 31), "checkpoint too large");
  const int per = dtype == DSV4_F32 ? 4 : 8;
  const bool vec = aligned16(out) && ldo % per == 0;
  const dim3 grid(static_cast<unsigned>(blocks));
  cudaStream_t st = as_stream(stream);
  const auto go = [&](auto kernel) {
    launch_pdl(kernel, grid, dim3(256), 0, st, codes, scales, m, k, k32, static_cast<uint32_t>(cb), out, ldo);
  };
  if (dtype == DSV4_F32) vec ? go(&restore_kernel<DSV4_F32, true>) : go(&restore_kernel<DSV4_F32, false>);
  else if (dtype == DSV4_F16) vec ? go(&restore_kernel<DSV4_F16, true>) : go(&restore_kernel<DSV4_F16, false>);
  else vec ? go(&restore_kernel<DSV4_BF16, true>) : go(&restore_kernel<DSV4_BF16, false>);
  return check_launch("restore_kernel");
}

int dsv4_b200_act_backward_slabs(int64_t m, int64_t n, int64_t* slabs) {
  DSV4_REQUIRE(slabs != nullptr, "slabs is null");
  DSV4_REQUIRE(m >= 0 && n >= 1 && m < kMaxDim && n < kMaxDim, "bad shape m=%lld n=%lld", (long long)m,
               (long long)n);
  // four blocks per SM, of at least 32 rows
  const int64_t cols = (n + 255) / 256;
  int64_t s = 4 * 148 / cols;
  if (s > (m + 31) / 32) s = (m + 31) / 32;
  *slabs = s < 1 ? 1 : s;
  return DSV4_OK;
}

int dsv4_b200_act_backward(const void* dy, int64_t lddy, const void* z_codes, int z_bits,
                           const float* z_scales, int64_t m, int64_t n,
                           int dtype, int activation, void* dz, int64_t lddz, float* partial,
                           int64_t slabs, void* dbias, void* stream) {
  if (int r = ensure_init()) return r;
  if (int r = check_common(m, n, 1, dtype, activation)) return r;
  if (int r = check_kept(z_codes, z_bits, z_scales)) return r;
  int64_t need = 0;
  if (int r = dsv4_b200_act_backward_slabs(m, n, &need)) return r;
  DSV4_REQUIRE((dbias == nullptr) == (partial == nullptr), "dbias and its workspace go together");
  DSV4_REQUIRE(!dbias || slabs >= need, "workspace of %lld slabs, %lld needed", (long long)slabs,
               (long long)need);
  DSV4_REQUIRE(activation == kActNone || m == 0 ||
                   (dz && lddz >= n && z_bits != 0), "an activation needs dz and the kept z");
  DSV4_REQUIRE(m == 0 || (dy && (lddy >= n || m == 1)), "bad dy");
  DSV4_REQUIRE(need < 65536, "too many rows");
  DSV4_REQUIRE(aligned_to(dy, 2) && aligned_to(dz, 2) && aligned_to(dbias, 2) && aligned_to(z_scales, 4) &&
                   aligned_to(partial, 4), "pointers must be aligned to their elements");
  cudaStream_t st = as_stream(stream);
  ActBackward p = {};
  p.dy = dy, p.lddy = lddy, p.vec_dy = mat16(dy, lddy).vec;
  p.zq = z_codes, p.zbits = z_bits, p.zs = z_scales, p.n32 = round_up(n, kGroup);
  p.dz = dz, p.lddz = lddz, p.vec_dz = mat16(dz, lddz).vec;
  p.partial = partial;
  p.m = m, p.n = n, p.act = activation;
  p.slab_rows = (m + need - 1) / need;
  const dim3 grid(static_cast<unsigned>((n + 255) / 256), static_cast<unsigned>(need));
  const dim3 sum_grid(static_cast<unsigned>((n + 31) / 32));
  const bool bf16 = dtype == DSV4_BF16;
  if (activation != kActNone || dbias) {
    if (m == 0 && !dbias) return DSV4_OK;
    if (bf16) launch_pdl(&act_backward_kernel<true>, grid, dim3(256), 0, st, p);
    else launch_pdl(&act_backward_kernel<false>, grid, dim3(256), 0, st, p);
    if (int r = check_launch("act_backward_kernel")) return r;
  }
  if (dbias) {
    if (bf16) launch_pdl(&column_sum_kernel<true>, sum_grid, dim3(256), 0, st, partial, need, n, dbias);
    else launch_pdl(&column_sum_kernel<false>, sum_grid, dim3(256), 0, st, partial, need, n, dbias);
    return check_launch("column_sum_kernel");
  }
  return DSV4_OK;
}

// dW = d^T x, with x as it is or restored from its 8-bit codes first: rounded to
// 16 bits, 2^-8 (fp16 2^-11) of a value that the codes hold to amax / 254.
static int weight_gradient(const void* d, int64_t ldd, int d_mn, const void* x, int64_t ldx, int x_mn,
                           const int8_t* x_codes, const float* x_scales, void* x_restored,
                           int64_t ldxr, int64_t rows, int64_t cols, int64_t m, int dtype, void* dw,
                           void* stream) {
  if (x_codes != nullptr) {
    if (int r = dsv4_b200_restore_int8(x_codes, x_scales, m, cols, x_restored, dtype, ldxr, stream))
      return r;
    x = x_restored, ldx = ldxr, x_mn = 0;
  }
  return dsv4_b200_dense_gemm(d, ldd, !d_mn, x, ldx, !x_mn, rows, cols, m, dtype, nullptr,
                              DSV4_ACT_NONE, nullptr, 0, dw, cols, nullptr, 0, nullptr, stream);
}

int dsv4_b200_gated_feed_forward_backward(
    const void* dy, int64_t lddy, int dy_mn, const void* x, int64_t ldx, int x_mn,
    const int8_t* x_codes, const float* x_scales, void* x_restored, int64_t ldxr, const void* w13,
    int64_t ldw13, int w13_mn, const void* w2, int64_t ldw2, int w2_mn, int64_t m, int64_t hidden,
    int64_t intermediate, int64_t out_cols, int dtype, int activation, int has_clamp,
    float clamp_limit, const void* z_codes, int z_bits, const float* z_scales, void* h, int64_t ldh,
    int form_h, void* dz, int64_t lddz, void* dx, void* dw13, void* dw2, void* stream) {
  if (m == 0) return DSV4_OK;
  if (dx != nullptr || dw13 != nullptr || (dw2 != nullptr && form_h)) {
    if (int r = dsv4_b200_gated_backward_gemm(dy, lddy, dy_mn, w2, ldw2, !w2_mn, m, intermediate,
                                              out_cols, dtype, activation, has_clamp, clamp_limit,
                                              z_codes, z_bits, z_scales, dz, lddz,
                                              form_h ? h : nullptr, ldh, stream))
      return r;
  }
  if (dw2 != nullptr) {
    if (int r = dsv4_b200_dense_gemm(dy, lddy, !dy_mn, h, ldh, 1, out_cols, intermediate, m, dtype,
                                     nullptr, DSV4_ACT_NONE, nullptr, 0, dw2, intermediate, nullptr, 0,
                                     nullptr, stream))
      return r;
  }
  if (dx != nullptr) {
    if (int r = dsv4_b200_dense_gemm(dz, lddz, 0, w13, ldw13, !w13_mn, m, hidden, 2 * intermediate,
                                     dtype, nullptr, DSV4_ACT_NONE, nullptr, 0, dx, hidden, nullptr, 0,
                                     nullptr, stream))
      return r;
  }
  if (dw13 != nullptr)
    return weight_gradient(dz, lddz, 0, x, ldx, x_mn, x_codes, x_scales, x_restored, ldxr,
                           2 * intermediate, hidden, m, dtype, dw13, stream);
  return DSV4_OK;
}

int dsv4_b200_dense_backward(const void* dy, int64_t lddy, const void* d, int64_t ldd, int d_mn,
                             const void* x, int64_t ldx, int x_mn, const int8_t* x_codes,
                             const float* x_scales, void* x_restored, int64_t ldxr, const void* w,
                             int64_t ldw, int w_mn, int64_t m, int64_t n, int64_t k, int dtype,
                             int activation, const void* z_codes, int z_bits, const float* z_scales,
                             float* partial, int64_t slabs, void* dx, void* dw, void* dbias,
                             void* stream) {
  if (m == 0) return DSV4_OK;
  if (activation != DSV4_ACT_NONE || dbias != nullptr) {
    DSV4_REQUIRE(activation == DSV4_ACT_NONE || !d_mn, "dz is written by rows");
    if (int r = dsv4_b200_act_backward(dy, lddy, z_codes, z_bits, z_scales, m, n, dtype, activation,
                                       activation == DSV4_ACT_NONE ? nullptr : const_cast<void*>(d),
                                       ldd, partial, slabs, dbias, stream))
      return r;
  }
  if (dx != nullptr) {
    if (int r = dsv4_b200_dense_gemm(d, ldd, d_mn, w, ldw, !w_mn, m, k, n, dtype, nullptr,
                                     DSV4_ACT_NONE, nullptr, 0, dx, k, nullptr, 0, nullptr, stream))
      return r;
  }
  if (dw != nullptr)
    return weight_gradient(d, ldd, d_mn, x, ldx, x_mn, x_codes, x_scales, x_restored, ldxr, n, k, m,
                           dtype, dw, stream);
  return DSV4_OK;
}

int dsv4_b200_pack_rows(const void* in, int64_t row_stride, int64_t col_stride, int64_t rows,
                        int64_t cols, void* out, int64_t ldo, void* stream) {
  if (int r = ensure_init()) return r;
  DSV4_REQUIRE(rows >= 0 && cols >= 0 && rows < kMaxDim && cols < kMaxDim && row_stride >= 0 &&
                   col_stride >= 0 && ldo >= cols, "bad shape");
  if (rows == 0 || cols == 0) return DSV4_OK;
  DSV4_REQUIRE(in && out, "null pointer argument");
  DSV4_REQUIRE(aligned_to(in, 2) && aligned_to(out, 2), "in and out must be aligned to their elements");
  const bool windows = col_stride == 1 && (row_stride >= cols || rows == 1) && aligned16(out) && ldo % 8 == 0;
  const int64_t width = windows ? 256 : 32, cb = (cols + width - 1) / width, blocks = (rows + 31) / 32 * cb;
  DSV4_REQUIRE(blocks < (1ll << 31), "matrix too large");
  if (windows) {
    launch_pdl(&pack_windows_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, as_stream(stream),
               static_cast<const uint16_t*>(in), row_stride, rows, cols, static_cast<uint32_t>(cb),
               static_cast<uint16_t*>(out), ldo);
    return check_launch("pack_windows_kernel");
  }
  launch_pdl(&pack_rows_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, as_stream(stream),
             static_cast<const uint16_t*>(in), row_stride, col_stride, rows, cols,
             static_cast<uint32_t>(cb),
             static_cast<uint16_t*>(out), ldo);
  return check_launch("pack_rows_kernel");
}

}  // extern "C"
