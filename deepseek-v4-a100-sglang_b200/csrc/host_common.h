// Host side shared by the translation units of libdsv4_b200.so (not exported):
// error reporting, launches, tensor-map encoding, per-device set-up.
#pragma once

#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <cstdlib>
#include <cstring>
#include <utility>

#include "dsv4_b200.h"

namespace dsv4 {

// Stores the message for dsv4_b200_last_error() and returns `code`.
int fail(int code, const char* fmt, ...);
int check_launch(const char* what);
bool pdl_enabled();
int ensure_init();
int sm_count();
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();

// feed_forward.cu: kernel attributes and status word of its kernels
int feed_forward_init();
int feed_forward_status(int* status, int reset);

#define DSV4_REQUIRE(cond, ...) \
  do {                          \
    if (!(cond)) return fail(DSV4_ERR_INVALID_ARGUMENT, __VA_ARGS__); \
  } while (0)

inline cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }

template <typename... KArgs, typename... Args>
void launch_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  // errors surface through cudaGetLastError in check_launch
  (void)cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

// Launch in clusters of `cluster` CTAs along x, with programmatic dependent
// launch as launch_pdl.
template <typename... KArgs, typename... Args>
void launch_cluster(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                    unsigned cluster, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  (void)cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

}  // namespace dsv4
