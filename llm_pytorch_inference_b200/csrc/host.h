// Host-side helpers shared by the C-ABI entry points.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <utility>

#include "../../include/mvb200.h"
#include "per_device.h"

namespace mvb {

// Records `msg` as this thread's last error and returns `code`.
int fail(int code, const char* fmt, ...);

// Returns MVB_ERR_CUDA with the CUDA error string when `e` is an error, else MVB_OK.
int cuda_status(cudaError_t e, const char* what);

// Device address of the status word on the current device (looked up once per device).
unsigned* device_status_ptr();

// SM count of the current device (cached per device).
int current_sm_count();

// Programmatic-dependent-launch switch (mvb_set_pdl).
bool pdl_enabled();

// cuTensorMapEncodeTiled through the runtime's driver entry point (no -lcuda needed).
int encode_tiled(CUtensorMap* map, CUtensorMapDataType dtype, uint32_t rank, const void* base,
                 const uint64_t* dims, const uint64_t* strides_bytes, const uint32_t* box, CUtensorMapSwizzle swz);

inline size_t dtype_size(int dtype) {
  switch (dtype) {
    case MVB_F32: return 4;
    case MVB_F16: return 2;
    case MVB_BF16: return 2;
    case MVB_I32: return 4;
    case MVB_I64: return 8;
    default: return 0;
  }
}

inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// Launch `kernel` with the PDL attribute when enabled.
template <typename... KArgs, typename... Args>
int launch(const char* name, void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
           Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  cfg.attrs = attr;
  cfg.numAttrs = 0;
  if (pdl_enabled()) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
  }
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
  return cuda_status(e, name);
}

// Launch `kernel` as the dependent of the launch just before it in the same entry point: always with
// the PDL attribute.  It may start while that kernel still runs and waits for it (griddepcontrol.wait)
// before it reads or writes anything.
template <typename... KArgs, typename... Args>
int launch_dependent(const char* name, void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem,
                     cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
  return cuda_status(e, name);
}

// Launch with a (cluster_x, 1, 1) thread-block cluster, plus the PDL attribute when enabled.
template <typename... KArgs, typename... Args>
int launch_cluster(const char* name, void (*kernel)(KArgs...), dim3 grid, dim3 block, unsigned cluster_x,
                   size_t smem, cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster_x;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (pdl_enabled()) {
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
  }
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
  return cuda_status(e, name);
}

// Opt a kernel into more than 48 KB of dynamic shared memory (idempotent).
template <typename... KArgs>
int set_smem(void (*kernel)(KArgs...), size_t bytes, const char* name) {
  cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  return cuda_status(e, name);
}

// The same, asked of the driver once per kernel and device: `done` is a static of the call site, a bit per device.
template <typename... KArgs>
int set_smem_once(std::atomic<uint64_t>& done, void (*kernel)(KArgs...), size_t bytes, const char* name) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return set_smem(kernel, bytes, name);
  if (done.load(std::memory_order_acquire) >> dev & 1u) return MVB_OK;
  const int rc = set_smem(kernel, bytes, name);
  if (rc == MVB_OK) done.fetch_or(uint64_t(1) << dev, std::memory_order_release);
  return rc;
}

// Clusters of `cluster` blocks of `kernel` that the current device holds at once.  They lie within its groups of SMs, so that
// larger ones leave SMs over (on B200, one block an SM: 74 of 2, 45 of 3, 33 of 4, 15 of 8).  Asked of the driver once per
// kernel, size and device: `known` is a static of the call site.  Where the driver does not say, 1 is taken for this call.
template <typename... KArgs>
int clusters_at_once(PerDevice& known, void (*kernel)(KArgs...), int cluster, int threads, size_t smem) {
  int device = -1;
  if (cudaGetDevice(&device) != cudaSuccess) device = -1;
  auto ask = [&] {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(cluster));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
      cudaGetLastError();
      n = 0;
    }
    return n;
  };
  return known.get(device, ask, 1);
}

}  // namespace mvb

#define MVB_REQUIRE(cond, ...)                                      \
  do {                                                              \
    if (!(cond)) return ::mvb::fail(MVB_ERR_INVALID_ARG, __VA_ARGS__); \
  } while (0)

#define MVB_TRY(expr)               \
  do {                              \
    int _mvb_rc = (expr);           \
    if (_mvb_rc != MVB_OK) return _mvb_rc; \
  } while (0)
