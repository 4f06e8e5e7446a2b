// What the C entries of the operators share: refusals, the GPU's size, launches.
#pragma once
#include <cstdint>
#include <cstdio>

#include "../../include/ocrvl_cuda.h"
#include "capi.h"

namespace ocrvl {

inline int invalid(const char *msg) { return api_fail(OCRVL_E_INVALID, msg); }

inline int cuda_fail(const char *what, cudaError_t e) {
  char msg[256];
  snprintf(msg, sizeof(msg), "%s: %s", what, cudaGetErrorString(e));
  return api_fail(OCRVL_E_CUDA, msg);
}

#define PCK(call)                                        \
  do {                                                   \
    cudaError_t e_ = (call);                             \
    if (e_ != cudaSuccess) return cuda_fail(#call, e_);  \
  } while (0)

inline int elem_bytes(int type) { return type == OCRVL_F32 ? 4 : type == OCRVL_F16 || type == OCRVL_BF16 ? 2 : 0; }

inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

inline int log2i(int x) {
  int n = 0;
  while (1 << n < x) n++;
  return n;
}

// The streaming multiprocessors of the current device.
inline int sm_count(int *out) {
  static int known[64];  // 0: not asked yet (a race stores the same value twice)
  int dev = 0;
  PCK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return invalid("device index out of range");
  if (!known[dev]) {
    int n = 0;
    PCK(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
    known[dev] = n;
  }
  *out = known[dev];
  return OCRVL_OK;
}

// Blocks that run at once in clusters of up to eight, one an SM: clusters lie within
// one of the GPU's partitions, so some SMs stay over (15 clusters of eight
// were resident on 148 SMs).
inline int cluster_room(int sms) { return sms * 4 / 5; }

// Bytes of dynamic shared memory: of this call, and the most that any call of
// the kernel takes.  The limit that a kernel has leave for is shared by all host threads, so it
// is always set to the same value.
struct Smem {
  int bytes, most;
  Smem(int all) : bytes(all), most(all) {}
  Smem(int bytes_, int most_) : bytes(bytes_), most(most_) {}
};

// Launches with dynamic shared memory; dependent: may start
// before the kernel launched just before it on the stream ends (both wait for
// it with griddepcontrol).
template <typename... Params, typename... Args>
int launch(const char *name, void (*kernel)(Params...), dim3 grid, int threads, Smem smem, cudaStream_t stream, bool dependent,
           int cluster, Args... args) {
  if (smem.bytes > 24 * 1024) {  // with a kernel's static share possibly past the 48 KB that need no leave
    cudaError_t e = cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem.most);
    if (e != cudaSuccess) return cuda_fail(name, e);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem.bytes;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (dependent) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = cluster;
    at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
    n++;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  return e == cudaSuccess ? OCRVL_OK : cuda_fail(name, e);
}

}  // namespace ocrvl
