// dc_cache.cuh -- what the cache operators share: types and the launch.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "dc_internal.cuh"
#include "dc_ptx.cuh"
#include "dc_span.h"

namespace dcc {

static inline bool is_type(int t) { return t == DC_F32 || t == DC_F16 || t == DC_BF16; }
static inline bool is_half(int t) { return t == DC_F16 || t == DC_BF16; }
static inline int elem_size(int t) { return t == DC_F32 ? 4 : 2; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// A call may come while another device is current: launches and kernel
// attributes belong to the context's own.
struct DeviceGuard {
  int old = -1;
  int enter(dc_ctx* ctx) {
    int cur = -1;
    DC_CUDA(ctx, cudaGetDevice(&cur));
    if (cur != ctx->device) {
      DC_CUDA(ctx, cudaSetDevice(ctx->device));
      old = cur;
    }
    return DC_OK;
  }
  ~DeviceGuard() {
    if (old >= 0) cudaSetDevice(old);
  }
};

// One launch on the context's stream, in clusters of `cluster` blocks along x, as a
// programmatic dependent of what runs before: it may begin while that still runs, so a
// kernel executes griddepcontrol.wait before it touches memory.  The exceptions are
// k_own and k_join of dc_prefix.cu where they are launched `behind` the kernel of the
// same call before them; the comments there say which earlier wait covers what they
// touch and which later one their end.  They may follow no other kernel in that form.
template <typename... P, typename... A>
static int launch(dc_ctx* ctx, void (*kern)(P...), dim3 grid, int threads, int smem, int cluster, const A&... args) {
  if (int rc = dc_set_smem(ctx, (const void*)kern, smem)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 1;
  if (cluster > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  cfg.attrs = attr;
  DC_CUDA(ctx, cudaLaunchKernelEx(&cfg, kern, args...));
  dc_count_launch();
  return DC_OK;
}

}  // namespace dcc
