// What the block operators share: element types, warp reductions and the
// checks of their C entries.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "pm_capi.h"
#include "pmb200_blocks.h"

namespace pm {
namespace blk {

using bf16 = __nv_bfloat16;
using fp16 = __half;

template <class T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<bf16>(bf16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float<fp16>(fp16 v) { return __half2float(v); }

template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 from_float<bf16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ fp16 from_float<fp16>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the CTA, the same on every thread; `red` holds 32 floats and may be
// reused by the next call only with another buffer in between.
__device__ __forceinline__ float cta_sum(float v, float* red) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int warps = blockDim.x >> 5;
  float r = 0.0f;
  for (int w = 0; w < warps; ++w) r += red[w];
  return r;
}

inline size_t type_bytes(int dtype) { return dtype == PM_DT_F32 ? 4 : 2; }
inline bool known_type(int dtype) { return dtype == PM_DT_F32 || dtype == PM_DT_BF16 || dtype == PM_DT_F16; }
inline bool aligned(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// SMs of the current device, remembered per ordinal; PM_E_* when there is none.
int sm_count(int* sms);

}  // namespace blk
}  // namespace pm
