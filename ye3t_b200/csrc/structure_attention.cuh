// Shared parts of the structure-attention kernels.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace y3b {

constexpr int kAttMaxWidth = 128;
constexpr float kLog2e = 1.44269504088896340736f;

// The arguments of one call as the kernels see them (strides in elements).
struct AttArgs {
  int H, Hk, D, group;  // group = H / Hk
  int64_t nq, nk;
  const void* q;
  const void* k;
  const void* v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  const float* x;       // query positions [nq, 3] or null
  const float* y;       // key positions [nk, 3]
  const float* slopes;  // [H]
  float scale2;         // scale * log2(e)
  float scale;
  const int32_t* q_off;  // [S + 1]
  const int32_t* k_off;  // [S + 1]
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

}  // namespace y3b
