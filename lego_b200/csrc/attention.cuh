// Shared by the attention kernels: the problem as the device sees it, which key a query
// sees, and the score's cap and distance bias.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace lego {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct AttnProblem {
  int batch, q_len, k_len, q_heads, k_heads, dim, group;   // group: query heads of one key head
  int offset;                                              // position of query 0: k_len - q_len
  int causal;
  float scale, softcap;
  long long q_stride[3], k_stride[3], v_stride[3];         // batch, token, head, in elements
  const float* slopes;
  const int* prefix;
  const int* documents;
};

__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ void from_f32(float v, __half* o) { *o = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16* o) { *o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f32(float v, float* o) { *o = v; }

// Refuses what the attention kernels do not take and fills in the device's view of the rest.
int32_t attention_problem(const lego_attention_t* d, AttnProblem* out);

}  // namespace lego
