// Entry points of the small-structure attention kernels (structure_attention_small.cu).
#pragma once

#include "structure_attention.cuh"

namespace y3b {

// One structure: first query, queries, first key, keys (up to 64 of each).
struct alignas(16) AttSmall {
  int q, nq, k, nk;
};

// `list` holds the structures of up to 32 queries and keys, then those of up to 64.
template <typename T>
int attention_small_forward(const AttArgs& a, const AttSmall* list, int64_t up_to_32, int64_t up_to_64, T* out,
                            float* lse, cudaStream_t s);

template <typename T>
int attention_small_backward(const AttArgs& a, const AttSmall* list, int64_t up_to_32, int64_t up_to_64, const T* grad,
                             T* dq, T* dk, T* dv, float* slope_part, float* dx_part, float* dy_part, cudaStream_t s);

}  // namespace y3b
