// Entry points of the few-query attention kernels (structure_attention_few.cu).
#pragma once

#include "structure_attention.cuh"

namespace y3b {

constexpr int kFewQueries = 2;  // queries of a structure, at most

struct AttItem;

// Partial results: one row of `width` floats per (slot, head, query), at ((slot * H + head) * kFewQueries + query) *
// width.  Forward: O [DP], m, l.  Query side: sum dS K [DP], the ten sums of the tile kernels and delta0
// [16], sum P K [DP].
template <typename T>
int attention_few_forward(const AttArgs& a, const AttItem* items, int64_t count, int DP, int width, float* part,
                          cudaStream_t s);

template <typename T>
int attention_few_query(const AttArgs& a, const AttItem* items, int64_t count, int DP, int width, const T* out,
                        const T* grad, const float* lse, float* part, cudaStream_t s);

// dk, dv and the position parts of the keys of `items` (rows: up to kTileRows keys of one structure, columns: its one to
// kFewQueries queries).
template <typename T>
int attention_few_key(const AttArgs& a, const AttItem* items, int64_t count, const T* grad, const float* lse,
                      const float* delta, T* dk, T* dv, float* dy_part, cudaStream_t s);

}  // namespace y3b
