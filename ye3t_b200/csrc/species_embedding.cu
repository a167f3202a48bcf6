// Learned per-species vectors: lookup with scaling and the table's gradient.
//
//   out[i, c]   = scale * table[z_i, c]
//   dtable[v, c] = scale * sum_{i : z_i = v} grad[i, c]
//
// The lookup is one pass over the output; the gradient orders the atoms by species
// (stable radix sort of the indices) and sums runs of equal species, so that no
// floating-point atomics are needed and results are bitwise repeatable.
#include <cuda_bf16.h>

#include <algorithm>

#include "common.cuh"

namespace y3b {
namespace {

template <typename T> struct Acc { using type = float; };
template <> struct Acc<double> { using type = double; };

template <typename T> __device__ __forceinline__ typename Acc<T>::type widen(T v) { return v; }
template <> __device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T narrow(typename Acc<T>::type v) { return T(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Pack { T v[VEC]; };

// A species of either integer width, -1 when it is outside [0, V).
template <typename I>
__device__ __forceinline__ int64_t species_at(const I* z, int64_t i, int64_t V) {
  const int64_t s = int64_t(z[i]);
  return s >= 0 && s < V ? s : -1;
}

// One thread per VEC consecutive channels of one atom; consecutive threads write
// consecutive addresses.  Bound by the output's store: the table stays in L2.
template <typename T, typename I, int VEC>
__global__ void __launch_bounds__(256) embedding_kernel(const T* __restrict__ table, int64_t V, int C,
                                                        const I* __restrict__ z, int64_t N,
                                                        typename Acc<T>::type scale, T* __restrict__ out,
                                                        int32_t* status) {
  using P = Pack<T, VEC>;
  const int per_row = C / VEC;
  const int64_t total = N * per_row;
  for (int64_t t = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; t < total; t += int64_t(gridDim.x) * blockDim.x) {
    const int64_t i = t / per_row;
    const int p = int(t - i * per_row);
    const int64_t s = species_at(z, i, V);
    P r;
    if (s >= 0) {
      r = *reinterpret_cast<const P*>(table + s * C + p * VEC);
#pragma unroll
      for (int k = 0; k < VEC; ++k) r.v[k] = narrow<T>(scale * widen<T>(r.v[k]));
    } else {
      if (status && p == 0) atomicOr(status, Y3B_STATUS_INDEX_RANGE);
#pragma unroll
      for (int k = 0; k < VEC; ++k) r.v[k] = narrow<T>(0);
    }
    *reinterpret_cast<P*>(out + t * VEC) = r;
  }
}

// ---------------------------------------------------------------------------
// Stable radix sort of (species, atom index), 8 bits a pass.  A tile is 4096 keys:
// 8 warps of 512, warp w's element e at tile * 4096 + w * 512 + e, so that the order
// (warp, step, lane) is the order of the keys.
constexpr int kSortThreads = 256;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortSteps = 16;
constexpr int kSortTile = kSortThreads * kSortSteps;

// The first pass reads the caller's species; an invalid one sorts last, as key V.
template <typename I>
__device__ __forceinline__ uint32_t first_key(const I* z, int64_t i, int64_t V, int32_t* status) {
  const int64_t s = species_at(z, i, V);
  if (s < 0 && status) atomicOr(status, Y3B_STATUS_INDEX_RANGE);
  return s < 0 ? uint32_t(V) : uint32_t(s);
}

// Counts of each digit in each tile: hist[digit * tiles + tile].
template <typename I, bool FIRST>
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const I* __restrict__ z,
                                                                  const uint32_t* __restrict__ keys, int64_t N,
                                                                  int64_t V, int shift, int64_t tiles,
                                                                  uint32_t* __restrict__ hist, int32_t* status) {
  __shared__ uint32_t count[256];
  count[threadIdx.x] = 0;
  __syncthreads();
  const int64_t base = blockIdx.x * int64_t(kSortTile);
  for (int e = 0; e < kSortSteps; ++e) {
    const int64_t i = base + e * kSortThreads + threadIdx.x;
    if (i < N) {
      uint32_t k;
      if constexpr (FIRST) k = first_key(z, i, V, status);
      else k = keys[i];
      atomicAdd(&count[(k >> shift) & 255u], 1u);
    }
  }
  __syncthreads();
  hist[threadIdx.x * tiles + blockIdx.x] = count[threadIdx.x];
}

// Block-wide exclusive scan of one value per thread; returns the block's total in *sum.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* warp_sums, uint32_t* sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  uint32_t before = 0, all = 0;
  for (int w = 0; w < warps; ++w) {
    const uint32_t s = warp_sums[w];
    if (w < warp) before += s;
    all += s;
  }
  __syncthreads();
  *sum = all;
  return before + x - v;
}

// One CTA per digit: its tiles' counts become exclusive prefixes; totals[digit] their sum.
__global__ void __launch_bounds__(256) sort_scan_kernel(uint32_t* __restrict__ hist, int64_t tiles,
                                                        uint32_t* __restrict__ totals) {
  __shared__ uint32_t warp_sums[8];
  uint32_t* h = hist + blockIdx.x * tiles;
  uint32_t carry = 0;
  for (int64_t t0 = 0; t0 < tiles; t0 += 256) {
    const int64_t t = t0 + threadIdx.x;
    const uint32_t v = t < tiles ? h[t] : 0u;
    uint32_t sum;
    const uint32_t x = block_scan(v, warp_sums, &sum);
    if (t < tiles) h[t] = carry + x;
    carry += sum;
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

// Moves every key to its place.  The rank of a key among the equal digits of its tile
// is found in two steps: the counts of each digit in each warp, then the order
// within the warp from a match of the lanes' digits.
template <typename I, bool FIRST>
__global__ void __launch_bounds__(kSortThreads) sort_move_kernel(
    const I* __restrict__ z, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ values, int64_t N,
    int64_t V, int shift, int64_t tiles, const uint32_t* __restrict__ hist, const uint32_t* __restrict__ totals,
    uint32_t* __restrict__ keys_out, uint32_t* __restrict__ values_out) {
  __shared__ uint32_t warp_sums[kSortWarps];
  __shared__ uint32_t place[kSortWarps][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tid = threadIdx.x;
  for (int w = 0; w < kSortWarps; ++w) place[w][tid] = 0;
  uint32_t all;
  const uint32_t digit_start = block_scan(totals[tid], warp_sums, &all) + hist[tid * tiles + blockIdx.x];
  __syncthreads();
  const int64_t base = blockIdx.x * int64_t(kSortTile) + warp * (32 * kSortSteps) + lane;
  uint32_t key[kSortSteps], rank[kSortSteps];
#pragma unroll
  for (int e = 0; e < kSortSteps; ++e) {
    const int64_t i = base + e * 32;
    key[e] = 0;
    if (i < N) {
      if constexpr (FIRST) key[e] = first_key(z, i, V, nullptr);
      else key[e] = keys[i];
    }
  }
#pragma unroll
  for (int e = 0; e < kSortSteps; ++e) {
    const bool there = base + e * 32 < N;
    const uint32_t digit = there ? (key[e] >> shift) & 255u : 256u;
    const uint32_t same = __match_any_sync(0xffffffffu, digit);
    uint32_t before = 0;
    const int leader = __ffs(int(same)) - 1;
    if (lane == leader && there) {
      before = place[warp][digit];
      place[warp][digit] = before + __popc(same);
    }
    before = __shfl_sync(0xffffffffu, before, leader);
    rank[e] = before + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
  }
  __syncthreads();
  // the counts of the warps before become each warp's first place of the digit
  uint32_t at = digit_start;
  for (int w = 0; w < kSortWarps; ++w) {
    const uint32_t c = place[w][tid];
    place[w][tid] = at;
    at += c;
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < kSortSteps; ++e) {
    const int64_t i = base + e * 32;
    if (i < N) {
      const uint32_t to = place[warp][(key[e] >> shift) & 255u] + rank[e];
      keys_out[to] = key[e];
      if constexpr (FIRST) values_out[to] = uint32_t(i);
      else values_out[to] = values[i];
    }
  }
}

// ---------------------------------------------------------------------------
// Sums over runs of equal species.  A warp takes one chunk of the sorted atoms and 32 *
// VEC channels.  A run inside the chunk is written to its table row; the part of a run
// that began in an earlier chunk goes to head[chunk], the part of one that goes on
// into the next chunk to tail[chunk].  Eight gradient rows are loaded ahead of
// their sums.
template <typename T, int VEC>
__global__ void __launch_bounds__(128) run_sum_kernel(const T* __restrict__ grad, const uint32_t* __restrict__ keys,
                                                      const uint32_t* __restrict__ order, int64_t N, int64_t V,
                                                      int C, int chunk_rows, int64_t chunks,
                                                      typename Acc<T>::type scale, T* __restrict__ dtable,
                                                      typename Acc<T>::type* __restrict__ head,
                                                      typename Acc<T>::type* __restrict__ tail) {
  using A = typename Acc<T>::type;
  using P = Pack<T, VEC>;
  using PA = Pack<A, VEC>;
  const int lane = threadIdx.x & 31;
  const int64_t chunk = blockIdx.x * int64_t(4) + (threadIdx.x >> 5);
  const int c = int(blockIdx.y) * 32 * VEC + lane * VEC;
  if (chunk >= chunks) return;
  const bool mine = c < C;
  const int64_t b = chunk * chunk_rows, e = b + chunk_rows < N ? b + chunk_rows : N;
  const uint32_t none = 0xffffffffu;
  const uint32_t before = b > 0 ? keys[b - 1] : none, after = e < N ? keys[e] : none;
  A acc[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = A(0);
  uint32_t current = keys[b];
  bool at_begin = true;  // the run holds the chunk's first row
  auto store = [&](uint32_t key, bool begins, bool ends) {
    if (!mine || key >= V) return;  // key V: atoms whose species is out of range
    if (begins && before == key) {
      PA p;
#pragma unroll
      for (int k = 0; k < VEC; ++k) p.v[k] = acc[k];
      *reinterpret_cast<PA*>(head + chunk * C + c) = p;
    } else if (ends && after == key) {
      PA p;
#pragma unroll
      for (int k = 0; k < VEC; ++k) p.v[k] = acc[k];
      *reinterpret_cast<PA*>(tail + chunk * C + c) = p;
    } else {
      P p;
#pragma unroll
      for (int k = 0; k < VEC; ++k) p.v[k] = narrow<T>(scale * acc[k]);
      *reinterpret_cast<P*>(dtable + int64_t(key) * C + c) = p;
    }
  };
  for (int64_t r0 = b; r0 < e; r0 += 32) {
    const int n = e - r0 < 32 ? int(e - r0) : 32;
    const uint32_t my_key = lane < n ? keys[r0 + lane] : none, my_row = lane < n ? order[r0 + lane] : 0u;
    for (int j0 = 0; j0 < n; j0 += 8) {
      P g[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t row = __shfl_sync(0xffffffffu, my_row, (j0 + j) & 31);
        if (j0 + j < n && mine) g[j] = *reinterpret_cast<const P*>(grad + int64_t(row) * C + c);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t key = __shfl_sync(0xffffffffu, my_key, (j0 + j) & 31);
        if (j0 + j < n) {  // uniform over the warp
          if (key != current) {
            store(current, at_begin, false);
            at_begin = false;
            current = key;
#pragma unroll
            for (int k = 0; k < VEC; ++k) acc[k] = A(0);
          }
          if (mine) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) acc[k] += widen<T>(g[j].v[k]);
          }
        }
      }
    }
  }
  store(current, at_begin, true);
}

// Joins the runs that cross chunks: the chunk in which such a run begins adds its own
// part and those of the chunks that follow.  Warp w takes every 8th chunk and the
// warps' sums are added in order; lanes are channels.
template <typename T>
__global__ void __launch_bounds__(256) run_join_kernel(const uint32_t* __restrict__ keys, int64_t N, int64_t V, int C,
                                                       int chunk_rows, int64_t chunks, typename Acc<T>::type scale,
                                                       T* __restrict__ dtable,
                                                       const typename Acc<T>::type* __restrict__ head,
                                                       const typename Acc<T>::type* __restrict__ tail) {
  using A = typename Acc<T>::type;
  __shared__ A part[8][32];
  const int64_t chunk = blockIdx.x;
  const int64_t e = (chunk + 1) * chunk_rows;
  if (e >= N) return;  // the last chunk has no run that goes on
  const uint32_t key = keys[e - 1];
  if (key >= V || keys[e] != key) return;
  const int64_t b = chunk * chunk_rows;
  if (b > 0 && keys[b - 1] == key && keys[b] == key) return;  // the run began earlier
  // the run's last chunk: chunks whose first key is still this one (keys are sorted)
  int64_t lo = chunk + 1, hi = chunks;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    if (keys[mid * chunk_rows] == key) lo = mid;
    else hi = mid;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int c0 = int(blockIdx.y) * 32; c0 < C; c0 += int(gridDim.y) * 32) {
    const int c = c0 + lane;
    A sum = A(0);
    if (c < C) {
      int64_t q = chunk + 1 + warp;
      for (; q + 24 <= lo; q += 32) {
        const A a0 = head[q * C + c], a1 = head[(q + 8) * C + c];
        const A a2 = head[(q + 16) * C + c], a3 = head[(q + 24) * C + c];
        sum += (a0 + a1) + (a2 + a3);
      }
      for (; q <= lo; q += 8) sum += head[q * C + c];
    }
    part[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && c < C) {
      A all = tail[chunk * C + c];
#pragma unroll
      for (int w = 0; w < 8; ++w) all += part[w][lane];
      dtable[int64_t(key) * C + c] = narrow<T>(scale * all);
    }
    __syncthreads();
  }
}

// Workspace: two pairs of (key, index) arrays, the tiles' digit counts, the digits'
// totals and the chunks' head and tail sums; every part 32-byte aligned.
struct AdjointPlan {
  int64_t tiles, chunks;
  int chunk_rows, passes;
  int64_t keys[2], order[2], hist, totals, head, tail, bytes;
};

int64_t align32(int64_t v) { return (v + 31) / 32 * 32; }

AdjointPlan adjoint_plan(int dtype, int64_t N, int64_t V, int64_t C) {
  AdjointPlan p;
  p.tiles = (N + kSortTile - 1) / kSortTile;
  p.chunk_rows = N < (int64_t(1) << 18) ? 32 : 128;
  p.chunks = (N + p.chunk_rows - 1) / p.chunk_rows;
  p.passes = 1;
  while (p.passes < 4 && (V >> (8 * p.passes)) != 0) ++p.passes;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += align32(bytes);
    return here;
  };
  for (int k = 0; k < 2; ++k) {
    p.keys[k] = take(N * 4);
    p.order[k] = take(N * 4);
  }
  p.hist = take(256 * p.tiles * 4);
  p.totals = take(256 * 4);
  const int64_t real = dtype == Y3B_F64 ? 8 : 4;
  p.head = take(p.chunks * C * real);
  p.tail = take(p.chunks * C * real);
  p.bytes = at;
  return p;
}

bool embedding_dtype(int dtype) { return dtype == Y3B_F32 || dtype == Y3B_F64 || dtype == Y3B_BF16; }

bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <typename T, typename I>
int lookup(const T* table, int64_t V, int C, const I* z, int64_t N, double scale, T* out, int32_t* status,
           cudaStream_t s) {
  using A = typename Acc<T>::type;
  constexpr int W = 16 / int(sizeof(T));
  if (C % W == 0 && aligned(table, 16) && aligned(out, 16)) {
    embedding_kernel<T, I, W><<<grid_for(N * (C / W), 256), 256, 0, s>>>(table, V, C, z, N, A(scale), out, status);
  } else {
    embedding_kernel<T, I, 1><<<grid_for(N * C, 256), 256, 0, s>>>(table, V, C, z, N, A(scale), out, status);
  }
  Y3B_LAUNCH_CHECK();
  return Y3B_OK;
}

template <typename T, int VEC>
int run_sums(const T* grad, const AdjointPlan& p, const uint32_t* keys, const uint32_t* order, int64_t N, int64_t V,
             int C, double scale, T* dtable, void* head, void* tail, cudaStream_t s) {
  using A = typename Acc<T>::type;
  const dim3 grid(unsigned((p.chunks + 3) / 4), unsigned((C + 32 * VEC - 1) / (32 * VEC)));
  run_sum_kernel<T, VEC><<<grid, 128, 0, s>>>(grad, keys, order, N, V, C, p.chunk_rows, p.chunks, A(scale), dtable,
                                              static_cast<A*>(head), static_cast<A*>(tail));
  Y3B_LAUNCH_CHECK();
  return Y3B_OK;
}

template <typename T, typename I>
int adjoint(int dtype, const T* grad, const I* z, int64_t N, int64_t V, int C, double scale, unsigned char* ws,
            T* dtable, int32_t* status, cudaStream_t s) {
  using A = typename Acc<T>::type;
  const AdjointPlan p = adjoint_plan(dtype, N, V, C);
  uint32_t* hist = reinterpret_cast<uint32_t*>(ws + p.hist);
  uint32_t* totals = reinterpret_cast<uint32_t*>(ws + p.totals);
  const unsigned tiles = unsigned(p.tiles);
  for (int pass = 0; pass < p.passes; ++pass) {
    const uint32_t* ki = reinterpret_cast<const uint32_t*>(ws + p.keys[(pass + 1) & 1]);
    const uint32_t* vi = reinterpret_cast<const uint32_t*>(ws + p.order[(pass + 1) & 1]);
    uint32_t* ko = reinterpret_cast<uint32_t*>(ws + p.keys[pass & 1]);
    uint32_t* vo = reinterpret_cast<uint32_t*>(ws + p.order[pass & 1]);
    if (pass == 0)
      sort_count_kernel<I, true><<<tiles, kSortThreads, 0, s>>>(z, nullptr, N, V, 0, p.tiles, hist, status);
    else
      sort_count_kernel<I, false><<<tiles, kSortThreads, 0, s>>>(nullptr, ki, N, V, 8 * pass, p.tiles, hist, nullptr);
    sort_scan_kernel<<<256, 256, 0, s>>>(hist, p.tiles, totals);
    if (pass == 0)
      sort_move_kernel<I, true><<<tiles, kSortThreads, 0, s>>>(z, nullptr, nullptr, N, V, 0, p.tiles, hist, totals,
                                                              ko, vo);
    else
      sort_move_kernel<I, false><<<tiles, kSortThreads, 0, s>>>(nullptr, ki, vi, N, V, 8 * pass, p.tiles, hist,
                                                               totals, ko, vo);
    Y3B_LAUNCH_CHECK();
  }
  const uint32_t* keys = reinterpret_cast<const uint32_t*>(ws + p.keys[(p.passes - 1) & 1]);
  const uint32_t* order = reinterpret_cast<const uint32_t*>(ws + p.order[(p.passes - 1) & 1]);
  Y3B_CUDA_TRY(cudaMemsetAsync(dtable, 0, size_t(V) * C * sizeof(T), s));
  // the widest load that still gives most lanes a channel
  constexpr int W = 16 / int(sizeof(T));
  int rc;
  if (C >= 16 * W && C % W == 0 && aligned(grad, 16) && aligned(dtable, 16))
    rc = run_sums<T, W>(grad, p, keys, order, N, V, C, scale, dtable, ws + p.head, ws + p.tail, s);
  else if (C >= 48 && C % 2 == 0 && aligned(grad, 2 * sizeof(T)) && aligned(dtable, 2 * sizeof(T)))
    rc = run_sums<T, 2>(grad, p, keys, order, N, V, C, scale, dtable, ws + p.head, ws + p.tail, s);
  else
    rc = run_sums<T, 1>(grad, p, keys, order, N, V, C, scale, dtable, ws + p.head, ws + p.tail, s);
  if (rc) return rc;
  const dim3 grid(unsigned(p.chunks), unsigned(std::min((C + 31) / 32, 64)));
  run_join_kernel<T><<<grid, 256, 0, s>>>(keys, N, V, C, p.chunk_rows, p.chunks, A(scale), dtable,
                                          reinterpret_cast<const A*>(ws + p.head),
                                          reinterpret_cast<const A*>(ws + p.tail));
  Y3B_LAUNCH_CHECK();
  return Y3B_OK;
}

#define Y3B_EMBEDDING_DISPATCH(dtype, bytes, T, I, ...)                        \
  if (bytes == 4) {                                                            \
    using I = int32_t;                                                         \
    if (dtype == Y3B_F32) { using T = float; __VA_ARGS__; }                    \
    else if (dtype == Y3B_F64) { using T = double; __VA_ARGS__; }              \
    else { using T = __nv_bfloat16; __VA_ARGS__; }                             \
  } else {                                                                     \
    using I = int64_t;                                                         \
    if (dtype == Y3B_F32) { using T = float; __VA_ARGS__; }                    \
    else if (dtype == Y3B_F64) { using T = double; __VA_ARGS__; }              \
    else { using T = __nv_bfloat16; __VA_ARGS__; }                             \
  }

}  // namespace
}  // namespace y3b

using namespace y3b;

extern "C" int y3b_species_embedding(int dtype, const void* table, int64_t species_count, int64_t channels,
                                     const void* species, int species_bytes, int64_t atom_count, double scale,
                                     void* out, int32_t* status, void* stream) {
  Y3B_CHECK_ARG(embedding_dtype(dtype), "species_embedding: dtype must be F32, F64 or BF16");
  Y3B_CHECK_ARG(species_bytes == 4 || species_bytes == 8, "species_embedding: species must be int32 or int64");
  Y3B_CHECK_ARG(species_count >= 0 && atom_count >= 0, "species_embedding: negative size");
  Y3B_CHECK_ARG(channels >= 1 && channels <= (1 << 20), "species_embedding: 1 to 2^20 channels");
  if (atom_count == 0) return Y3B_OK;
  Y3B_CHECK_ARG((table || species_count == 0) && species && out, "species_embedding: null pointer argument");
  Y3B_EMBEDDING_DISPATCH(dtype, species_bytes, T, I,
                         return lookup<T, I>(static_cast<const T*>(table), species_count, int(channels),
                                             static_cast<const I*>(species), atom_count, scale, static_cast<T*>(out),
                                             status, as_stream(stream)))
}

extern "C" int64_t y3b_species_embedding_adjoint_workspace_bytes(int dtype, int64_t atom_count, int64_t species_count,
                                                                 int64_t channels) {
  if (!embedding_dtype(dtype) || atom_count < 0 || atom_count > INT32_MAX || species_count < 0 ||
      species_count > INT32_MAX || channels < 1 || channels > (1 << 20))
    return -1;
  return adjoint_plan(dtype, atom_count, species_count, channels).bytes;
}

extern "C" int y3b_species_embedding_adjoint(int dtype, const void* grad, const void* species, int species_bytes,
                                             int64_t atom_count, int64_t species_count, int64_t channels,
                                             double scale, void* workspace, int64_t workspace_bytes,
                                             void* table_grad, int32_t* status, void* stream) {
  const int64_t need = y3b_species_embedding_adjoint_workspace_bytes(dtype, atom_count, species_count, channels);
  Y3B_CHECK_ARG(need >= 0,
                "species_embedding_adjoint: dtype F32, F64 or BF16, up to 2^31 - 1 atoms and species, 1 to 2^20 "
                "channels");
  Y3B_CHECK_ARG(species_bytes == 4 || species_bytes == 8, "species_embedding_adjoint: species must be int32 or int64");
  if (species_count == 0) return Y3B_OK;
  Y3B_CHECK_ARG(table_grad, "species_embedding_adjoint: null pointer argument");
  if (atom_count == 0) {
    const size_t real = dtype == Y3B_F64 ? 8 : dtype == Y3B_F32 ? 4 : 2;
    Y3B_CUDA_TRY(cudaMemsetAsync(table_grad, 0, size_t(species_count) * size_t(channels) * real, as_stream(stream)));
    return Y3B_OK;
  }
  Y3B_CHECK_ARG(grad && species && workspace, "species_embedding_adjoint: null pointer argument");
  Y3B_CHECK_ARG(aligned(workspace, 32), "species_embedding_adjoint: workspace must be 32-byte aligned");
  if (workspace_bytes < need)
    return fail(Y3B_ERR_WORKSPACE, "species_embedding_adjoint: workspace of %lld bytes, %lld needed",
                (long long)workspace_bytes, (long long)need);
  Y3B_EMBEDDING_DISPATCH(dtype, species_bytes, T, I,
                         return adjoint<T, I>(dtype, static_cast<const T*>(grad), static_cast<const I*>(species),
                                              atom_count, species_count, int(channels), scale,
                                              static_cast<unsigned char*>(workspace), static_cast<T*>(table_grad),
                                              status, as_stream(stream)))
}
