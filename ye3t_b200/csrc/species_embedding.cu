// Learned per-species vectors: lookup with scaling and the table's gradient.
//
//   out[i, c]   = scale * table[z_i, c]
//   dtable[v, c] = scale * sum_{i : z_i = v} grad[i, c]
//
// The lookup is one pass over the output.  The gradient of a small table (up to 26 species; 108, in fp64 53, where the
// channels are no multiple of the vectors' width) is summed in copies of the table in shared memory; that of a larger one
// orders the atoms by species (stable radix sort of the indices) and sums runs of equal species.  Neither needs
// floating-point atomics, and results are bitwise repeatable.
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

// A CTA is X threads along the channels by 256 / X along the atoms; a thread writes VEC channels of kLookups atoms.
// The table stays in L2.  2^20 atoms x 32 in fp32: 37 us, 3.6 TB/s of output; issue is 63 % active and DRAM writes 2 TB/s
// (the rest of the output is still in L2), so that neither is the bound by itself.
constexpr int kLookups = 4;

template <typename T, typename I, int VEC>
__global__ void __launch_bounds__(256) embedding_kernel(const T* __restrict__ table, int64_t V, int C,
                                                        const I* __restrict__ z, int64_t N,
                                                        typename Acc<T>::type scale, T* __restrict__ out,
                                                        int32_t* status) {
  using P = Pack<T, VEC>;
  const int64_t first = blockIdx.x * int64_t(blockDim.y * kLookups) + threadIdx.y;
  int64_t s[kLookups];
#pragma unroll
  for (int k = 0; k < kLookups; ++k) {
    const int64_t i = first + k * blockDim.y;
    s[k] = i < N ? species_at(z, i, V) : -2;
    if (s[k] == -1 && status && threadIdx.x == 0 && blockIdx.y == 0) atomicOr(status, Y3B_STATUS_INDEX_RANGE);
  }
  const int c = int(blockIdx.y * blockDim.x + threadIdx.x) * VEC;
  if (c >= C) return;
  P r[kLookups];
#pragma unroll
  for (int k = 0; k < kLookups; ++k)
    if (s[k] >= 0) r[k] = *reinterpret_cast<const P*>(table + s[k] * C + c);
#pragma unroll
  for (int k = 0; k < kLookups; ++k) {
    if (s[k] == -2) continue;
#pragma unroll
    for (int q = 0; q < VEC; ++q) r[k].v[q] = s[k] >= 0 ? narrow<T>(scale * widen<T>(r[k].v[q])) : narrow<T>(0);
    *reinterpret_cast<P*>(out + (first + k * blockDim.y) * C + c) = r[k];
  }
}

// ---------------------------------------------------------------------------
// Gradient of a small table.  A unit of L lanes has a copy of L * VEC of the table's channels in shared
// memory (and one row more, for atoms without a species) and adds its rows to it, in order; lanes are
// channels, so nothing is shared between lanes.  The copies are added in order of the units, and the CTAs' sums
// (one part each) by part_sum_kernel.  Bound by reading the gradients once: a unit keeps eight rows in flight while
// it adds the eight before, and adds four at a time (their table rows are loaded together, equal species among
// them taken from registers).
constexpr int kTableRows = 8;
constexpr int kTableThreads = 256;
constexpr int kTableSmem = 109 * 1024;  // of the copies: two CTAs an SM

template <typename T, typename I, int VEC, int L>
__global__ void __launch_bounds__(kTableThreads) table_sum_kernel(
    const T* __restrict__ grad, const I* __restrict__ z, int64_t N, int V, int C, int64_t rows_per_unit,
    typename Acc<T>::type scale, T* __restrict__ dtable, typename Acc<T>::type* __restrict__ part, int32_t* status) {
  using A = typename Acc<T>::type;
  using P = Pack<T, VEC>;
  using PA = Pack<A, VEC>;
  extern __shared__ __align__(32) unsigned char table_smem[];
  A* copies = reinterpret_cast<A*>(table_smem);  // [unit][V + 1][L * VEC]
  constexpr int S = L * VEC, kUnits = kTableThreads / L;
  const int lane = threadIdx.x % L, unit = threadIdx.x / L;
  const int copy = (V + 1) * S;
  for (int u = threadIdx.x; u < kUnits * copy; u += kTableThreads) copies[u] = A(0);
  __syncthreads();
  A* mine = copies + unit * copy + lane * VEC;
  const int c = int(blockIdx.y) * S + lane * VEC;
  const bool there = c < C;
  const int64_t b = (blockIdx.x * int64_t(kUnits) + unit) * rows_per_unit;
  const int64_t e = b + rows_per_unit < N ? b + rows_per_unit : N;
  const auto species = [&](int64_t r) {  // of the unit's row r + lane, by its first lanes
    if (lane >= kTableRows || r + lane >= e) return V;
    const int64_t s = species_at(z, r + lane, V);
    if (s < 0 && status && blockIdx.y == 0) atomicOr(status, Y3B_STATUS_INDEX_RANGE);
    return s < 0 ? V : int(s);
  };
  const auto fetch = [&](int64_t r, P (&g)[kTableRows]) {
#pragma unroll
    for (int j = 0; j < kTableRows; ++j) {
#pragma unroll
      for (int q = 0; q < VEC; ++q) g[j].v[q] = narrow<T>(0);
      if (r + j < e && there) g[j] = *reinterpret_cast<const P*>(grad + (r + j) * C + c);
    }
  };
  const auto add_rows = [&](const P (&g)[kTableRows], int zs) {
#pragma unroll
    for (int j = 0; j < kTableRows; j += 4) {
      int k[4];
      PA r[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        k[u] = __shfl_sync(0xffffffffu, zs, j + u, L);
        r[u] = *reinterpret_cast<const PA*>(mine + k[u] * S);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
#pragma unroll
        for (int w = 0; w < u; ++w)
          if (k[w] == k[u]) r[u] = r[w];  // the latest of the equal ones stays
#pragma unroll
        for (int q = 0; q < VEC; ++q) r[u].v[q] += widen<T>(g[j + u].v[q]);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) *reinterpret_cast<PA*>(mine + k[u] * S) = r[u];
    }
  };
  // every unit takes the same number of steps, so that the shuffles find all lanes
  P g0[kTableRows], g1[kTableRows];
  int z0 = species(b), z1;
  fetch(b, g0);
  for (int64_t r = 0; r < rows_per_unit; r += 2 * kTableRows) {
    z1 = species(b + r + kTableRows);
    fetch(b + r + kTableRows, g1);
    add_rows(g0, z0);
    z0 = species(b + r + 2 * kTableRows);
    fetch(b + r + 2 * kTableRows, g0);
    add_rows(g1, z1);
  }
  __syncthreads();
  for (int u = threadIdx.x; u < V * S; u += kTableThreads) {
    const int v = u / S, cc = int(blockIdx.y) * S + u - v * S;
    if (cc >= C) continue;
    A sum = copies[u];
    for (int w = 1; w < kUnits; ++w) sum += copies[w * copy + u];
    if (part) part[(int64_t(blockIdx.x) * V + v) * C + cc] = sum;
    else dtable[int64_t(v) * C + cc] = narrow<T>(scale * sum);
  }
}

// dtable = scale * the parts' sums: 32 entries a CTA, every 32nd part a warp, the warps in order.
template <typename T>
__global__ void __launch_bounds__(1024) part_sum_kernel(const typename Acc<T>::type* __restrict__ part, int64_t parts,
                                                        int64_t entries, typename Acc<T>::type scale,
                                                        T* __restrict__ dtable) {
  using A = typename Acc<T>::type;
  __shared__ A sums[32][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t u = blockIdx.x * int64_t(32) + lane;
  A sum = A(0);
  if (u < entries) {
#pragma unroll 4
    for (int64_t p = warp; p < parts; p += 32) sum += part[p * entries + u];
  }
  sums[warp][lane] = sum;
  __syncthreads();
  if (warp == 0 && u < entries) {
    A all = sums[0][lane];
#pragma unroll
    for (int w = 1; w < 32; ++w) all += sums[w][lane];
    dtable[u] = narrow<T>(scale * all);
  }
}

// ---------------------------------------------------------------------------
// Stable radix sort of (species, atom index), 8 bits a pass.  A tile is 1024 keys: 8 warps of
// 128, warp w's element e at tile * 1024 + w * 128 + e, so that the order (warp, step, lane) is the
// order of the keys.
constexpr int kSortThreads = 256;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortSteps = 4;
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

// The whole sort in one CTA for up to kOneSort atoms, where the launches of a pass would cost more than its work: 500
// atoms 5.3 us against 7.6 in three launches, 4,096 atoms 8.4 against 8.7 with one digit, 15.3 against 18.4 in six
// launches with two.
constexpr int kOneSort = 4096;
constexpr int kOneWarps = 32;
constexpr int kOneSmem = kOneSort * 8 + kOneWarps * 256 * 2;

template <typename I>
__global__ void __launch_bounds__(32 * kOneWarps) one_sort_kernel(const I* __restrict__ z, int N, int64_t V, int passes,
                                                                 uint32_t* __restrict__ keys_out,
                                                                 uint32_t* __restrict__ values_out, int32_t* status) {
  extern __shared__ __align__(16) unsigned char sort_smem[];
  uint32_t* s_key = reinterpret_cast<uint32_t*>(sort_smem);
  uint32_t* s_val = s_key + kOneSort;
  uint16_t* place = reinterpret_cast<uint16_t*>(s_val + kOneSort);  // [warp][256]
  __shared__ uint32_t warp_sums[kOneWarps];
  constexpr int STEPS = kOneSort / (32 * kOneWarps);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, base = warp * (32 * STEPS) + lane;
  for (int e = 0; e < STEPS; ++e) {
    const int i = base + e * 32;
    if (i < N) {
      s_key[i] = first_key(z, i, V, status);
      s_val[i] = uint32_t(i);
    }
  }
  for (int pass = 0; pass < passes; ++pass) {
    for (int u = tid; u < kOneWarps * 256; u += blockDim.x) place[u] = 0;
    __syncthreads();
    uint32_t key[STEPS], value[STEPS], rank[STEPS];
#pragma unroll
    for (int e = 0; e < STEPS; ++e) {
      const int i = base + e * 32;
      const bool there = i < N;
      key[e] = there ? s_key[i] : 0u;
      value[e] = there ? s_val[i] : 0u;
      const uint32_t digit = there ? (key[e] >> (8 * pass)) & 255u : 256u;
      const uint32_t same = __match_any_sync(0xffffffffu, digit);
      const int leader = __ffs(int(same)) - 1;
      uint32_t before = 0;
      if (lane == leader && there) {
        before = place[warp * 256 + digit];
        place[warp * 256 + digit] = uint16_t(before + __popc(same));
      }
      before = __shfl_sync(0xffffffffu, before, leader);
      rank[e] = before + __popc(same & ((1u << lane) - 1u));
      __syncwarp();
    }
    __syncthreads();
    // exclusive prefix of each digit over the warps, then over the digits
    uint32_t total = 0;
    if (tid < 256) {
      for (int w = 0; w < kOneWarps; ++w) {
        const uint32_t c = place[w * 256 + tid];
        place[w * 256 + tid] = uint16_t(total);
        total += c;
      }
    }
    uint32_t all;
    const uint32_t start = block_scan(total, warp_sums, &all);
    if (tid < 256) {
      for (int w = 0; w < kOneWarps; ++w) place[w * 256 + tid] = uint16_t(place[w * 256 + tid] + start);
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < STEPS; ++e) {
      if (base + e * 32 < N) {
        const uint32_t to = place[warp * 256 + ((key[e] >> (8 * pass)) & 255u)] + rank[e];
        s_key[to] = key[e];
        s_val[to] = value[e];
      }
    }
    __syncthreads();
  }
  for (int i = tid; i < N; i += blockDim.x) {
    keys_out[i] = s_key[i];
    values_out[i] = s_val[i];
  }
}

// ---------------------------------------------------------------------------
// Sums over runs of equal species.  A unit of L lanes takes one chunk of the sorted atoms and L *
// VEC channels.  A run inside the chunk is written to its table row; the part of a run
// that began in an earlier chunk goes to head[chunk], the part of one that goes on
// into the next chunk to tail[chunk].  Eight gradient rows load while the eight before are added.
template <typename T, int VEC, int L>
__global__ void __launch_bounds__(128) run_sum_kernel(const T* __restrict__ grad, const uint32_t* __restrict__ keys,
                                                      const uint32_t* __restrict__ order, int64_t N, int64_t V,
                                                      int C, int chunk_rows, int64_t chunks,
                                                      typename Acc<T>::type scale, T* __restrict__ dtable,
                                                      typename Acc<T>::type* __restrict__ head,
                                                      typename Acc<T>::type* __restrict__ tail) {
  using A = typename Acc<T>::type;
  using P = Pack<T, VEC>;
  using PA = Pack<A, VEC>;
  constexpr int kRows = 8;
  const int lane = threadIdx.x % L;
  const int64_t chunk = blockIdx.x * int64_t(128 / L) + threadIdx.x / L;
  const int c = (int(blockIdx.y) * L + lane) * VEC;
  const bool mine = c < C && chunk < chunks;
  const int64_t b = chunk * chunk_rows < N ? chunk * chunk_rows : N, e = b + chunk_rows < N ? b + chunk_rows : N;
  const uint32_t none = 0xffffffffu;
  const uint32_t before = b > 0 && b < N ? keys[b - 1] : none, after = e < N ? keys[e] : none;
  A acc[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = A(0);
  uint32_t current = b < e ? keys[b] : none;
  bool at_begin = true;  // the run holds the chunk's first row
  auto store = [&](bool ends) {
    if (!mine || current >= V) return;  // key V: atoms whose species is out of range
    A* to = at_begin && before == current ? head : ends && after == current ? tail : nullptr;
    if (to) {
      PA p;
#pragma unroll
      for (int k = 0; k < VEC; ++k) p.v[k] = acc[k];
      *reinterpret_cast<PA*>(to + chunk * C + c) = p;
    } else {
      P p;
#pragma unroll
      for (int k = 0; k < VEC; ++k) p.v[k] = narrow<T>(scale * acc[k]);
      *reinterpret_cast<P*>(dtable + int64_t(current) * C + c) = p;
    }
  };
  uint32_t key = none, row = 0u;
  const auto index = [&](int64_t r) {  // of the unit's row r + lane, by its first lanes
    const bool ok = lane < kRows && r + lane < e;
    key = ok ? keys[r + lane] : none;
    row = ok ? order[r + lane] : 0u;
  };
  const auto fetch = [&](P (&g)[kRows]) {
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const uint32_t from = __shfl_sync(0xffffffffu, row, j, L);
      if (mine) g[j] = *reinterpret_cast<const P*>(grad + int64_t(from) * C + c);  // row 0 past the end
    }
  };
  const auto add_rows = [&](uint32_t keys_of, const P (&g)[kRows]) {
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const uint32_t k = __shfl_sync(0xffffffffu, keys_of, j, L);
      if (k == none) continue;  // past the chunk's end
      if (k != current) {
        store(false);
        at_begin = false;
        current = k;
#pragma unroll
        for (int q = 0; q < VEC; ++q) acc[q] = A(0);
      }
      if (mine) {
#pragma unroll
        for (int q = 0; q < VEC; ++q) acc[q] += widen<T>(g[j].v[q]);
      }
    }
  };
  // the indices run two steps ahead of the sums, the gradients one
  P g0[kRows], g1[kRows];
  index(b);
  uint32_t k0 = key, k1;
  fetch(g0);
  index(b + kRows);
  for (int r = 0; r < chunk_rows; r += 2 * kRows) {
    k1 = key;
    fetch(g1);
    index(b + r + 2 * kRows);
    add_rows(k0, g0);
    k0 = key;
    fetch(g0);
    index(b + r + 3 * kRows);
    add_rows(k1, g1);
  }
  store(true);
}

// Joins the runs that cross chunks: the chunk in which such a run begins adds its own
// part and those of the chunks that follow.  A CTA looks at 8 chunks, one after the other; warp w takes
// every 8th of a run's chunks and the warps' sums are added in order; lanes are channels.
constexpr int kJoinChunks = 8;

template <typename T>
__global__ void __launch_bounds__(256) run_join_kernel(const uint32_t* __restrict__ keys, int64_t N, int64_t V, int C,
                                                       int chunk_rows, int64_t chunks, typename Acc<T>::type scale,
                                                       T* __restrict__ dtable,
                                                       const typename Acc<T>::type* __restrict__ head,
                                                       const typename Acc<T>::type* __restrict__ tail) {
  using A = typename Acc<T>::type;
  __shared__ A part[8][32];
  __shared__ uint32_t run_key[kJoinChunks];
  __shared__ int64_t run_last[kJoinChunks];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // each warp looks at one chunk: does a run begin in it and go on, and up to which chunk?
  {
    const int64_t chunk = blockIdx.x * int64_t(kJoinChunks) + warp, b = chunk * chunk_rows, e = b + chunk_rows;
    uint32_t key = 0xffffffffu;
    int64_t lo = chunk;
    if (e < N) {
      key = keys[e - 1];
      const bool earlier = b > 0 && keys[b - 1] == key && keys[b] == key;
      if (key >= V || keys[e] != key || earlier) key = 0xffffffffu;
    }
    if (key != 0xffffffffu) {
      // keys are sorted: the last chunk whose first key is still this one, by 32 probes a round
      lo = chunk + 1;
      int64_t hi = chunks;  // first chunk known to begin with another key
      while (hi - lo > 1) {
        const int64_t step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step;
        const bool same = at < hi && keys[at * chunk_rows] == key;
        const int n = __popc(__ballot_sync(0xffffffffu, same));
        const int64_t up = lo + int64_t(n + 1) * step;
        lo += n * step;
        hi = up < hi ? up : hi;
      }
    }
    // a short run is the warp's own work, a long one the CTA's
    const bool brief = key != 0xffffffffu && lo - chunk <= 16;
    if (brief) {
      for (int c = int(blockIdx.y) * 32 + lane; c < C; c += int(gridDim.y) * 32) {
        A sum = tail[chunk * C + c];
#pragma unroll 4
        for (int64_t q = chunk + 1; q <= lo; ++q) sum += head[q * C + c];
        dtable[int64_t(key) * C + c] = narrow<T>(scale * sum);
      }
    }
    if (lane == 0) {
      run_key[warp] = brief ? 0xffffffffu : key;
      run_last[warp] = lo;
    }
  }
  __syncthreads();
  for (int k = 0; k < kJoinChunks; ++k) {
    const uint32_t key = run_key[k];
    if (key == 0xffffffffu) continue;
    const int64_t chunk = blockIdx.x * int64_t(kJoinChunks) + k, last = run_last[k];
    for (int c0 = int(blockIdx.y) * 32; c0 < C; c0 += int(gridDim.y) * 32) {
      const int c = c0 + lane;
      A sum = A(0);
      if (c < C) {
#pragma unroll 4
        for (int64_t q = chunk + 1 + warp; q <= last; q += 8) sum += head[q * C + c];
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
}

// How the gradient of one call is formed.  A table is small where an SM holds a copy of lanes * vec of its
// channels for each unit of two CTAs (26 species in fp32): fewer warps do not keep the memory busy.
// Workspace: the parts of the small path; of the other two pairs of (key, index) arrays, the
// tiles' digit counts, the digits' totals and the chunks' head and tail sums; 32-byte aligned.
struct AdjointPlan {
  bool small;
  int vec, lanes;  // of the small path
  int64_t parts, rows_per_unit;
  int64_t tiles, chunks;
  int chunk_rows, passes;
  int64_t keys[2], order[2], hist, totals, head, tail, bytes;
};

int64_t align32(int64_t v) { return (v + 31) / 32 * 32; }

// Lanes of a unit: the fewest of 8, 16 and 32 that hold C channels by VEC.
int unit_lanes(int64_t C, int vec) { return C <= 8 * vec ? 8 : C <= 16 * vec ? 16 : 32; }

AdjointPlan adjoint_plan(int dtype, int64_t N, int64_t V, int64_t C) {
  AdjointPlan p{};
  const int64_t real = dtype == Y3B_F64 ? 8 : 4;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += align32(bytes);
    return here;
  };
  // an odd number of bf16 channels has no aligned pairs
  const int wide = dtype == Y3B_F64 ? 2 : 4;
  p.vec = C % wide == 0 ? wide : 1;
  p.lanes = unit_lanes(C, p.vec);
  const int64_t units = kTableThreads / p.lanes, copies = units * (V + 1) * p.lanes * p.vec * real;
  p.small = copies <= kTableSmem;
  if (p.small) {
    const int64_t slabs = (C + p.lanes * p.vec - 1) / (p.lanes * p.vec);
    const int64_t per_sm = std::min<int64_t>(2048 / kTableThreads, 220 * 1024 / (copies + 1024));
    const int64_t most = std::max<int64_t>(1, kSMs * per_sm / slabs);
    // at least 64 rows a unit: fewer do not pay for another part
    p.parts = std::min(most, std::max<int64_t>(1, (N + units * 64 - 1) / (units * 64)));
    p.rows_per_unit = (N + p.parts * units - 1) / (p.parts * units);
    p.head = take(p.parts > 1 ? p.parts * V * C * real : 0);
    p.bytes = at;
    return p;
  }
  p.tiles = (N + kSortTile - 1) / kSortTile;
  // Short chunks fill the SMs, long ones leave fewer runs to join.  Kernels of a step with 32 and with 128 rows, us: 30,000
  // atoms of 118 species x 64 23 and 29; 65,536 of 50,021 x 100 45 and 52; 98,304 59 and 59; 200,003 92 and 82; 2^19 of 118
  // x 64 147 and 98.
  p.chunk_rows = N < 3 * (int64_t(1) << 15) ? 32 : 128;
  p.chunks = (N + p.chunk_rows - 1) / p.chunk_rows;
  p.passes = 1;
  while (p.passes < 4 && (V >> (8 * p.passes)) != 0) ++p.passes;
  for (int k = 0; k < 2; ++k) {
    p.keys[k] = take(N * 4);
    p.order[k] = take(N * 4);
  }
  p.hist = take(256 * p.tiles * 4);
  p.totals = take(256 * 4);
  p.head = take(p.chunks * C * real);
  p.tail = take(p.chunks * C * real);
  p.bytes = at;
  return p;
}

bool embedding_dtype(int dtype) { return dtype == Y3B_F32 || dtype == Y3B_F64 || dtype == Y3B_BF16; }

bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <typename T, typename I, int VEC>
int lookup(const T* table, int64_t V, int C, const I* z, int64_t N, double scale, T* out, int32_t* status,
           cudaStream_t s) {
  using A = typename Acc<T>::type;
  const int per_row = C / VEC;
  unsigned x = 1;
  while (x < 256 && int(x) < per_row) x *= 2;
  const unsigned y = 256 / x;
  const int64_t ctas = (N + y * kLookups - 1) / (y * kLookups), slabs = (per_row + x - 1) / x;
  if (ctas > INT32_MAX || slabs > 65535)
    return fail(Y3B_ERR_UNSUPPORTED, "species_embedding: %lld atoms of %d channels", (long long)N, C);
  embedding_kernel<T, I, VEC><<<dim3(unsigned(ctas), unsigned(slabs)), dim3(x, y), 0, s>>>(table, V, C, z, N, A(scale),
                                                                                          out, status);
  Y3B_LAUNCH_CHECK();
  return Y3B_OK;
}

template <typename T, typename I>
int lookup(const T* table, int64_t V, int C, const I* z, int64_t N, double scale, T* out, int32_t* status,
           cudaStream_t s) {
  constexpr int W = 16 / int(sizeof(T));
  if (C % W == 0 && aligned(table, 16) && aligned(out, 16))
    return lookup<T, I, W>(table, V, C, z, N, scale, out, status, s);
  return lookup<T, I, 1>(table, V, C, z, N, scale, out, status, s);
}

template <typename T, int VEC, int L>
int run_sums(const T* grad, const AdjointPlan& p, const uint32_t* keys, const uint32_t* order, int64_t N, int64_t V,
             int C, double scale, T* dtable, void* head, void* tail, cudaStream_t s) {
  using A = typename Acc<T>::type;
  const dim3 grid(unsigned((p.chunks * L + 127) / 128), unsigned((C + L * VEC - 1) / (L * VEC)));
  run_sum_kernel<T, VEC, L><<<grid, 128, 0, s>>>(grad, keys, order, N, V, C, p.chunk_rows, p.chunks, A(scale), dtable,
                                                 static_cast<A*>(head), static_cast<A*>(tail));
  Y3B_LAUNCH_CHECK();
  return Y3B_OK;
}

template <typename T, int VEC>
int run_sums(const T* grad, const AdjointPlan& p, const uint32_t* keys, const uint32_t* order, int64_t N, int64_t V,
             int C, double scale, T* dtable, void* head, void* tail, cudaStream_t s) {
  const int lanes = unit_lanes(C, VEC);
  if (lanes == 8) return run_sums<T, VEC, 8>(grad, p, keys, order, N, V, C, scale, dtable, head, tail, s);
  if (lanes == 16) return run_sums<T, VEC, 16>(grad, p, keys, order, N, V, C, scale, dtable, head, tail, s);
  return run_sums<T, VEC, 32>(grad, p, keys, order, N, V, C, scale, dtable, head, tail, s);
}

template <typename T, typename I, int VEC, int L>
int table_sums(const AdjointPlan& p, const T* grad, const I* z, int64_t N, int64_t V, int C, double scale,
               unsigned char* ws, T* dtable, int32_t* status, cudaStream_t s) {
  using A = typename Acc<T>::type;
  const auto kernel = table_sum_kernel<T, I, VEC, L>;
  const int smem = int(kTableThreads * (V + 1) * VEC * int64_t(sizeof(A))), slabs = (C + L * VEC - 1) / (L * VEC);
  // the kernel's limit is that of every table, so that calls of several threads only ever set the same value
  Y3B_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kTableSmem));
  A* part = p.parts > 1 ? reinterpret_cast<A*>(ws + p.head) : nullptr;
  kernel<<<dim3(unsigned(p.parts), unsigned(slabs)), kTableThreads, smem, s>>>(grad, z, N, int(V), C, p.rows_per_unit,
                                                                              A(scale), dtable, part, status);
  Y3B_LAUNCH_CHECK();
  if (part) {
    part_sum_kernel<T><<<unsigned((V * C + 31) / 32), 1024, 0, s>>>(part, p.parts, V * C, A(scale), dtable);
    Y3B_LAUNCH_CHECK();
  }
  return Y3B_OK;
}

// The lanes follow from the plan's; a gradient off the vectors' alignment is read value by value by as many
// lanes, in more slabs.
template <typename T, typename I>
int table_sums(const AdjointPlan& p, const T* grad, const I* z, int64_t N, int64_t V, int C, double scale,
               unsigned char* ws, T* dtable, int32_t* status, cudaStream_t s) {
  constexpr int W = sizeof(T) == 8 ? 2 : 4;
  const bool wide = p.vec == W && aligned(grad, sizeof(T) * W);
#define Y3B_TABLE(L)                                                                              \
  return wide ? table_sums<T, I, W, L>(p, grad, z, N, V, C, scale, ws, dtable, status, s)         \
              : table_sums<T, I, 1, L>(p, grad, z, N, V, C, scale, ws, dtable, status, s)
  if (p.lanes == 8) { Y3B_TABLE(8); }
  if (p.lanes == 16) { Y3B_TABLE(16); }
  Y3B_TABLE(32);
#undef Y3B_TABLE
}

template <typename T, typename I>
int adjoint(int dtype, const T* grad, const I* z, int64_t N, int64_t V, int C, double scale, unsigned char* ws,
            T* dtable, int32_t* status, cudaStream_t s) {
  using A = typename Acc<T>::type;
  const AdjointPlan p = adjoint_plan(dtype, N, V, C);
  if (p.small) return table_sums<T, I>(p, grad, z, N, V, C, scale, ws, dtable, status, s);
  uint32_t* hist = reinterpret_cast<uint32_t*>(ws + p.hist);
  uint32_t* totals = reinterpret_cast<uint32_t*>(ws + p.totals);
  const unsigned tiles = unsigned(p.tiles);
  const bool one = N <= kOneSort;
  if (one) {
    Y3B_CUDA_TRY(cudaFuncSetAttribute(one_sort_kernel<I>, cudaFuncAttributeMaxDynamicSharedMemorySize, kOneSmem));
    const int to = (p.passes - 1) & 1;
    one_sort_kernel<I><<<1, 32 * kOneWarps, kOneSmem, s>>>(z, int(N), V, p.passes,
                                                           reinterpret_cast<uint32_t*>(ws + p.keys[to]),
                                                           reinterpret_cast<uint32_t*>(ws + p.order[to]), status);
    Y3B_LAUNCH_CHECK();
  }
  for (int pass = 0; !one && pass < p.passes; ++pass) {
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
  constexpr int W = sizeof(T) == 8 ? 2 : 4;
  const bool wide = C % W == 0 && aligned(grad, W * sizeof(T)) && aligned(dtable, W * sizeof(T));
  const int rc = wide ? run_sums<T, W>(grad, p, keys, order, N, V, C, scale, dtable, ws + p.head, ws + p.tail, s)
                      : run_sums<T, 1>(grad, p, keys, order, N, V, C, scale, dtable, ws + p.head, ws + p.tail, s);
  if (rc) return rc;
  if (p.chunks == 1) return Y3B_OK;
  const dim3 grid(unsigned((p.chunks + kJoinChunks - 1) / kJoinChunks), unsigned(std::min((C + 31) / 32, 64)));
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
