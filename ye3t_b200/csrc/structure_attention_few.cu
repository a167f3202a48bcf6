// Structure attention of one or two queries over many keys: a pooled readout, or one new atom against a structure.
//
// A CTA takes a chunk of a structure's keys, one key head and two of the (query, head) rows that it serves.
// LPK lanes hold one key's components, 16 bytes each, so that every load is a full line of K or V; a warp takes
// 32 / LPK keys at a time, four steps in flight.  Each group of lanes keeps its own running maximum, sum and
// accumulator in fp32; they are joined at the end of the chunk, and the chunks by the join kernels.  Bound by
// reading K and V once (two rows of arithmetic a key take about half of that time); a tile of the tensor cores would
// hold two rows of 128.  Readout of 8 structures of 16,384 keys on average, 8 heads of 64 on 4 key heads: 50 us,
// 3.0 TB/s.
#include "structure_attention_few.cuh"
#include "structure_attention_tile.cuh"

namespace y3b {
namespace {

constexpr int kFewWarps = 4;
constexpr int kFewSteps = 4;  // two steps and more CTAs an SM take 64 us where four take 50 (the readout below)
constexpr int kFewRows = 2;
// Keys in flight on the key side and CTAs an SM that the registers are held to: 20 structures of 5,000 keys, 3 heads of
// 128, fp32, 139 us; four keys and 120 registers 167, one key 180.
constexpr int kFewKeySteps = 2, kFewKeyCtas = 8;

// W components of a row from `p`, as fp32, zeros from `left` on.
template <typename T, int W>
__device__ __forceinline__ void load_part(float (&v)[W], const T* p, int left, bool vec) {
  if (vec) {
    if (left > 0) {  // whole parts: left is a multiple of W
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] = to_float(t[k]);
    } else {
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] = 0.0f;
    }
  } else {
#pragma unroll
    for (int k = 0; k < W; ++k) v[k] = k < left ? to_float(p[k]) : 0.0f;
  }
}

// The same as raw bits, to be in flight while other work is done; VEC: the rows start on 16 bytes.
template <typename T, int W, bool VEC>
__device__ __forceinline__ uint4 raw_part(const T* p, int left) {
  uint4 u = make_uint4(0u, 0u, 0u, 0u);
  if constexpr (VEC) {
    if (left > 0) u = *reinterpret_cast<const uint4*>(p);
  } else {
    T* t = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int k = 0; k < W; ++k)
      if (k < left) t[k] = p[k];
  }
  return u;
}
template <typename T, int W>
__device__ __forceinline__ void widen_part(float (&v)[W], const uint4& u) {
  const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int k = 0; k < W; ++k) v[k] = to_float(t[k]);
}

template <int LPK>
__device__ __forceinline__ float part_sum(float v) {
#pragma unroll
  for (int o = LPK / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T, int LPK, bool BACKWARD, bool VEC>
__global__ void __launch_bounds__(32 * kFewWarps) few_kernel(const __grid_constant__ AttArgs a,
                                                            const AttItem* __restrict__ items, int DP, int width,
                                                            int vec, const T* __restrict__ out,
                                                            const T* __restrict__ grad,
                                                            const float* __restrict__ lse, float* __restrict__ part) {
  constexpr int W = 16 / int(sizeof(T)), KPW = 32 / LPK;
  constexpr int SUMS = BACKWARD ? 10 : 2, ACC = BACKWARD ? 2 : 1;
  __shared__ float s_sum[kFewWarps][kFewRows][SUMS];
  __shared__ float s_acc[kFewWarps][kFewRows][ACC][LPK * W];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, slot = lane / LPK, d0 = (lane % LPK) * W;
  const int blocks = (kFewQueries * a.group + kFewRows - 1) / kFewRows;
  unsigned task = blockIdx.x;
  const int block = int(task % unsigned(blocks));
  task /= unsigned(blocks);
  const int hk = int(task % unsigned(a.Hk));
  const AttItem it = items[task / unsigned(a.Hk)];
  const int row_count = it.rows * a.group, first = block * kFewRows;
  if (first >= row_count) return;
  const bool bias = a.slopes != nullptr;

  // the rows: (query, head) = (r / group, r % group)
  int head[kFewRows];
  int64_t query[kFewRows];
  float q[kFewRows][W], g[kFewRows][W], slope2[kFewRows], px[kFewRows], py[kFewRows], pz[kFewRows], L[kFewRows],
      delta0[kFewRows];
#pragma unroll
  for (int r = 0; r < kFewRows; ++r) {
    const int u = first + r < row_count ? first + r : first;
    query[r] = int64_t(it.row) + u / a.group;
    head[r] = hk * a.group + u % a.group;
    const int64_t at = (query[r] * a.H + head[r]) * a.D + d0;
    load_part<T, W>(q[r], static_cast<const T*>(a.q) + query[r] * a.q_row + head[r] * a.q_head + d0, a.D - d0, vec & 1);
#pragma unroll
    for (int k = 0; k < W; ++k) q[r][k] *= a.scale2;
    if constexpr (BACKWARD) {
      float o[W];
      load_part<T, W>(g[r], grad + at, a.D - d0, vec & 8);
      load_part<T, W>(o, out + at, a.D - d0, vec & 8);
      float x = 0.0f;
#pragma unroll
      for (int k = 0; k < W; ++k) x = fmaf(o[k], g[r][k], x);
      delta0[r] = part_sum<LPK>(x);
      L[r] = lse[query[r] * a.H + head[r]];
    }
    slope2[r] = bias ? a.slopes[head[r]] * kLog2e : 0.0f;
    px[r] = bias ? a.x[3 * query[r]] : 0.0f;
    py[r] = bias ? a.x[3 * query[r] + 1] : 0.0f;
    pz[r] = bias ? a.x[3 * query[r] + 2] : 0.0f;
  }

  float m[kFewRows], acc[kFewRows][ACC][W], sum[kFewRows][SUMS];
#pragma unroll
  for (int r = 0; r < kFewRows; ++r) {
    m[r] = -INFINITY;
#pragma unroll
    for (int k = 0; k < SUMS; ++k) sum[r][k] = 0.0f;
#pragma unroll
    for (int u = 0; u < ACC; ++u)
#pragma unroll
      for (int k = 0; k < W; ++k) acc[r][u][k] = 0.0f;
  }

  const T* kp = static_cast<const T*>(a.k) + hk * a.k_head + d0;
  const T* vp = static_cast<const T*>(a.v) + hk * a.v_head + d0;
  const int64_t end = int64_t(it.col) + it.cols;
  // the keys of the next round load while this one's are worked on
  struct Round {
    uint4 k[kFewSteps], v[kFewSteps];
    float x[kFewSteps], y[kFewSteps], z[kFewSteps];
  };
  const auto fetch = [&](int64_t j0, Round& f) {
#pragma unroll
    for (int t = 0; t < kFewSteps; ++t) {
      const int64_t j = j0 + t * KPW + slot, jj = j < end ? j : end - 1;
      f.k[t] = raw_part<T, W, VEC>(kp + jj * a.k_row, a.D - d0);
      f.v[t] = raw_part<T, W, VEC>(vp + jj * a.v_row, a.D - d0);
      f.x[t] = bias ? a.y[3 * jj] : 0.0f;
      f.y[t] = bias ? a.y[3 * jj + 1] : 0.0f;
      f.z[t] = bias ? a.y[3 * jj + 2] : 0.0f;
    }
  };
  constexpr int kStride = kFewWarps * KPW * kFewSteps;
  Round next;
  const int64_t begin = int64_t(it.col) + warp * (KPW * kFewSteps);
  if (begin < end) fetch(begin, next);
  for (int64_t j0 = begin; j0 < end; j0 += kStride) {
    const Round now = next;
    if (j0 + kStride < end) fetch(j0 + kStride, next);
    float kv[kFewSteps][W], vv[kFewSteps][W];
    bool there[kFewSteps];
#pragma unroll
    for (int t = 0; t < kFewSteps; ++t) {
      there[t] = j0 + t * KPW + slot < end;
      widen_part<T, W>(kv[t], now.k[t]);
      widen_part<T, W>(vv[t], now.v[t]);
    }
#pragma unroll
    for (int r = 0; r < kFewRows; ++r) {
      float s[kFewSteps], d[kFewSteps], rd[kFewSteps];
#pragma unroll
      for (int t = 0; t < kFewSteps; ++t) {
        float x = 0.0f;
#pragma unroll
        for (int k = 0; k < W; ++k) x = fmaf(q[r][k], kv[t][k], x);
        x = part_sum<LPK>(x);
        d[t] = rd[t] = 0.0f;
        if (bias) {
          const float dx = px[r] - now.x[t], dy = py[r] - now.y[t], dz = pz[r] - now.z[t];
          const float sq = fmaf(dz, dz, fmaf(dy, dy, fmaf(dx, dx, 1e-30f)));
          rd[t] = tc::rsqrt_approx(sq);
          d[t] = sq * rd[t];
          x = fmaf(d[t], -slope2[r], x);
        }
        s[t] = there[t] ? x : -INFINITY;
      }
      if constexpr (!BACKWARD) {
        float top = m[r];
#pragma unroll
        for (int t = 0; t < kFewSteps; ++t) top = fmaxf(top, s[t]);
        const float ref = top == -INFINITY ? 0.0f : top, shrink = tc::ex2(m[r] - ref);
        m[r] = top;
        sum[r][1] *= shrink;
#pragma unroll
        for (int k = 0; k < W; ++k) acc[r][0][k] *= shrink;
#pragma unroll
        for (int t = 0; t < kFewSteps; ++t) {
          const float p = tc::ex2(s[t] - ref);
          sum[r][1] += p;
          if (there[t]) {  // the stand-in of a missing key may hold anything
#pragma unroll
            for (int k = 0; k < W; ++k) acc[r][0][k] = fmaf(p, vv[t][k], acc[r][0][k]);
          }
        }
      } else {
#pragma unroll
        for (int t = 0; t < kFewSteps; ++t) {
          float x = 0.0f;
#pragma unroll
          for (int k = 0; k < W; ++k) x = fmaf(g[r][k], vv[t][k], x);
          x = part_sum<LPK>(x);
          if (there[t]) {
            const float p = tc::ex2(s[t] - L[r]), ds = p * (x - delta0[r]);
            const float dx = px[r] - now.x[t], dy = py[r] - now.y[t], dz = pz[r] - now.z[t];
            const float u = ds * rd[t], w = p * rd[t];
            sum[r][0] += ds;
            sum[r][1] = fmaf(d[t], ds, sum[r][1]);
            sum[r][2] = fmaf(d[t], p, sum[r][2]);
            sum[r][3] = fmaf(u, dx, sum[r][3]);
            sum[r][4] = fmaf(u, dy, sum[r][4]);
            sum[r][5] = fmaf(u, dz, sum[r][5]);
            sum[r][6] = fmaf(w, dx, sum[r][6]);
            sum[r][7] = fmaf(w, dy, sum[r][7]);
            sum[r][8] = fmaf(w, dz, sum[r][8]);
            sum[r][9] += p;
#pragma unroll
            for (int k = 0; k < W; ++k) {
              acc[r][0][k] = fmaf(ds, kv[t][k], acc[r][0][k]);
              acc[r][1][k] = fmaf(p, kv[t][k], acc[r][1][k]);
            }
          }
        }
      }
    }
  }

  // the warp's groups of lanes, then the CTA's warps
#pragma unroll
  for (int r = 0; r < kFewRows; ++r) {
    float f = 1.0f;
    bool none = false;
    if constexpr (!BACKWARD) {
      float top = m[r];
#pragma unroll
      for (int o = LPK; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      // a group that saw no key above -inf has nothing to add; one whose weight underflows may hold NaN
      none = m[r] == -INFINITY && sum[r][1] == 0.0f;
      f = none ? 0.0f : tc::ex2(m[r] - (top == -INFINITY ? 0.0f : top));
      sum[r][0] = top;
      sum[r][1] *= f;
    }
#pragma unroll
    for (int u = 0; u < ACC; ++u) {
#pragma unroll
      for (int k = 0; k < W; ++k) {
        float x = none ? 0.0f : acc[r][u][k] * f;
#pragma unroll
        for (int o = LPK; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        if (slot == 0) s_acc[warp][r][u][d0 + k] = x;
      }
    }
#pragma unroll
    for (int k = BACKWARD ? 0 : 1; k < SUMS; ++k) {
#pragma unroll
      for (int o = LPK; o < 32; o <<= 1) sum[r][k] += __shfl_xor_sync(0xffffffffu, sum[r][k], o);
    }
    if (lane == 0) {
#pragma unroll
      for (int k = 0; k < SUMS; ++k) s_sum[warp][r][k] = sum[r][k];
    }
  }
  __syncthreads();
  if (warp >= kFewRows || first + warp >= row_count) return;
  const int r = warp, u = first + r;
  float* p = part + ((int64_t(it.slot) * a.H + hk * a.group + u % a.group) * kFewQueries + u / a.group) * width;
  float f[kFewWarps];
  if constexpr (!BACKWARD) {
    float top = -INFINITY, l = 0.0f;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) top = fmaxf(top, s_sum[w][r][0]);
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
      const float mw = s_sum[w][r][0], lw = s_sum[w][r][1];
      f[w] = mw == -INFINITY && lw == 0.0f ? 0.0f : tc::ex2(mw - (top == -INFINITY ? 0.0f : top));
      l += lw * f[w];  // the maxima pass over NaN, so that only the sums carry it
    }
    if (lane == 0) {
      p[DP] = top;
      p[DP + 1] = l;
    }
  } else {
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) f[w] = 1.0f;
    if (lane < 10) {
      float x = 0.0f;
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) x += s_sum[w][r][lane];
      p[DP + lane] = x;
    }
    float mine = delta0[0];
#pragma unroll
    for (int k = 1; k < kFewRows; ++k)
      if (r == k) mine = delta0[k];
    if (lane == 10) p[DP + 10] = mine;
  }
  for (int d = lane; d < a.D; d += 32) {
#pragma unroll
    for (int c = 0; c < ACC; ++c) {
      float x = 0.0f;
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) x += s_acc[w][r][c][d] * f[w];
      p[c * (DP + 16) + d] = x;
    }
  }
}

// Gradients of keys that one or two queries see: LPK lanes hold a key's components of K and V and those of its
// gradients, in fp32, and go over the query heads that share the key head.  The loads of two keys are in flight
// together.  A CTA takes part of an item of up to kTileRows keys that the same queries see.  fp32 is bound by reading K
// and V and writing their gradients once (705 MB of the case above: 143 us, 4.9 TB/s; by an entry a key 139), bf16 by the
// arithmetic of its eight components a lane (8 structures of 16,384 keys, 8 heads of 64 on 4: 297 MB, 111 us, 2.7
// TB/s; by an entry a key 124, on tiles 209).
template <typename T, int LPK, bool VEC>
__global__ void __launch_bounds__(32 * kFewWarps, kFewKeyCtas) few_key_kernel(const __grid_constant__ AttArgs a,
                                                                const AttItem* __restrict__ items, int vec,
                                                                const T* __restrict__ grad,
                                                                const float* __restrict__ lse,
                                                                const float* __restrict__ delta, T* __restrict__ dk,
                                                                T* __restrict__ dv, float* __restrict__ dy_part) {
  constexpr int W = 16 / int(sizeof(T)), KPW = 32 / LPK;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, slot = lane / LPK, d0 = (lane % LPK) * W;
  constexpr int KEYS = kFewWarps * KPW * kFewKeySteps;  // of a CTA
  constexpr unsigned CTAS = kTileRows / KEYS;           // of an item
  const int hk = int(blockIdx.y), cta0 = int(blockIdx.x % CTAS) * KEYS;
  const AttItem it = items[blockIdx.x / CTAS];
  if (cta0 >= it.rows) return;
  const int e0 = cta0 + warp * (KPW * kFewKeySteps) + slot;
  const bool bias = a.slopes != nullptr;
  int key[kFewKeySteps];  // past the end the last one, which is not stored again
#pragma unroll
  for (int t = 0; t < kFewKeySteps; ++t) key[t] = it.row + min(e0 + t * KPW, it.rows - 1);
  const T* kp = static_cast<const T*>(a.k) + hk * a.k_head + d0;
  const T* vp = static_cast<const T*>(a.v) + hk * a.v_head + d0;
  uint4 kr[kFewKeySteps], vr[kFewKeySteps];
  float y[kFewKeySteps][3];
#pragma unroll
  for (int t = 0; t < kFewKeySteps; ++t) {
    kr[t] = raw_part<T, W, VEC>(kp + int64_t(key[t]) * a.k_row, a.D - d0);
    vr[t] = raw_part<T, W, VEC>(vp + int64_t(key[t]) * a.v_row, a.D - d0);
#pragma unroll
    for (int c = 0; c < 3; ++c) y[t][c] = bias ? a.y[3 * int64_t(key[t]) + c] : 0.0f;
  }
#pragma unroll
  for (int t = 0; t < kFewKeySteps; ++t) {
    float kv[W], vv[W], gk[W], gv[W], f[3] = {0.0f, 0.0f, 0.0f};
    widen_part<T, W>(kv, kr[t]);
    widen_part<T, W>(vv, vr[t]);
#pragma unroll
    for (int k = 0; k < W; ++k) gk[k] = gv[k] = 0.0f;
    for (int n = 0; n < it.cols; ++n) {
      const int64_t i = int64_t(it.col) + n;
      for (int h = hk * a.group; h < (hk + 1) * a.group; ++h) {
        float q[W], g[W], s = 0.0f, x = 0.0f;
        load_part<T, W>(q, static_cast<const T*>(a.q) + i * a.q_row + h * a.q_head + d0, a.D - d0, vec & 1);
        load_part<T, W>(g, grad + (i * a.H + h) * a.D + d0, a.D - d0, vec & 8);
        const float L = lse[i * a.H + h], about = delta[i * a.H + h];
        float away[3] = {0.0f, 0.0f, 0.0f}, slope = 0.0f;
        if (bias) {
          slope = a.slopes[h];
#pragma unroll
          for (int c = 0; c < 3; ++c) away[c] = a.x[3 * i + c] - y[t][c];
        }
#pragma unroll
        for (int k = 0; k < W; ++k) {
          s = fmaf(q[k] * a.scale2, kv[k], s);
          x = fmaf(g[k], vv[k], x);
        }
        s = part_sum<LPK>(s);
        x = part_sum<LPK>(x);
        float rd = 0.0f;
        if (bias) {
          const float sq = fmaf(away[2], away[2], fmaf(away[1], away[1], fmaf(away[0], away[0], 1e-30f)));
          rd = tc::rsqrt_approx(sq);
          s = fmaf(sq * rd, -slope * kLog2e, s);
        }
        const float p = tc::ex2(s - L), ds = p * (x - about), e = slope * ds * rd;
#pragma unroll
        for (int c = 0; c < 3; ++c) f[c] = fmaf(e, away[c], f[c]);
#pragma unroll
        for (int k = 0; k < W; ++k) {
          gk[k] = fmaf(ds, q[k], gk[k]);
          gv[k] = fmaf(p, g[k], gv[k]);
        }
      }
    }
    if (e0 + t * KPW >= it.rows) continue;
    const int64_t at = int64_t(key[t]) * a.Hk + hk;
    alignas(16) T ok[W], ov[W];
#pragma unroll
    for (int k = 0; k < W; ++k) {
      ok[k] = from_float<T>(gk[k] * a.scale);
      ov[k] = from_float<T>(gv[k]);
    }
    if (vec & 16) {
      if (d0 < a.D) {
        *reinterpret_cast<uint4*>(dk + at * a.D + d0) = *reinterpret_cast<const uint4*>(ok);
        *reinterpret_cast<uint4*>(dv + at * a.D + d0) = *reinterpret_cast<const uint4*>(ov);
      }
    } else {
#pragma unroll
      for (int k = 0; k < W; ++k) {
        if (d0 + k < a.D) {
          dk[at * a.D + d0 + k] = ok[k];
          dv[at * a.D + d0 + k] = ov[k];
        }
      }
    }
    if (bias && lane % LPK == 0) {
#pragma unroll
      for (int c = 0; c < 3; ++c) dy_part[at * 3 + c] = f[c];
    }
  }
}

template <typename T, bool BACKWARD>
int few(const AttArgs& a, const AttItem* items, int64_t count, int DP, int width, const T* out, const T* grad,
        const float* lse, float* part, cudaStream_t s) {
  if (count == 0) return Y3B_OK;
  constexpr int W = 16 / int(sizeof(T));
  const auto fits = [&](const void* p, int64_t row, int64_t head) {
    return a.D % W == 0 && row % W == 0 && head % W == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  };
  const int64_t dense = int64_t(a.H) * a.D;
  const int vec = (fits(a.q, a.q_row, a.q_head) ? 1 : 0) |
                  (BACKWARD && fits(out, dense, a.D) && fits(grad, dense, a.D) ? 8 : 0);
  const bool loads = fits(a.k, a.k_row, a.k_head) && fits(a.v, a.v_row, a.v_head);
  const int64_t blocks = (kFewQueries * a.group + kFewRows - 1) / kFewRows, grid = count * a.Hk * blocks;
  if (grid > INT32_MAX) return fail(Y3B_ERR_UNSUPPORTED, "structure_attention: too many chunks");
#define Y3B_FEW(LPK)                                                                                           \
  do {                                                                                                         \
    if (loads)                                                                                                 \
      few_kernel<T, LPK, BACKWARD, true>                                                                       \
          <<<unsigned(grid), 32 * kFewWarps, 0, s>>>(a, items, DP, width, vec, out, grad, lse, part);          \
    else                                                                                                       \
      few_kernel<T, LPK, BACKWARD, false>                                                                      \
          <<<unsigned(grid), 32 * kFewWarps, 0, s>>>(a, items, DP, width, vec, out, grad, lse, part);          \
  } while (0)
  const int lanes = (a.D + W - 1) / W;
  if (lanes <= 4) Y3B_FEW(4);
  else if (lanes <= 8) Y3B_FEW(8);
  else if (lanes <= 16) Y3B_FEW(16);
  else if constexpr (sizeof(T) == 4) Y3B_FEW(32);
#undef Y3B_FEW
  Y3B_LAUNCH_CHECK();
  return Y3B_OK;
}

}  // namespace

template <typename T>
int attention_few_key(const AttArgs& a, const AttItem* items, int64_t count, const T* grad, const float* lse,
                      const float* delta, T* dk, T* dv, float* dy_part, cudaStream_t s) {
  constexpr int W = 16 / int(sizeof(T));
  const auto fits = [&](const void* p, int64_t row, int64_t head) {
    return a.D % W == 0 && row % W == 0 && head % W == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  };
  const int vec = (fits(a.q, a.q_row, a.q_head) ? 1 : 0) | (fits(grad, int64_t(a.H) * a.D, a.D) ? 8 : 0) |
                  (fits(dk, a.D, a.D) && fits(dv, a.D, a.D) ? 16 : 0);
  const bool loads = fits(a.k, a.k_row, a.k_head) && fits(a.v, a.v_row, a.v_head);
#define Y3B_FEW_KEY(LPK)                                                                                       \
  do {                                                                                                         \
    const int64_t grid = count * (kTileRows / (kFewWarps * (32 / LPK) * kFewKeySteps));                        \
    if (grid > INT32_MAX) return fail(Y3B_ERR_UNSUPPORTED, "structure_attention: too many keys");              \
    const dim3 ctas(unsigned(grid), unsigned(a.Hk));                                                           \
    if (loads)                                                                                                 \
      few_key_kernel<T, LPK, true><<<ctas, 32 * kFewWarps, 0, s>>>(a, items, vec, grad, lse, delta, dk, dv,    \
                                                                   dy_part);                                   \
    else                                                                                                       \
      few_key_kernel<T, LPK, false><<<ctas, 32 * kFewWarps, 0, s>>>(a, items, vec, grad, lse, delta, dk, dv,   \
                                                                    dy_part);                                  \
  } while (0)
  const int lanes = (a.D + W - 1) / W;
  if (lanes <= 4) Y3B_FEW_KEY(4);
  else if (lanes <= 8) Y3B_FEW_KEY(8);
  else if (lanes <= 16) Y3B_FEW_KEY(16);
  else if constexpr (sizeof(T) == 4) Y3B_FEW_KEY(32);
#undef Y3B_FEW_KEY
  Y3B_LAUNCH_CHECK();
  return Y3B_OK;
}

template <typename T>
int attention_few_forward(const AttArgs& a, const AttItem* items, int64_t count, int DP, int width, float* part,
                          cudaStream_t s) {
  return few<T, false>(a, items, count, DP, width, nullptr, nullptr, nullptr, part, s);
}

template <typename T>
int attention_few_query(const AttArgs& a, const AttItem* items, int64_t count, int DP, int width, const T* out,
                        const T* grad, const float* lse, float* part, cudaStream_t s) {
  return few<T, true>(a, items, count, DP, width, out, grad, lse, part, s);
}

template int attention_few_key<float>(const AttArgs&, const AttItem*, int64_t, const float*, const float*, const float*,
                                      float*, float*, float*, cudaStream_t);
template int attention_few_key<__nv_bfloat16>(const AttArgs&, const AttItem*, int64_t, const __nv_bfloat16*, const float*,
                                              const float*, __nv_bfloat16*, __nv_bfloat16*, float*, cudaStream_t);
template int attention_few_forward<float>(const AttArgs&, const AttItem*, int64_t, int, int, float*, cudaStream_t);
template int attention_few_forward<__nv_bfloat16>(const AttArgs&, const AttItem*, int64_t, int, int, float*,
                                                  cudaStream_t);
template int attention_few_query<float>(const AttArgs&, const AttItem*, int64_t, int, int, const float*, const float*,
                                        const float*, float*, cudaStream_t);
template int attention_few_query<__nv_bfloat16>(const AttArgs&, const AttItem*, int64_t, int, int,
                                                const __nv_bfloat16*, const __nv_bfloat16*, const float*, float*,
                                                cudaStream_t);

}  // namespace y3b
