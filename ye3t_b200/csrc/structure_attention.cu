// Attention among the atoms of each structure of a packed batch, scores lowered with
// distance:
//   s_ij = scale q_i . k_j - slope_h |x_i - y_j|      j over the keys of i's structure
//   P_ij = exp(s_ij) / sum_j exp(s_ij)                o_i = sum_j P_ij v_j
// and its gradients, with dP_ij = do_i . v_j, delta_i = sum_j P_ij dP_ij and
// dS_ij = P_ij (dP_ij - delta_i):
//   dq_i = scale sum_j dS_ij k_j     dk_j = scale sum_i dS_ij q_i     dv_j = sum_i P_ij do_i
//   dslope_h = -sum_ij dS_ij |x_i - y_j|
//   dx_i = -sum_hj slope_h dS_ij (x_i - y_j) / |x_i - y_j|, dy_j the same summed over i with
//   the other sign; a pair at distance zero has no direction and contributes nothing.
// Key head h / (H / Hk) serves query head h.  A row whose structure has no keys, or whose
// scores are all -inf, gives zeros.  Scores and statistics are kept in fp32 and in
// units of log2; lse holds m + log2(l), +inf for rows that give zeros (P = 0 in the backward).
//
// Row kernels: one warp per (row, head); lanes take 32 columns at a time for the scores and
// then the D components for the sums.
#include <algorithm>

#include "structure_attention_few.cuh"
#include "structure_attention_small.cuh"
#include "structure_attention_tile.cuh"

namespace y3b {
namespace {

constexpr int kRowWarps = 4;
constexpr int kRowAcc = kAttMaxWidth / 32;

struct Range {
  int64_t b, e;
};

// Rows of a structure, within the array whatever the offsets hold.
__device__ __forceinline__ Range rows_of(const int32_t* off, int structure, int64_t n) {
  Range r{off[structure], off[structure + 1]};
  if (r.b < 0) r.b = 0;
  if (r.e > n) r.e = n;
  return r;
}

template <typename T>
__device__ __forceinline__ float dot(const float* __restrict__ s, const T* __restrict__ g, int D) {
  float acc = 0.0f;
#pragma unroll 4
  for (int d = 0; d < D; ++d) acc = fmaf(s[d], to_float(g[d]), acc);
  return acc;
}

struct Apart {
  float x, y, z, d;
};
__device__ __forceinline__ Apart apart(float ax, float ay, float az, const float* __restrict__ p) {
  Apart r;
  r.x = ax - p[0];
  r.y = ay - p[1];
  r.z = az - p[2];
  r.d = sqrtf(fmaf(r.x, r.x, fmaf(r.y, r.y, r.z * r.z)));
  return r;
}

template <typename T>
__global__ void __launch_bounds__(32 * kRowWarps) row_forward_kernel(AttArgs a, const int2* __restrict__ rows,
                                                                     int64_t row_count, T* __restrict__ out,
                                                                     float* __restrict__ lse) {
  __shared__ float s_q[kRowWarps][kAttMaxWidth];
  __shared__ float s_p[kRowWarps][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t task = blockIdx.x * int64_t(kRowWarps) + w;
  if (task >= row_count * a.H) return;
  const int2 of = rows[task / a.H];  // (row, structure)
  const int64_t i = of.x;
  const int h = int(task % a.H), hk = h / a.group;
  const T* q = static_cast<const T*>(a.q) + i * a.q_row + h * a.q_head;
  const T* k = static_cast<const T*>(a.k) + hk * a.k_head;
  const T* v = static_cast<const T*>(a.v) + hk * a.v_head;
  for (int d = lane; d < a.D; d += 32) s_q[w][d] = to_float(q[d]) * a.scale2;
  float slope2 = 0.0f, px = 0.0f, py = 0.0f, pz = 0.0f;
  if (a.slopes) {
    slope2 = a.slopes[h] * kLog2e;
    px = a.x[3 * i];
    py = a.x[3 * i + 1];
    pz = a.x[3 * i + 2];
  }
  __syncwarp();
  const Range r = rows_of(a.k_off, of.y, a.nk);
  float m = -INFINITY, l = 0.0f, acc[kRowAcc];
#pragma unroll
  for (int t = 0; t < kRowAcc; ++t) acc[t] = 0.0f;
  for (int64_t j0 = r.b; j0 < r.e; j0 += 32) {
    const int64_t j = j0 + lane;
    const bool ok = j < r.e;
    float s = -INFINITY;
    if (ok) {
      s = dot(s_q[w], k + j * a.k_row, a.D);
      if (a.slopes) s = fmaf(-slope2, apart(px, py, pz, a.y + 3 * j).d, s);
    }
    const float top = fmaxf(m, warp_max(s));
    const float ref = top == -INFINITY ? 0.0f : top;
    const float shrink = exp2f(m - ref);
    const float p = ok ? exp2f(s - ref) : 0.0f;
    l = l * shrink + warp_sum(p);
    m = top;
    s_p[w][lane] = p;
    __syncwarp();
    const int n = r.e - j0 < 32 ? int(r.e - j0) : 32;
#pragma unroll
    for (int t = 0; t < kRowAcc; ++t) {
      const int d = lane + 32 * t;
      if (d < a.D) {
        float x = acc[t] * shrink;
        for (int c = 0; c < n; ++c) x = fmaf(s_p[w][c], to_float(v[(j0 + c) * a.v_row + d]), x);
        acc[t] = x;
      }
    }
    __syncwarp();
  }
  const bool none = r.b >= r.e || (m == -INFINITY && l == 0.0f);
  const float inv = none ? 0.0f : 1.0f / l;
#pragma unroll
  for (int t = 0; t < kRowAcc; ++t) {
    const int d = lane + 32 * t;
    if (d < a.D) out[(i * a.H + h) * a.D + d] = from_float<T>(none ? 0.0f : acc[t] * inv);
  }
  if (lane == 0) lse[i * a.H + h] = none ? INFINITY : m + log2f(l);
}

// Query side of the backward: delta, dq and this row's parts of dslope and dx.
template <typename T>
__global__ void __launch_bounds__(32 * kRowWarps) row_backward_query_kernel(
    AttArgs a, const int2* __restrict__ rows, int64_t row_count, const T* __restrict__ grad,
    const float* __restrict__ lse, float* __restrict__ delta, T* __restrict__ dq, float* __restrict__ dslope_part,
    float* __restrict__ dx_part) {
  __shared__ float s_q[kRowWarps][kAttMaxWidth];
  __shared__ float s_g[kRowWarps][kAttMaxWidth];
  __shared__ float s_p[kRowWarps][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t task = blockIdx.x * int64_t(kRowWarps) + w;
  if (task >= row_count * a.H) return;
  const int2 of = rows[task / a.H];  // (row, structure)
  const int64_t i = of.x;
  const int h = int(task % a.H), hk = h / a.group;
  const T* q = static_cast<const T*>(a.q) + i * a.q_row + h * a.q_head;
  const T* k = static_cast<const T*>(a.k) + hk * a.k_head;
  const T* v = static_cast<const T*>(a.v) + hk * a.v_head;
  for (int d = lane; d < a.D; d += 32) {
    s_q[w][d] = to_float(q[d]) * a.scale2;
    s_g[w][d] = to_float(grad[(i * a.H + h) * a.D + d]);
  }
  float slope = 0.0f, px = 0.0f, py = 0.0f, pz = 0.0f;
  if (a.slopes) {
    slope = a.slopes[h];
    px = a.x[3 * i];
    py = a.x[3 * i + 1];
    pz = a.x[3 * i + 2];
  }
  const float slope2 = slope * kLog2e;
  __syncwarp();
  const Range r = rows_of(a.k_off, of.y, a.nk);
  const float L = lse[i * a.H + h];
  float dl = 0.0f;
  for (int64_t j = r.b + lane; j < r.e; j += 32) {
    float s = dot(s_q[w], k + j * a.k_row, a.D);
    if (a.slopes) s = fmaf(-slope2, apart(px, py, pz, a.y + 3 * j).d, s);
    dl = fmaf(exp2f(s - L), dot(s_g[w], v + j * a.v_row, a.D), dl);
  }
  dl = warp_sum(dl);
  float acc[kRowAcc], sd = 0.0f, fx = 0.0f, fy = 0.0f, fz = 0.0f;
#pragma unroll
  for (int t = 0; t < kRowAcc; ++t) acc[t] = 0.0f;
  for (int64_t j0 = r.b; j0 < r.e; j0 += 32) {
    const int64_t j = j0 + lane;
    float ds = 0.0f;
    if (j < r.e) {
      float s = dot(s_q[w], k + j * a.k_row, a.D);
      Apart p{};
      if (a.slopes) {
        p = apart(px, py, pz, a.y + 3 * j);
        s = fmaf(-slope2, p.d, s);
      }
      ds = exp2f(s - L) * (dot(s_g[w], v + j * a.v_row, a.D) - dl);
      if (a.slopes) {
        sd = fmaf(ds, p.d, sd);
        const float u = p.d > 0.0f ? ds / p.d : 0.0f;
        fx = fmaf(u, p.x, fx);
        fy = fmaf(u, p.y, fy);
        fz = fmaf(u, p.z, fz);
      }
    }
    s_p[w][lane] = ds;
    __syncwarp();
    const int n = r.e - j0 < 32 ? int(r.e - j0) : 32;
#pragma unroll
    for (int t = 0; t < kRowAcc; ++t) {
      const int d = lane + 32 * t;
      if (d < a.D) {
        float x = acc[t];
        for (int c = 0; c < n; ++c) x = fmaf(s_p[w][c], to_float(k[(j0 + c) * a.k_row + d]), x);
        acc[t] = x;
      }
    }
    __syncwarp();
  }
#pragma unroll
  for (int t = 0; t < kRowAcc; ++t) {
    const int d = lane + 32 * t;
    if (d < a.D) dq[(i * a.H + h) * a.D + d] = from_float<T>(acc[t] * a.scale);
  }
  if (lane == 0) delta[i * a.H + h] = dl;
  if (a.slopes) {
    sd = warp_sum(sd);
    fx = warp_sum(fx);
    fy = warp_sum(fy);
    fz = warp_sum(fz);
    if (lane == 0) {
      dslope_part[i * a.H + h] = -sd;
      dx_part[(i * a.H + h) * 3] = -slope * fx;
      dx_part[(i * a.H + h) * 3 + 1] = -slope * fy;
      dx_part[(i * a.H + h) * 3 + 2] = -slope * fz;
    }
  }
}

// Key side: dk, dv and dy of one (key, key head), over the query heads that share it.
template <typename T>
__global__ void __launch_bounds__(32 * kRowWarps) row_backward_key_kernel(
    AttArgs a, const int2* __restrict__ rows, int64_t row_count, const T* __restrict__ grad,
    const float* __restrict__ lse, const float* __restrict__ delta, T* __restrict__ dk, T* __restrict__ dv,
    float* __restrict__ dy_part) {
  __shared__ float s_k[kRowWarps][kAttMaxWidth];
  __shared__ float s_v[kRowWarps][kAttMaxWidth];
  __shared__ float s_p[kRowWarps][32];
  __shared__ float s_d[kRowWarps][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t task = blockIdx.x * int64_t(kRowWarps) + w;
  if (task >= row_count * a.Hk) return;
  const int2 of = rows[task / a.Hk];  // (row, structure)
  const int64_t j = of.x;
  const int hk = int(task % a.Hk);
  const T* k = static_cast<const T*>(a.k) + j * a.k_row + hk * a.k_head;
  const T* v = static_cast<const T*>(a.v) + j * a.v_row + hk * a.v_head;
  for (int d = lane; d < a.D; d += 32) {
    s_k[w][d] = to_float(k[d]) * a.scale2;
    s_v[w][d] = to_float(v[d]);
  }
  __syncwarp();
  const Range r = rows_of(a.q_off, of.y, a.nq);
  float acc_k[kRowAcc], acc_v[kRowAcc], fx = 0.0f, fy = 0.0f, fz = 0.0f;
#pragma unroll
  for (int t = 0; t < kRowAcc; ++t) acc_k[t] = acc_v[t] = 0.0f;
  float px = 0.0f, py = 0.0f, pz = 0.0f;
  if (a.slopes) {
    px = a.y[3 * j];
    py = a.y[3 * j + 1];
    pz = a.y[3 * j + 2];
  }
  for (int h = hk * a.group; h < (hk + 1) * a.group; ++h) {
    const T* q = static_cast<const T*>(a.q) + h * a.q_head;
    const T* g = grad + h * a.D;
    const int64_t g_row = int64_t(a.H) * a.D;
    const float slope = a.slopes ? a.slopes[h] : 0.0f, slope2 = slope * kLog2e;
    for (int64_t i0 = r.b; i0 < r.e; i0 += 32) {
      const int64_t i = i0 + lane;
      float p = 0.0f, ds = 0.0f;
      if (i < r.e) {
        float s = dot(s_k[w], q + i * a.q_row, a.D);
        Apart t{};
        if (a.slopes) {
          t = apart(px, py, pz, a.x + 3 * i);
          s = fmaf(-slope2, t.d, s);
        }
        p = exp2f(s - lse[i * a.H + h]);
        ds = p * (dot(s_v[w], g + i * g_row, a.D) - delta[i * a.H + h]);
        if (a.slopes) {
          const float u = t.d > 0.0f ? slope * ds / t.d : 0.0f;
          fx = fmaf(u, t.x, fx);
          fy = fmaf(u, t.y, fy);
          fz = fmaf(u, t.z, fz);
        }
      }
      s_p[w][lane] = p;
      s_d[w][lane] = ds;
      __syncwarp();
      const int n = r.e - i0 < 32 ? int(r.e - i0) : 32;
#pragma unroll
      for (int t = 0; t < kRowAcc; ++t) {
        const int d = lane + 32 * t;
        if (d < a.D) {
          float x = acc_k[t], y = acc_v[t];
          for (int c = 0; c < n; ++c) {
            x = fmaf(s_d[w][c], to_float(q[(i0 + c) * a.q_row + d]), x);
            y = fmaf(s_p[w][c], to_float(g[(i0 + c) * g_row + d]), y);
          }
          acc_k[t] = x;
          acc_v[t] = y;
        }
      }
      __syncwarp();
    }
  }
#pragma unroll
  for (int t = 0; t < kRowAcc; ++t) {
    const int d = lane + 32 * t;
    if (d < a.D) {
      dk[(j * a.Hk + hk) * a.D + d] = from_float<T>(acc_k[t] * a.scale);
      dv[(j * a.Hk + hk) * a.D + d] = from_float<T>(acc_v[t]);
    }
  }
  if (a.slopes) {
    fx = warp_sum(fx);
    fy = warp_sum(fy);
    fz = warp_sum(fz);
    if (lane == 0) {
      // the direction here is y - x, so the gradient by y carries the same sign as dx
      dy_part[(j * a.Hk + hk) * 3] = -fx;
      dy_part[(j * a.Hk + hk) * 3 + 1] = -fy;
      dy_part[(j * a.Hk + hk) * 3 + 2] = -fz;
    }
  }
}

// What the parts add up to, in one launch: dx[i] = sum over heads of dx_part (and of dy_part where queries and keys
// are the same atoms), dy[j] likewise, one thread a component; then dslope[h] = sum over rows, one CTA a head,
// in fp64 and a fixed order.
struct FinishArgs {
  const float* dx_part;
  const float* dy_part;
  const float* slope_part;
  float* dx;
  float* dy;  // null: dx takes both sums
  float* dslopes;
  int64_t nq, nk;
  int H, Hk;
  unsigned x_ctas, y_ctas;
};
constexpr int kFinishThreads = 512;

__device__ __forceinline__ float head_sum(const float* part, int64_t i, int c, int heads) {
  float sum = 0.0f;
#pragma unroll 4
  for (int h = 0; h < heads; ++h) sum += part[(i * heads + h) * 3 + c];
  return sum;
}

__global__ void __launch_bounds__(kFinishThreads) finish_kernel(const __grid_constant__ FinishArgs a) {
  __shared__ double s[kFinishThreads];
  if (blockIdx.x < a.x_ctas + a.y_ctas) {
    const bool keys = blockIdx.x >= a.x_ctas;
    const int64_t t = (blockIdx.x - (keys ? a.x_ctas : 0u)) * int64_t(kFinishThreads) + threadIdx.x;
    if (t >= (keys ? a.nk : a.nq) * 3) return;
    const int64_t i = t / 3;
    const int c = int(t - 3 * i);
    if (keys) {
      a.dy[t] = head_sum(a.dy_part, i, c, a.Hk);
    } else {
      float sum = head_sum(a.dx_part, i, c, a.H);
      if (a.dy == nullptr && a.nk > 0) sum += head_sum(a.dy_part, i, c, a.Hk);
      a.dx[t] = sum;
    }
    return;
  }
  const int h = int(blockIdx.x - a.x_ctas - a.y_ctas);
  double sum = 0.0;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < a.nq; i += kFinishThreads) sum += double(a.slope_part[i * a.H + h]);
  s[threadIdx.x] = sum;
  __syncthreads();
  for (int o = kFinishThreads / 2; o > 0; o >>= 1) {
    if (int(threadIdx.x) < o) s[threadIdx.x] += s[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) a.dslopes[h] = float(s[0]);
}

int unpack(const y3b_structure_attention_args* p, const char* what, AttArgs* a) {
  Y3B_CHECK_ARG(p != nullptr, "%s: null arguments", what);
  Y3B_CHECK_ARG(p->dtype == Y3B_F32 || p->dtype == Y3B_BF16, "%s: dtype must be F32 or BF16", what);
  Y3B_CHECK_ARG(p->heads >= 1 && p->key_heads >= 1 && p->heads % p->key_heads == 0,
                "%s: the query heads (%d) must be a multiple of the key heads (%d)", what, p->heads, p->key_heads);
  Y3B_CHECK_ARG(p->heads <= 1024, "%s: at most 1024 heads", what);
  Y3B_CHECK_ARG(p->width >= 1 && p->width <= kAttMaxWidth, "%s: head width 1 to %d, got %d", what, kAttMaxWidth,
                p->width);
  Y3B_CHECK_ARG(p->query_count >= 0 && p->key_count >= 0 && p->structure_count >= 0 &&
                    p->query_count <= INT32_MAX && p->key_count <= INT32_MAX && p->structure_count < INT32_MAX,
                "%s: bad query, key or structure count", what);
  if (p->query_count > 0 || p->key_count > 0) {
    Y3B_CHECK_ARG(p->structure_count >= 1, "%s: atoms without a structure", what);
    Y3B_CHECK_ARG(p->query_offsets && p->key_offsets, "%s: null offsets", what);
  }
  Y3B_CHECK_ARG(p->query_count == 0 || p->query, "%s: null query argument", what);
  Y3B_CHECK_ARG(p->key_count == 0 || (p->key && p->value), "%s: null key or value", what);
  Y3B_CHECK_ARG((p->slopes != nullptr) || (!p->positions && !p->key_positions), "%s: positions without slopes", what);
  if (p->slopes) {
    Y3B_CHECK_ARG(p->query_count == 0 || p->positions, "%s: slopes without positions", what);
    Y3B_CHECK_ARG(p->key_count == 0 || p->key_positions, "%s: slopes without key positions", what);
  }
  Y3B_CHECK_ARG(p->small_32_count >= 0 && p->small_64_count >= 0 &&
                    (p->small_32_count + p->small_64_count == 0 || p->small),
                "%s: bad table of small structures", what);
  Y3B_CHECK_ARG(p->few_item_count >= 0 && p->few_join_count >= 0 &&
                    (p->few_item_count == 0 || (p->few_items && p->few_joins && p->few_join_count > 0)),
                "%s: bad table of few-query structures", what);
  Y3B_CHECK_ARG(p->forward_item_count >= 0 && p->forward_join_count >= 0 && p->forward_slot_count >= 0 &&
                    (p->forward_item_count == 0 || p->forward_items) && (p->forward_join_count == 0 || p->forward_joins),
                "%s: bad table of the forward", what);
  Y3B_CHECK_ARG(p->query_item_count >= 0 && p->query_join_count >= 0 && p->query_slot_count >= 0 &&
                    p->query_row_count >= 0 && p->key_item_count >= 0 && p->key_join_count >= 0 &&
                    p->key_slot_count >= 0 && p->key_row_count >= 0 && p->few_key_item_count >= 0 &&
                    p->few_key_item_count <= p->key_item_count && (p->few_key_item_count == 0 || p->query_count > 0),
                "%s: negative table size", what);
  Y3B_CHECK_ARG((p->query_item_count == 0 || p->query_items) && (p->query_join_count == 0 || p->query_joins) &&
                    (p->query_row_count == 0 || p->query_rows) && (p->key_item_count == 0 || p->key_items) &&
                    (p->key_join_count == 0 || p->key_joins) && (p->key_row_count == 0 || p->key_rows),
                "%s: null table", what);
  a->H = p->heads;
  a->Hk = p->key_heads;
  a->D = p->width;
  a->group = p->heads / p->key_heads;
  a->nq = p->query_count;
  a->nk = p->key_count;
  a->q = p->query;
  a->k = p->key;
  a->v = p->value;
  a->q_row = p->query_row_stride;
  a->q_head = p->query_head_stride;
  a->k_row = p->key_row_stride;
  a->k_head = p->key_head_stride;
  a->v_row = p->value_row_stride;
  a->v_head = p->value_head_stride;
  a->slopes = p->slopes;
  a->x = p->slopes ? p->positions : nullptr;
  a->y = p->slopes ? p->key_positions : nullptr;
  a->scale = p->scale;
  a->scale2 = p->scale * kLog2e;
  a->q_off = p->query_offsets;
  a->k_off = p->key_offsets;
  return Y3B_OK;
}

// ---------------------------------------------------------------------------
// Operands for the tile kernels: rows padded to a multiple of 8 values, fp32 as three bf16
// pieces.  A non-finite value keeps its first piece and zeros for the rest.  One thread per 8
// values of one head of one row.
struct PackSource {
  const void* p;
  int64_t row, head, rows;
  int heads;
  __nv_bfloat16* out;
};
struct PackArgs {
  PackSource s[4];
  int D, chunks;
};

template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ PackArgs a) {
  const PackSource& o = a.s[blockIdx.y];
  const int64_t per_row = int64_t(o.heads) * a.chunks, total = o.rows * per_row, piece = total * 8;
  for (int64_t t = blockIdx.x * int64_t(256) + threadIdx.x; t < total; t += int64_t(gridDim.x) * 256) {
    const int64_t r = t / per_row;
    const int u = int(t - r * per_row), h = u / a.chunks, c = u - h * a.chunks;
    const T* src = static_cast<const T*>(o.p) + r * o.row + h * o.head + c * 8;
    const int n = a.D - c * 8;
    uint32_t out[3][4];
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
      const float x = k < n ? to_float(src[k]) : 0.0f, y = k + 1 < n ? to_float(src[k + 1]) : 0.0f;
      if constexpr (sizeof(T) == 4) {
        uint32_t q[3];
        split_pair<3>(x, y, q);
        // the rest of a value that is not finite in bf16 would be NaN
        const uint32_t keep = ((q[0] & 0x7f80u) == 0x7f80u ? 0u : 0xffffu) |
                              ((q[0] & 0x7f800000u) == 0x7f800000u ? 0u : 0xffff0000u);
        out[0][k / 2] = q[0];
        out[1][k / 2] = q[1] & keep;
        out[2][k / 2] = q[2] & keep;
      } else {
        out[0][k / 2] = tc::bf16x2(x, y);
      }
    }
#pragma unroll
    for (int p = 0; p < (sizeof(T) == 4 ? 3 : 1); ++p)
      *reinterpret_cast<uint4*>(o.out + p * piece + t * 8) = make_uint4(out[p][0], out[p][1], out[p][2], out[p][3]);
  }
}

// Joins of split items, one warp a row, four a CTA.  Partial results lie at ((slot * heads + head) * RS + row) * W
// floats: RS is kTileRows, or kFewQueries for the few-query kernels.

template <typename T>
__global__ void __launch_bounds__(128) join_forward_kernel(const AttJoin* __restrict__ joins,
                                                           const float* __restrict__ part, int W, int DP, int D, int H,
                                                           T* __restrict__ out, float* __restrict__ lse) {
  constexpr int RS = kTileRows;
  const unsigned ctas = unsigned(RS + 3) / 4, task = blockIdx.x / ctas;
  const AttJoin jn = joins[task / unsigned(H)];
  const int h = int(task % unsigned(H)), lane = threadIdx.x & 31;
  const int r = int(blockIdx.x % ctas) * 4 + (threadIdx.x >> 5);
  if (r >= jn.rows) return;
  const int64_t step = int64_t(H) * RS * W;
  const float* p = part + ((int64_t(jn.first) * H + h) * RS + r) * W;
  float m = -INFINITY;
  for (int k = lane; k < jn.count; k += 32) m = fmaxf(m, p[k * step + DP]);
  m = warp_max(m);
  const float ref = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  for (int k = lane; k < jn.count; k += 32) l += p[k * step + DP + 1] * exp2f(p[k * step + DP] - ref);
  l = warp_sum(l);
  const bool none = m == -INFINITY && l == 0.0f;
  const int64_t at = (int64_t(jn.row) + r) * H + h;
  const float inv = none ? 0.0f : 1.0f / l;
  float o[kAttMaxWidth / 32] = {};
  for (int k0 = 0; k0 < jn.count; k0 += 32) {
    // lane k weighs part k0 + k; a part without any score above -inf holds zeros, one whose weight underflows may
    // hold NaN
    float weight = 0.0f;
    if (k0 + lane < jn.count) {
      const float mk = p[(k0 + lane) * step + DP];
      if (!(mk == -INFINITY && p[(k0 + lane) * step + DP + 1] == 0.0f)) weight = exp2f(mk - ref);
    }
    const int n = jn.count - k0 < 32 ? jn.count - k0 : 32;
#pragma unroll 8
    for (int k = 0; k < n; ++k) {
      const float f = __shfl_sync(0xffffffffu, weight, k);
#pragma unroll
      for (int t = 0; t < kAttMaxWidth / 32; ++t) {
        const int d = lane + 32 * t;
        if (d < D) {
          o[t] = fmaf(p[(k0 + k) * step + d], f, o[t]);
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < kAttMaxWidth / 32; ++t) {
    const int d = lane + 32 * t;
    if (d < D) out[at * D + d] = from_float<T>(none ? 0.0f : o[t] * inv);
  }
  if (lane == 0) lse[at] = none ? INFINITY : m + log2f(l);
}

// The same where one or two rows have many parts: a CTA a (join, head, query), whose warps take every fourth part.
template <typename T>
__global__ void __launch_bounds__(128) join_few_kernel(const AttJoin* __restrict__ joins, const float* __restrict__ part,
                                                       int W, int DP, int D, int H, T* __restrict__ out,
                                                       float* __restrict__ lse) {
  __shared__ float s_o[4][kAttMaxWidth];
  __shared__ float s_m[4], s_l[4];
  const unsigned task = blockIdx.x / kFewQueries;
  const AttJoin jn = joins[task / unsigned(H)];
  const int h = int(task % unsigned(H)), r = int(blockIdx.x % kFewQueries);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (r >= jn.rows) return;
  const int64_t step = int64_t(H) * kFewQueries * W;
  const float* p = part + ((int64_t(jn.first) * H + h) * kFewQueries + r) * W;
  float m = -INFINITY;
  for (int k = threadIdx.x; k < jn.count; k += 128) m = fmaxf(m, p[k * step + DP]);
  m = warp_max(m);
  if (lane == 0) s_m[warp] = m;
  __syncthreads();
  m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  const float ref = m == -INFINITY ? 0.0f : m;
  float o[kAttMaxWidth / 32] = {}, l = 0.0f;
#pragma unroll 4
  for (int k = warp; k < jn.count; k += 4) {
    // a part without any score above -inf holds zeros, one whose weight underflows may hold NaN
    const float mk = p[k * step + DP], lk = p[k * step + DP + 1];
    const float f = mk == -INFINITY && lk == 0.0f ? 0.0f : exp2f(mk - ref);
    l += lk * f;  // NaN where the part's scores held one, whatever its maximum
#pragma unroll
    for (int t = 0; t < kAttMaxWidth / 32; ++t) {
      const int d = lane + 32 * t;
      const float x = d < D ? p[k * step + d] : 0.0f;
      o[t] = fmaf(x, f, o[t]);
    }
  }
#pragma unroll
  for (int t = 0; t < kAttMaxWidth / 32; ++t) s_o[warp][lane + 32 * t] = o[t];
  if (lane == 0) s_l[warp] = l;
  __syncthreads();
  l = (s_l[0] + s_l[1]) + (s_l[2] + s_l[3]);
  const bool none = m == -INFINITY && l == 0.0f;
  const int64_t at = (int64_t(jn.row) + r) * H + h;
  const int d = threadIdx.x;
  if (d < D)
    out[at * D + d] = from_float<T>(none ? 0.0f : ((s_o[0][d] + s_o[1][d]) + (s_o[2][d] + s_o[3][d])) / l);
  if (d == 0) lse[at] = none ? INFINITY : m + log2f(l);
}

__device__ __forceinline__ float sum_parts(const float* p, int64_t step, int count) {
  float s = 0.0f;
#pragma unroll 8
  for (int k = 0; k < count; ++k) s += p[k * step];
  return s;
}

// FEW: one row a CTA, its components over all threads (few rows of many parts: 8 structures of 16,384 keys, 8 heads,
// 14 us, by a warp a row 36); else four rows.
template <typename T, bool FEW>
__global__ void __launch_bounds__(128) join_query_kernel(const AttJoin* __restrict__ joins,
                                                         const float* __restrict__ part, int RS, int W, int DP, int D,
                                                         int H, float scale, bool fix, const float* __restrict__ slopes,
                                                         T* __restrict__ dq, float* __restrict__ delta,
                                                         float* __restrict__ slope_part,
                                                         float* __restrict__ place_part) {
  constexpr int ROWS = FEW ? 1 : 4;
  const unsigned ctas = unsigned(RS + ROWS - 1) / ROWS, task = blockIdx.x / ctas;
  const AttJoin jn = joins[task / unsigned(H)];
  const int h = int(task % unsigned(H)), lane = threadIdx.x & 31;
  const int r = int(blockIdx.x % ctas) * ROWS + (FEW ? 0 : threadIdx.x >> 5), mine = FEW ? int(threadIdx.x) : lane;
  if (r >= jn.rows) return;
  const int64_t step = int64_t(H) * RS * W;
  const float* p = part + ((int64_t(jn.first) * H + h) * RS + r) * W;
  const int64_t at = (int64_t(jn.row) + r) * H + h;
  const float s = lane < 10 ? sum_parts(p + DP + lane, step, jn.count) : 0.0f;
  const float all = __shfl_sync(0xffffffffu, s, 9), inv = all == 0.0f ? 0.0f : 1.0f / all;
  const float off = __shfl_sync(0xffffffffu, s, 0) * inv;  // what delta0 is short of delta
  const float low = __shfl_sync(0xffffffffu, s, lane < 3 ? 6 + lane : 2);
  const float high = __shfl_sync(0xffffffffu, s, lane < 3 ? 3 + lane : 1);
  if (mine == 0) delta[at] = p[DP + 10] + off;
  for (int d = mine; d < D; d += 128 / ROWS) {
    float x = sum_parts(p + d, step, jn.count);
    // fix: dS was formed with delta from the rounded result, and P K follows the sums
    if (fix) x = fmaf(-off, sum_parts(p + DP + 16 + d, step, jn.count), x);
    dq[at * D + d] = from_float<T>(scale * x);
  }
  if (slopes) {
    if (mine < 3) place_part[at * 3 + mine] = -slopes[h] * inv * (high - off * low);
    if (mine == 3) slope_part[at] = -inv * (high - off * low);
  }
}

template <typename T>
__global__ void __launch_bounds__(128) join_key_kernel(const AttJoin* __restrict__ joins,
                                                       const float* __restrict__ part, int RS, int W, int DP, int D,
                                                       int Hk, float scale, T* __restrict__ dk, T* __restrict__ dv,
                                                       float* __restrict__ place_part) {
  const unsigned ctas = unsigned(RS + 3) / 4, task = blockIdx.x / ctas;
  const AttJoin jn = joins[task / unsigned(Hk)];
  const int h = int(task % unsigned(Hk)), lane = threadIdx.x & 31;
  const int r = int(blockIdx.x % ctas) * 4 + (threadIdx.x >> 5);
  if (r >= jn.rows) return;
  const int64_t step = int64_t(Hk) * RS * W;
  const float* p = part + ((int64_t(jn.first) * Hk + h) * RS + r) * W;
  const int64_t at = (int64_t(jn.row) + r) * Hk + h;
  for (int d = lane; d < D; d += 32) {
    dv[at * D + d] = from_float<T>(sum_parts(p + d, step, jn.count));
    dk[at * D + d] = from_float<T>(scale * sum_parts(p + DP + d, step, jn.count));
  }
  if (place_part && lane < 3) place_part[at * 3 + lane] = -sum_parts(p + 2 * DP + lane, step, jn.count);
}

// ---------------------------------------------------------------------------
constexpr int kJoinCtas = kTileRows / 4;  // CTAs of a tile's join

unsigned row_grid(int64_t tasks) { return unsigned((tasks + kRowWarps - 1) / kRowWarps); }

// Launch grids that the tables ask for stay within 2^31 - 1 CTAs.
int check_grids(const y3b_structure_attention_args* p, const char* what) {
  const int64_t most = int64_t(INT32_MAX) / kJoinCtas;
  if (p->query_row_count * p->heads > INT32_MAX || p->key_row_count * p->key_heads > INT32_MAX ||
      p->query_join_count * p->heads > most || p->forward_join_count * p->heads > most ||
      p->few_join_count * p->heads > most || p->key_join_count * p->key_heads > most)
    return fail(Y3B_ERR_UNSUPPORTED, "%s: the batch's tables ask for more than 2^31 - 1 CTAs", what);
  return Y3B_OK;
}

bool on16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// How one call uses its workspace (offsets in bytes, parts 16-byte aligned).
struct AttPlan {
  int pieces, DP, chunks, Wf, Wq, Wk;
  bool tiles;
  bool direct[3];  // query, key, value are read in place
  int64_t packed[4], delta, slope, dx, dy, part_q, part_k, part_few, bytes;
};

bool in_place(const y3b_structure_attention_args* p, const void* base, int64_t row, int64_t head) {
  // a tensor map takes positive strides below 2^40 bytes
  const auto fits = [](int64_t v) { return v > 0 && v % 8 == 0 && v < (int64_t(1) << 39); };
  return p->dtype == Y3B_BF16 && p->width % 8 == 0 && fits(row) && fits(head) && on16(base);
}

AttPlan make_plan(const y3b_structure_attention_args* p, bool adjoint) {
  AttPlan w;
  const int64_t H = p->heads, Hk = p->key_heads, nq = p->query_count, nk = p->key_count;
  w.pieces = p->dtype == Y3B_F32 ? 3 : 1;
  w.DP = p->width > 64 ? 128 : 64;
  w.chunks = (p->width + 7) / 8;
  w.Wf = w.DP + 16;
  w.Wq = (w.pieces == 1 ? 2 : 1) * w.DP + 16;
  w.Wk = 2 * w.DP + 16;
  w.tiles = adjoint ? p->query_item_count > 0 || p->key_item_count > p->few_key_item_count : p->forward_item_count > 0;
  w.direct[0] = in_place(p, p->query, p->query_row_stride, p->query_head_stride);
  w.direct[1] = in_place(p, p->key, p->key_row_stride, p->key_head_stride);
  w.direct[2] = in_place(p, p->value, p->value_row_stride, p->value_head_stride);
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 15) / 16 * 16;
    return here;
  };
  const int64_t row = int64_t(w.pieces) * w.chunks * 16;
  w.packed[0] = take(w.tiles && !w.direct[0] ? nq * H * row : 0);
  w.packed[1] = take(w.tiles && !w.direct[1] ? nk * Hk * row : 0);
  w.packed[2] = take(w.tiles && !w.direct[2] ? nk * Hk * row : 0);
  w.packed[3] = take(w.tiles && adjoint ? nq * H * row : 0);
  w.delta = take(adjoint ? nq * H * 4 : 0);
  w.slope = take(adjoint ? nq * H * 4 : 0);
  w.dx = take(adjoint ? nq * H * 12 : 0);
  w.dy = take(adjoint ? nk * Hk * 12 : 0);
  w.part_q = take(adjoint ? p->query_slot_count * H * kTileRows * w.Wq * 4
                          : p->forward_slot_count * H * kTileRows * w.Wf * 4);
  w.part_k = take(adjoint ? p->key_slot_count * Hk * kTileRows * w.Wk * 4 : 0);
  w.part_few = take(p->few_item_count * H * kFewQueries * ((adjoint ? 2 : 1) * w.DP + 16) * 4);
  w.bytes = at;
  return w;
}

// Operand views of the call, packed where they cannot be read in place.
int operands(const y3b_structure_attention_args* p, const AttPlan& w, const void* grad, unsigned char* ws,
             AttTileArgs* t, cudaStream_t s) {
  const int64_t H = p->heads, Hk = p->key_heads, D = p->width;
  const PackSource src[4] = {
      {p->query, p->query_row_stride, p->query_head_stride, p->query_count, int(H), nullptr},
      {p->key, p->key_row_stride, p->key_head_stride, p->key_count, int(Hk), nullptr},
      {p->value, p->value_row_stride, p->value_head_stride, p->key_count, int(Hk), nullptr},
      {grad, H * D, D, p->query_count, int(H), nullptr}};
  AttOperand* dst[4] = {&t->q, &t->k, &t->v, &t->g};
  PackArgs a;
  a.D = int(D);
  a.chunks = w.chunks;
  int n = 0;
  int64_t most = 0;
  for (int k = 0; k < (grad ? 4 : 3); ++k) {
    if (k < 3 ? w.direct[k] : in_place(p, grad, H * D, D)) {
      *dst[k] = {static_cast<const __nv_bfloat16*>(src[k].p), src[k].row, src[k].head, 0};
      continue;
    }
    PackSource o = src[k];
    o.out = reinterpret_cast<__nv_bfloat16*>(ws + w.packed[k]);
    const int64_t wide = int64_t(w.chunks) * 8;
    *dst[k] = {o.out, o.heads * wide, wide, o.rows * o.heads * wide};
    if (o.rows > 0) {
      a.s[n++] = o;
      most = std::max(most, o.rows * o.heads * w.chunks);
    }
  }
  if (n) {
    const dim3 grid(unsigned(std::min<int64_t>((most + 255) / 256, kSMs * 16)), unsigned(n));
    if (p->dtype == Y3B_F32) pack_kernel<float><<<grid, 256, 0, s>>>(a);
    else pack_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(a);
    Y3B_LAUNCH_CHECK();
  }
  return Y3B_OK;
}

AttTileArgs tile_args(const y3b_structure_attention_args* p, const AttArgs& a, const AttPlan& w, int32_t* status) {
  AttTileArgs t{};
  t.nq = a.nq;
  t.nk = a.nk;
  t.H = a.H;
  t.Hk = a.Hk;
  t.D = a.D;
  t.group = a.group;
  t.chunks = w.chunks;
  t.x = a.x;
  t.y = a.y;
  t.slopes = a.slopes;
  t.scale = a.scale;
  t.scale2 = a.scale2;
  t.status = status;
  return t;
}

template <typename T>
int forward(const y3b_structure_attention_args* p, const AttArgs& a, const AttPlan& w, unsigned char* ws, void* out,
            float* lse, int32_t* status, cudaStream_t s) {
  if (p->small_32_count + p->small_64_count > 0) {
    const int rc = attention_small_forward<T>(a, reinterpret_cast<const AttSmall*>(p->small), p->small_32_count,
                                              p->small_64_count, static_cast<T*>(out), lse, s);
    if (rc) return rc;
  }
  if (p->query_row_count > 0) {
    row_forward_kernel<T><<<row_grid(p->query_row_count * a.H), 32 * kRowWarps, 0, s>>>(
        a, reinterpret_cast<const int2*>(p->query_rows), p->query_row_count, static_cast<T*>(out), lse);
    Y3B_LAUNCH_CHECK();
  }
  if (p->few_item_count > 0) {
    float* part = reinterpret_cast<float*>(ws + w.part_few);
    const int rc = attention_few_forward<T>(a, reinterpret_cast<const AttItem*>(p->few_items), p->few_item_count, w.DP,
                                            w.DP + 16, part, s);
    if (rc) return rc;
    join_few_kernel<T><<<unsigned(p->few_join_count * a.H * kFewQueries), 128, 0, s>>>(
        reinterpret_cast<const AttJoin*>(p->few_joins), part, w.DP + 16, w.DP, a.D, a.H, static_cast<T*>(out), lse);
    Y3B_LAUNCH_CHECK();
  }
  if (p->forward_item_count > 0) {
    AttTileArgs t = tile_args(p, a, w, status);
    int rc = operands(p, w, nullptr, ws, &t, s);
    if (rc) return rc;
    t.items = reinterpret_cast<const AttItem*>(p->forward_items);
    t.out0 = out;
    t.lse = lse;
    t.part = reinterpret_cast<float*>(ws + w.part_q);
    t.vec = a.D * sizeof(T) % 16 == 0 && on16(out);
    rc = attention_forward_tiles(w.pieces, t, p->forward_item_count, s);
    if (rc) return rc;
    if (p->forward_join_count > 0) {
      join_forward_kernel<T><<<unsigned(p->forward_join_count * a.H * kJoinCtas), 128, 0, s>>>(
          reinterpret_cast<const AttJoin*>(p->forward_joins), t.part, w.Wf, w.DP, a.D, a.H, static_cast<T*>(out), lse);
      Y3B_LAUNCH_CHECK();
    }
  }
  return Y3B_OK;
}

template <typename T>
int backward(const y3b_structure_attention_args* p, const AttArgs& a, const AttPlan& w, unsigned char* ws,
             const void* out, const void* grad, const float* lse, void* dq, void* dk, void* dv, float* dx, float* dy,
             float* dslopes, int32_t* status, cudaStream_t s) {
  float* delta = reinterpret_cast<float*>(ws + w.delta);
  float* slope_part = reinterpret_cast<float*>(ws + w.slope);
  float* dx_part = reinterpret_cast<float*>(ws + w.dx);
  float* dy_part = reinterpret_cast<float*>(ws + w.dy);
  const T* g = static_cast<const T*>(grad);
  AttTileArgs t = tile_args(p, a, w, status);
  if (w.tiles) {
    const int rc = operands(p, w, grad, ws, &t, s);
    if (rc) return rc;
  }
  t.lse = const_cast<float*>(lse);
  t.delta = delta;
  t.slope_part = slope_part;
  if (p->small_32_count + p->small_64_count > 0) {
    const int rc = attention_small_backward<T>(a, reinterpret_cast<const AttSmall*>(p->small), p->small_32_count,
                                               p->small_64_count, g, static_cast<T*>(dq), static_cast<T*>(dk),
                                               static_cast<T*>(dv), slope_part, dx_part, dy_part, s);
    if (rc) return rc;
  }
  // query side: it also gives delta, which the key side reads
  if (p->query_row_count > 0) {
    row_backward_query_kernel<T><<<row_grid(p->query_row_count * a.H), 32 * kRowWarps, 0, s>>>(
        a, reinterpret_cast<const int2*>(p->query_rows), p->query_row_count, g, lse, delta, static_cast<T*>(dq),
        slope_part, dx_part);
    Y3B_LAUNCH_CHECK();
  }
  if (p->few_item_count > 0) {
    float* part = reinterpret_cast<float*>(ws + w.part_few);
    const int rc = attention_few_query<T>(a, reinterpret_cast<const AttItem*>(p->few_items), p->few_item_count, w.DP,
                                          2 * w.DP + 16, static_cast<const T*>(out), g, lse, part, s);
    if (rc) return rc;
    join_query_kernel<T, true><<<unsigned(p->few_join_count * a.H * kFewQueries), 128, 0, s>>>(
        reinterpret_cast<const AttJoin*>(p->few_joins), part, kFewQueries, 2 * w.DP + 16, w.DP, a.D, a.H, a.scale, true,
        a.slopes, static_cast<T*>(dq), delta, slope_part, dx_part);
    Y3B_LAUNCH_CHECK();
  }
  if (p->query_item_count > 0) {
    t.items = reinterpret_cast<const AttItem*>(p->query_items);
    t.out_in = out;
    t.grad_in = grad;
    t.place_part = dx_part;
    t.out0 = dq;
    t.part = reinterpret_cast<float*>(ws + w.part_q);
    t.vec = a.D * sizeof(T) % 16 == 0 && on16(dq) && on16(out) && on16(grad);
    const int rc = attention_query_tiles(w.pieces, t, p->query_item_count, s);
    if (rc) return rc;
    if (p->query_join_count > 0) {
      join_query_kernel<T, false><<<unsigned(p->query_join_count * a.H * kJoinCtas), 128, 0, s>>>(
          reinterpret_cast<const AttJoin*>(p->query_joins), t.part, kTileRows, w.Wq, w.DP, a.D, a.H, a.scale,
          w.pieces == 1, a.slopes,
          static_cast<T*>(dq), delta, slope_part, dx_part);
      Y3B_LAUNCH_CHECK();
    }
  }
  const AttItem* key_items = reinterpret_cast<const AttItem*>(p->key_items);
  const int64_t key_tiles = p->key_item_count - p->few_key_item_count;
  if (p->few_key_item_count > 0) {
    const int rc = attention_few_key<T>(a, key_items + key_tiles, p->few_key_item_count, g, lse, delta,
                                        static_cast<T*>(dk), static_cast<T*>(dv), dy_part, s);
    if (rc) return rc;
  }
  if (p->key_row_count > 0) {
    row_backward_key_kernel<T><<<row_grid(p->key_row_count * a.Hk), 32 * kRowWarps, 0, s>>>(
        a, reinterpret_cast<const int2*>(p->key_rows), p->key_row_count, g, lse, delta, static_cast<T*>(dk),
        static_cast<T*>(dv), dy_part);
    Y3B_LAUNCH_CHECK();
  }
  if (key_tiles > 0) {
    t.items = key_items;
    t.place_part = dy_part;
    t.out0 = dv;
    t.out1 = dk;
    t.part = reinterpret_cast<float*>(ws + w.part_k);
    t.vec = a.D * sizeof(T) % 16 == 0 && on16(dk) && on16(dv);
    const int rc = attention_key_tiles(w.pieces, t, key_tiles, s);
    if (rc) return rc;
    if (p->key_join_count > 0) {
      join_key_kernel<T><<<unsigned(p->key_join_count * a.Hk * kJoinCtas), 128, 0, s>>>(
          reinterpret_cast<const AttJoin*>(p->key_joins), t.part, kTileRows, w.Wk, w.DP, a.D, a.Hk, a.scale,
          static_cast<T*>(dk), static_cast<T*>(dv), a.slopes ? dy_part : nullptr);
      Y3B_LAUNCH_CHECK();
    }
  }
  if (a.slopes) {
    const auto ctas = [](int64_t n) { return unsigned((n * 3 + kFinishThreads - 1) / kFinishThreads); };
    const FinishArgs f{dx_part, dy_part, slope_part, dx, dy, dslopes, a.nq, a.nk, a.H, a.Hk, ctas(a.nq),
                       dy ? ctas(a.nk) : 0u};
    finish_kernel<<<f.x_ctas + f.y_ctas + unsigned(a.H), kFinishThreads, 0, s>>>(f);
    Y3B_LAUNCH_CHECK();
  }
  return Y3B_OK;
}

}  // namespace
}  // namespace y3b

using namespace y3b;

namespace y3b {

int encode_columns(CUtensorMap* map, const AttOperand& o, int D, int heads, int64_t rows, int pieces, int box_rows) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult got;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &got) != cudaSuccess ||
        got != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<Encode>(f);
  }();
  if (rows == 0) return Y3B_OK;  // no column is loaded
  if (!encode) return fail(Y3B_ERR_CUDA, "structure_attention: the driver has no cuTensorMapEncodeTiled");
  // the encoder is a driver call: a thread that has not used the runtime yet (as autograd's) has no context current
  int device = 0;
  Y3B_CUDA_TRY(cudaGetDevice(&device));
  Y3B_CUDA_TRY(cudaSetDevice(device));
  const int width = (D + 7) / 8 * 8;
  const cuuint64_t size[4] = {cuuint64_t(width), cuuint64_t(heads), cuuint64_t(rows), cuuint64_t(pieces)};
  const cuuint64_t stride[3] = {cuuint64_t(o.head) * 2, cuuint64_t(o.row) * 2,
                                cuuint64_t(pieces > 1 ? o.piece : o.row) * 2};
  const cuuint32_t box[4] = {64, 1, cuuint32_t(box_rows), 1}, step[4] = {1, 1, 1, 1};
  const CUresult rc = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<__nv_bfloat16*>(o.p), size, stride,
                             box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) return fail(Y3B_ERR_CUDA, "structure_attention: tensor map refused (%d)", int(rc));
  return Y3B_OK;
}

}  // namespace y3b

extern "C" int64_t y3b_structure_attention_workspace_bytes(const y3b_structure_attention_args* args, int adjoint) {
  AttArgs a;
  if (unpack(args, "structure_attention_workspace_bytes", &a)) return -1;
  return make_plan(args, adjoint != 0).bytes;
}

namespace {
int check_workspace(const AttPlan& w, const void* workspace, int64_t bytes, const char* what) {
  if (w.bytes == 0) return Y3B_OK;
  Y3B_CHECK_ARG(workspace && on16(workspace), "%s: workspace must be 16-byte aligned", what);
  if (bytes < w.bytes)
    return fail(Y3B_ERR_WORKSPACE, "%s: workspace of %lld bytes, %lld needed", what, (long long)bytes,
                (long long)w.bytes);
  return Y3B_OK;
}
}  // namespace

extern "C" int y3b_structure_attention(const y3b_structure_attention_args* args, void* workspace,
                                       int64_t workspace_bytes, void* out, float* lse, int32_t* status,
                                       void* stream) {
  AttArgs a;
  int rc = unpack(args, "structure_attention", &a);
  if (rc) return rc;
  if (a.nq == 0) return Y3B_OK;
  rc = check_grids(args, "structure_attention");
  if (rc) return rc;
  Y3B_CHECK_ARG(out && lse, "structure_attention: null output");
  const AttPlan w = make_plan(args, false);
  rc = check_workspace(w, workspace, workspace_bytes, "structure_attention");
  if (rc) return rc;
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  return args->dtype == Y3B_F32 ? forward<float>(args, a, w, ws, out, lse, status, as_stream(stream))
                                : forward<__nv_bfloat16>(args, a, w, ws, out, lse, status, as_stream(stream));
}

extern "C" int y3b_structure_attention_adjoint(const y3b_structure_attention_args* args, const void* out,
                                               const void* out_grad, const float* lse, void* workspace,
                                               int64_t workspace_bytes, void* query_grad, void* key_grad,
                                               void* value_grad, float* positions_grad, float* key_positions_grad,
                                               float* slopes_grad, int32_t* status, void* stream) {
  AttArgs a;
  int rc = unpack(args, "structure_attention_adjoint", &a);
  if (rc) return rc;
  Y3B_CHECK_ARG(a.nq == 0 || (out && out_grad && lse && query_grad),
                "structure_attention_adjoint: null query-side argument");
  Y3B_CHECK_ARG(a.nk == 0 || (key_grad && value_grad), "structure_attention_adjoint: null key-side gradient");
  Y3B_CHECK_ARG(!a.slopes || (slopes_grad && (a.nq == 0 || positions_grad)),
                "structure_attention_adjoint: null position or slope gradient");
  Y3B_CHECK_ARG(!a.slopes || key_positions_grad || a.nk == 0 || a.nq == a.nk,
                "structure_attention_adjoint: one position gradient needs as many queries as keys");
  rc = check_grids(args, "structure_attention_adjoint");
  if (rc) return rc;
  const AttPlan w = make_plan(args, true);
  rc = check_workspace(w, workspace, workspace_bytes, "structure_attention_adjoint");
  if (rc) return rc;
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  cudaStream_t s = as_stream(stream);
  return args->dtype == Y3B_F32
             ? backward<float>(args, a, w, ws, out, out_grad, lse, query_grad, key_grad, value_grad, positions_grad,
                               key_positions_grad, slopes_grad, status, s)
             : backward<__nv_bfloat16>(args, a, w, ws, out, out_grad, lse, query_grad, key_grad, value_grad,
                                       positions_grad, key_positions_grad, slopes_grad, status, s);
}
