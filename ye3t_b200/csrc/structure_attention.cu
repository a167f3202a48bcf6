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
#include "structure_attention.cuh"

namespace y3b {
namespace {

constexpr int kRowWarps = 4;
constexpr int kRowAcc = kAttMaxWidth / 32;

struct Range {
  int64_t b, e;
};

__device__ __forceinline__ Range keys_of(const AttArgs& a, int64_t i) {
  const int s = a.q_struct[i];
  Range r{a.k_off[s], a.k_off[s + 1]};
  if (r.b < 0) r.b = 0;
  if (r.e > a.nk) r.e = a.nk;
  return r;
}

__device__ __forceinline__ Range queries_of(const AttArgs& a, int64_t j) {
  const int s = a.k_struct[j];
  Range r{a.q_off[s], a.q_off[s + 1]};
  if (r.b < 0) r.b = 0;
  if (r.e > a.nq) r.e = a.nq;
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
__global__ void __launch_bounds__(32 * kRowWarps) row_forward_kernel(AttArgs a, T* __restrict__ out,
                                                                     float* __restrict__ lse) {
  __shared__ float s_q[kRowWarps][kAttMaxWidth];
  __shared__ float s_p[kRowWarps][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t task = blockIdx.x * int64_t(kRowWarps) + w;
  if (task >= a.nq * a.H) return;
  const int64_t i = task / a.H;
  const int h = int(task - i * a.H), hk = h / a.group;
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
  const Range r = keys_of(a, i);
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
    AttArgs a, const T* __restrict__ grad, const float* __restrict__ lse, float* __restrict__ delta,
    T* __restrict__ dq, float* __restrict__ dslope_part, float* __restrict__ dx_part) {
  __shared__ float s_q[kRowWarps][kAttMaxWidth];
  __shared__ float s_g[kRowWarps][kAttMaxWidth];
  __shared__ float s_p[kRowWarps][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t task = blockIdx.x * int64_t(kRowWarps) + w;
  if (task >= a.nq * a.H) return;
  const int64_t i = task / a.H;
  const int h = int(task - i * a.H), hk = h / a.group;
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
  const Range r = keys_of(a, i);
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
    AttArgs a, const T* __restrict__ grad, const float* __restrict__ lse, const float* __restrict__ delta,
    T* __restrict__ dk, T* __restrict__ dv, float* __restrict__ dy_part) {
  __shared__ float s_k[kRowWarps][kAttMaxWidth];
  __shared__ float s_v[kRowWarps][kAttMaxWidth];
  __shared__ float s_p[kRowWarps][32];
  __shared__ float s_d[kRowWarps][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t task = blockIdx.x * int64_t(kRowWarps) + w;
  if (task >= a.nk * a.Hk) return;
  const int64_t j = task / a.Hk;
  const int hk = int(task - j * a.Hk);
  const T* k = static_cast<const T*>(a.k) + j * a.k_row + hk * a.k_head;
  const T* v = static_cast<const T*>(a.v) + j * a.v_row + hk * a.v_head;
  for (int d = lane; d < a.D; d += 32) {
    s_k[w][d] = to_float(k[d]) * a.scale2;
    s_v[w][d] = to_float(v[d]);
  }
  __syncwarp();
  const Range r = queries_of(a, j);
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

// dx[i] = sum over heads of dx_part (and of dy_part where queries and keys are the same
// atoms); dy[j] likewise.  One thread per component.
__global__ void __launch_bounds__(256) position_grad_kernel(const float* __restrict__ part, int64_t n, int heads,
                                                            const float* __restrict__ other, int other_heads,
                                                            float* __restrict__ out) {
  const int64_t t = blockIdx.x * int64_t(blockDim.x) + threadIdx.x;
  if (t >= n * 3) return;
  const int64_t i = t / 3;
  const int c = int(t - 3 * i);
  float sum = 0.0f;
  for (int h = 0; h < heads; ++h) sum += part[(i * heads + h) * 3 + c];
  if (other)
    for (int h = 0; h < other_heads; ++h) sum += other[(i * other_heads + h) * 3 + c];
  out[t] = sum;
}

// dslope[h] = sum over rows, one CTA a head, summed in fp64 in a fixed order.
__global__ void __launch_bounds__(256) slope_grad_kernel(const float* __restrict__ part, int64_t n, int H,
                                                         float* __restrict__ out) {
  __shared__ double s[256];
  const int h = blockIdx.x;
  double sum = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 256) sum += double(part[i * H + h]);
  s[threadIdx.x] = sum;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (int(threadIdx.x) < o) s[threadIdx.x] += s[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) out[h] = float(s[0]);
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
  Y3B_CHECK_ARG(p->query_count == 0 || (p->query && p->query_structure), "%s: null query argument", what);
  Y3B_CHECK_ARG(p->key_count == 0 || (p->key && p->value && p->key_structure), "%s: null key or value", what);
  Y3B_CHECK_ARG((p->slopes != nullptr) || (!p->positions && !p->key_positions), "%s: positions without slopes", what);
  if (p->slopes) {
    Y3B_CHECK_ARG(p->query_count == 0 || p->positions, "%s: slopes without positions", what);
    Y3B_CHECK_ARG(p->key_count == 0 || p->key_positions, "%s: slopes without key positions", what);
  }
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
  a->q_struct = p->query_structure;
  a->k_struct = p->key_structure;
  return Y3B_OK;
}

unsigned row_grid(int64_t tasks) { return unsigned((tasks + kRowWarps - 1) / kRowWarps); }

template <typename T>
int forward(const AttArgs& a, void* out, float* lse, cudaStream_t s) {
  row_forward_kernel<T><<<row_grid(a.nq * a.H), 32 * kRowWarps, 0, s>>>(a, static_cast<T*>(out), lse);
  Y3B_LAUNCH_CHECK();
  return Y3B_OK;
}

// Workspace of the backward: delta [nq, H], the rows' parts of dslope [nq, H] and dx
// [nq, H, 3], and of dy [nk, Hk, 3], all fp32.
int64_t backward_floats(int64_t nq, int64_t nk, int64_t H, int64_t Hk) { return nq * H * 5 + nk * Hk * 3; }

template <typename T>
int backward(const AttArgs& a, const void* grad, const float* lse, float* ws, void* dq, void* dk, void* dv,
             float* dx, float* dy, float* dslopes, cudaStream_t s) {
  float* delta = ws;
  float* slope_part = delta + a.nq * a.H;
  float* dx_part = slope_part + a.nq * a.H;
  float* dy_part = dx_part + a.nq * a.H * 3;
  const T* g = static_cast<const T*>(grad);
  if (a.nq > 0) {
    row_backward_query_kernel<T><<<row_grid(a.nq * a.H), 32 * kRowWarps, 0, s>>>(a, g, lse, delta,
                                                                                static_cast<T*>(dq), slope_part,
                                                                                dx_part);
    Y3B_LAUNCH_CHECK();
  }
  if (a.nk > 0) {
    row_backward_key_kernel<T><<<row_grid(a.nk * a.Hk), 32 * kRowWarps, 0, s>>>(
        a, g, lse, delta, static_cast<T*>(dk), static_cast<T*>(dv), dy_part);
    Y3B_LAUNCH_CHECK();
  }
  if (a.slopes) {
    // dy == null: queries and keys are the same atoms and dx takes both sums
    if (a.nq > 0)
      position_grad_kernel<<<unsigned((a.nq * 3 + 255) / 256), 256, 0, s>>>(
          dx_part, a.nq, a.H, dy == nullptr && a.nk > 0 ? dy_part : nullptr, a.Hk, dx);
    if (dy && a.nk > 0)
      position_grad_kernel<<<unsigned((a.nk * 3 + 255) / 256), 256, 0, s>>>(dy_part, a.nk, a.Hk, nullptr, 0, dy);
    slope_grad_kernel<<<a.H, 256, 0, s>>>(slope_part, a.nq, a.H, dslopes);
    Y3B_LAUNCH_CHECK();
  }
  return Y3B_OK;
}

}  // namespace
}  // namespace y3b

using namespace y3b;

extern "C" int y3b_structure_attention(const y3b_structure_attention_args* args, void* out, float* lse,
                                       void* stream) {
  AttArgs a;
  const int rc = unpack(args, "structure_attention", &a);
  if (rc) return rc;
  if (a.nq == 0) return Y3B_OK;
  Y3B_CHECK_ARG(out && lse, "structure_attention: null output");
  return args->dtype == Y3B_F32 ? forward<float>(a, out, lse, as_stream(stream))
                                : forward<__nv_bfloat16>(a, out, lse, as_stream(stream));
}

extern "C" int64_t y3b_structure_attention_adjoint_workspace_bytes(int64_t query_count, int64_t key_count,
                                                                   int64_t heads, int64_t key_heads) {
  if (query_count < 0 || key_count < 0 || heads < 1 || key_heads < 1) return -1;
  return backward_floats(query_count, key_count, heads, key_heads) * 4;
}

extern "C" int y3b_structure_attention_adjoint(const y3b_structure_attention_args* args, const void* out_grad,
                                               const float* lse, void* workspace, int64_t workspace_bytes,
                                               void* query_grad, void* key_grad, void* value_grad,
                                               float* positions_grad, float* key_positions_grad, float* slopes_grad,
                                               void* stream) {
  AttArgs a;
  const int rc = unpack(args, "structure_attention_adjoint", &a);
  if (rc) return rc;
  const int64_t need = backward_floats(a.nq, a.nk, a.H, a.Hk) * 4;
  Y3B_CHECK_ARG(a.nq == 0 || (out_grad && lse && query_grad), "structure_attention_adjoint: null query-side argument");
  Y3B_CHECK_ARG(a.nk == 0 || (key_grad && value_grad), "structure_attention_adjoint: null key-side gradient");
  Y3B_CHECK_ARG(!a.slopes || (slopes_grad && (a.nq == 0 || positions_grad)),
                "structure_attention_adjoint: null position or slope gradient");
  Y3B_CHECK_ARG(!a.slopes || key_positions_grad || a.nk == 0 || a.nq == a.nk,
                "structure_attention_adjoint: one position gradient needs as many queries as keys");
  if (need > 0) {
    Y3B_CHECK_ARG(workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
                  "structure_attention_adjoint: workspace must be 16-byte aligned");
    if (workspace_bytes < need)
      return fail(Y3B_ERR_WORKSPACE, "structure_attention_adjoint: workspace of %lld bytes, %lld needed",
                  (long long)workspace_bytes, (long long)need);
  }
  float* ws = static_cast<float*>(workspace);
  cudaStream_t s = as_stream(stream);
  return args->dtype == Y3B_F32
             ? backward<float>(a, out_grad, lse, ws, query_grad, key_grad, value_grad, positions_grad,
                               key_positions_grad, slopes_grad, s)
             : backward<__nv_bfloat16>(a, out_grad, lse, ws, query_grad, key_grad, value_grad, positions_grad,
                                       key_positions_grad, slopes_grad, s);
}
