// Structure attention of small structures: up to 64 queries and 64 keys, one CTA a (structure, head) on the
// forward and a (structure, key head) on the backward.
//
// Molecules of some ten atoms would fill a sixth of a 128-row tile and take one tile's latency each.  Here a
// structure's operands sit in shared memory, a warp takes 16 rows, and the products run on mma.sync.  fp32 data is
// split in two tf32 parts with three products (hi hi + hi lo + lo hi, to about 2^-22).  bf16 scores and results use
// bf16 operands straight from shared memory (ldmatrix): with the conversions to tf32 2,048 molecules of 0-39 atoms, 8
// heads of 32, took 75 us, without them 63.  dK and dV of bf16 data take P and dS, which are kept in fp32, as one tf32
// part (11 bits: 2^-12 of a probability beside the result's rounding of 2^-8; 512 molecules of 32 atoms 1.67e-3 of the
// norm off 64 bits, the rounding alone 1.66e-3) and the data itself, which tf32 holds exactly.  fp32 leaves out the
// product of both low parts: results are 3 to 4e-7 of the norm off, those of fp32 arithmetic 2e-7.  The backward forms P
// once more from the scores (so it needs nothing of the forward), keeps P and dS in shared memory and gives every
// gradient in one launch.  Rows and columns past the structure's end are zeros in shared memory.
//
// The forward is bound by instruction issue (70 % of the cycles): of some 1,200 instructions that a warp of 16 rows
// executes, the 11 scores a lane take about 300, the rest goes into the addresses, loads, masks and stores of rows
// that hold 20 atoms on average.  Without integer divisions, exact reciprocals and masks of full blocks: 63 -> 57 us.
// Two heads a CTA, which share their distances, took twice the registers and 87 us.  The backward is bound by latency:
// its registers leave two or three CTAs an SM.
//
// Fragments of the tf32 products: lane = 4 g + c.  A (16 x 8): rows g, g + 8, columns c, c + 4; B (8 x 8): rows c,
// c + 4, column g; accumulator: rows g, g + 8, columns 2 c, 2 c + 1.  An accumulator serves as A of the next product
// with the columns taken in the order 2 c, 2 c + 1, and the rows of B in the same order.
#include "structure_attention_small.cuh"

#include <algorithm>

#include "tcgen05.cuh"

namespace y3b {
namespace {

template <typename T> struct Parts;
template <> struct Parts<__nv_bfloat16> { static constexpr int N = 1; };
template <> struct Parts<float> { static constexpr int N = 2; };

// A value as one (bf16) or two (fp32) tf32 parts.
template <int N> struct Tf32 { uint32_t v[N]; };
__device__ __forceinline__ uint32_t tf32(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;\n" : "=r"(r) : "f"(x));
  return r;
}
// EXACT: x came from bf16 and is a tf32 number as it is.
template <int N, bool EXACT> __device__ __forceinline__ Tf32<N> split(float x) {
  Tf32<N> r;
  if constexpr (N == 1) {
    r.v[0] = EXACT ? __float_as_uint(x) : tf32(x);
  } else {
    r.v[0] = tf32(x);
    r.v[1] = tf32(x - __uint_as_float(r.v[0]));
  }
  return r;
}

__device__ __forceinline__ void mma8(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
      "%2, %3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int N> struct FragA { uint32_t v[N][4]; };
template <int N, bool EXACT>
__device__ __forceinline__ FragA<N> frag_a(float a0, float a1, float a2, float a3) {
  FragA<N> f;
  const Tf32<N> s[4] = {split<N, EXACT>(a0), split<N, EXACT>(a1), split<N, EXACT>(a2), split<N, EXACT>(a3)};
#pragma unroll
  for (int p = 0; p < N; ++p)
#pragma unroll
    for (int k = 0; k < 4; ++k) f.v[p][k] = s[k].v[p];
  return f;
}
template <int N>
__device__ __forceinline__ void product(float (&d)[4], const FragA<N>& a, float b0, float b1) {
  const Tf32<N> s0 = split<N, true>(b0), s1 = split<N, true>(b1);
  if constexpr (N == 2) {
    mma8(d, a.v[1], s0.v[0], s1.v[0]);
    mma8(d, a.v[0], s0.v[1], s1.v[1]);
  }
  mma8(d, a.v[0], s0.v[0], s1.v[0]);
}

// bf16 operands straight from shared memory: four (two) blocks of 8 x 8 values, one address a row.
__device__ __forceinline__ void blocks4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void blocks2(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0, %1}, [%2];\n"
               : "=r"(r[0]), "=r"(r[1]) : "r"(at) : "memory");
}
__device__ __forceinline__ void blocks4_turned(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void blocks2_turned(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];\n"
               : "=r"(r[0]), "=r"(r[1]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
      "%2, %3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5}, {%6}, {%0, %1, %2, %3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(b));
}

// Two neighbouring values as bf16 and what the rounding left of them, also as bf16: 16 bits of each.
__device__ __forceinline__ void halves(float x, float y, uint32_t& high, uint32_t& low) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  const float2 f = __bfloat1622float2(h);
  const __nv_bfloat162 l = __floats2bfloat162_rn(x - f.x, y - f.y);
  high = *reinterpret_cast<const uint32_t*>(&h);
  low = *reinterpret_cast<const uint32_t*>(&l);
}

__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}

// Rows [0, n) of one head into shared memory (`rows` rows of `stride` values), zeros elsewhere.  The copies are
// asynchronous, so that those of all operands are in flight together: arrived() waits for them.  2^shift threads take
// a row's 16-byte parts.
template <typename T>
__device__ __forceinline__ void load_rows(T* dst, int stride, const T* src, int64_t row, int n, int rows, int D,
                                          int shift, bool vec) {
  constexpr int W = 16 / int(sizeof(T));
  const int width = (D + 7) / 8 * 8;
  if (vec) {
    const int d = int(threadIdx.x & ((1u << shift) - 1u)) * W;
    if (d < width) {
      const int r0 = int(threadIdx.x >> shift), step = int(blockDim.x >> shift);
      uint32_t to = tc::smem_addr(dst) + uint32_t(r0 * stride + d) * uint32_t(sizeof(T));
      const T* from = src + r0 * row + d;
      for (int r = r0; r < rows; r += step) {
        tc::cp16(to, r < n ? from : src, r < n);
        to += uint32_t(step * stride) * uint32_t(sizeof(T));
        from += step * row;
      }
    }
  } else {
    for (int u = threadIdx.x; u < rows * width; u += blockDim.x) {
      const int r = u / width, d = u - r * width;
      dst[r * stride + d] = r < n && d < D ? src[r * row + d] : from_float<T>(0.0f);
    }
  }
}

__device__ __forceinline__ void load_places(float* dst, const float* src, int n, int rows) {
  for (int u = threadIdx.x; u < rows * 3; u += blockDim.x)
    tc::cp4(tc::smem_addr(dst + u), u < n * 3 ? src + u : src, u < n * 3);
}
__device__ __forceinline__ void arrived() {
  tc::cp_commit();
  tc::cp_wait<0>();
  __syncthreads();
}

template <typename T>
__device__ __forceinline__ void store_pair(T* dst, int d, int D, float a, float b) {
  if (d < D) dst[d] = from_float<T>(a);
  if (d + 1 < D) dst[d + 1] = from_float<T>(b);
}
// Two neighbouring values: one store where the row starts on a pair.
template <typename T>
__device__ __forceinline__ void store_pair(T* dst, int d, int D, float a, float b, bool even) {
  if (even && d + 1 < D) {
    if constexpr (sizeof(T) == 2) *reinterpret_cast<__nv_bfloat162*>(dst + d) = __floats2bfloat162_rn(a, b);
    else *reinterpret_cast<float2*>(dst + d) = make_float2(a, b);
  } else {
    store_pair(dst, d, D, a, b);
  }
}

// Two neighbouring values of a row.
__device__ __forceinline__ float2 pair_at(const float* p) { return *reinterpret_cast<const float2*>(p); }

// Products of 16 rows of X with the rows of Y in bf16, in steps of 16 components (the last one may have 8): out[t] (rows
// g, g + 8; columns 8 t + 2 c, + 1) = X Y^T.  Rows up to the next multiple of 16 are read.
template <int NT>
__device__ __forceinline__ void scores_bf16(float (&out)[NT][4], const __nv_bfloat16* x, const __nv_bfloat16* y,
                                            int stride, int nt, int width, int lane) {
#pragma unroll
  for (int t = 0; t < NT; ++t) out[t][0] = out[t][1] = out[t][2] = out[t][3] = 0.0f;
  const uint32_t xa = tc::smem_addr(x) + 2 * ((lane & 15) * stride + (lane >> 4) * 8);
  const uint32_t ya = tc::smem_addr(y) + 2 * (((lane & 7) + (lane >> 4) * 8) * stride + (lane >> 3 & 1) * 8);
  uint32_t a[4], b[4];
  int k = 0;
#pragma unroll 2
  for (; k + 16 <= width; k += 16) {
    blocks4(a, xa + 2 * k);
#pragma unroll
    for (int t = 0; t < NT; t += 2) {
      if (t < nt) {
        blocks4(b, ya + 2 * (8 * t * stride + k));
        mma16(out[t], a, b[0], b[1]);
        if (t + 1 < nt) mma16(out[t + 1], a, b[2], b[3]);
      }
    }
  }
  if (k < width) {
    blocks2(a, xa + 2 * k);
    const uint32_t y8 = tc::smem_addr(y) + 2 * ((lane & 15) * stride + k);
#pragma unroll
    for (int t = 0; t < NT; t += 2) {
      if (t < nt) {
        blocks2(b, y8 + 2 * (8 * t * stride));
        mma8_bf16(out[t], a, b[0]);
        if (t + 1 < nt) mma8_bf16(out[t + 1], a, b[1]);
      }
    }
  }
}

// The same for either type.  fp32: both operands take the components of a step in the order 2 c, 2 c + 1, which are read
// as a pair.  The tensor cores cut a sum towards zero each time that they add to it, which is the same way for every
// score; each step's products are therefore added to the score outside (a readout's slope gradient 3.4e-6 -> 2.0e-6 off,
// for 4 % of the backward's time).
template <typename T, int NT>
__device__ __forceinline__ void scores(float (&out)[NT][4], const T* x, const T* y, int stride, int nt, int width,
                                       int g, int c) {
  if constexpr (sizeof(T) == 2) {
    scores_bf16<NT>(out, x, y, stride, nt, width, 4 * g + c);
  } else {
    constexpr int N = Parts<T>::N;
#pragma unroll
    for (int t = 0; t < NT; ++t) out[t][0] = out[t][1] = out[t][2] = out[t][3] = 0.0f;
#pragma unroll 2
    for (int k = 0; k < width; k += 8) {
      const T* x0 = x + g * stride + k + 2 * c;
      const float2 a0 = pair_at(x0), a1 = pair_at(x0 + 8 * stride);
      const FragA<N> a = frag_a<N, true>(a0.x, a1.x, a0.y, a1.y);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (t < nt) {
          const float2 b = pair_at(y + (8 * t + g) * stride + k + 2 * c);
          float step[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          product<N>(step, a, b.x, b.y);
#pragma unroll
          for (int u = 0; u < 4; ++u) out[t][u] += step[u];
        }
      }
    }
  }
}

// Distances of a thread's pairs of rows and columns, and their reciprocals: as in the tile kernels, a tiny term
// keeps the reciprocal finite at distance zero.
template <int NT> struct Places {
  float d[NT][4], r[NT][4];
};
struct Apart3 {
  float x, y, z;
};
__device__ __forceinline__ Apart3 apart3(const float* x, const float* y) {
  return {x[0] - y[0], x[1] - y[1], x[2] - y[2]};
}
__device__ __forceinline__ float square(const Apart3& a) {
  return fmaf(a.z, a.z, fmaf(a.y, a.y, fmaf(a.x, a.x, 1e-30f)));
}
template <int NT>
__device__ __forceinline__ void distances(Places<NT>& p, const float* x0, const float* x8, const float* y, int nt,
                                          int c) {
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (t < nt) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float q = square(apart3(k >> 1 ? x8 : x0, y + 3 * (8 * t + 2 * c + (k & 1))));
        p.r[t][k] = tc::rsqrt_approx(q);
        p.d[t][k] = q * p.r[t][k];
      }
    }
  }
}

struct Softmax {
  float m[2], l[2];
};

// Scores to probabilities (not yet divided by the sums l), columns past n to zero.
template <int NT>
__device__ __forceinline__ Softmax softmax(float (&s)[NT][4], int nt, int n, int c, float scale2, float slope2,
                                           bool bias, const Places<NT>& at) {
  Softmax r;
  r.m[0] = r.m[1] = -INFINITY;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (t < nt) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float v = s[t][k] * scale2;
        if (bias) v = fmaf(-slope2, at.d[t][k], v);
        if (8 * t + 8 > n) v = 8 * t + 2 * c + (k & 1) < n ? v : -INFINITY;
        s[t][k] = v;
        r.m[k >> 1] = fmaxf(r.m[k >> 1], v);
      }
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    r.m[h] = quad_max(r.m[h]);
    if (r.m[h] == -INFINITY) r.m[h] = 0.0f;
    r.l[h] = 0.0f;
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (t < nt) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        s[t][k] = tc::ex2(s[t][k] - r.m[k >> 1]);
        r.l[k >> 1] += s[t][k];
      }
    }
  }
  r.l[0] = quad_sum(r.l[0]);
  r.l[1] = quad_sum(r.l[1]);
  return r;
}

// out (16 rows x the width, not yet divided by the sums) = P V, row by row into `store`: P as tf32 parts.
template <typename T, int NT, typename Store>
__device__ __forceinline__ void weighted(const float (&s)[NT][4], const T* v, int stride, int nt, int width, int g,
                                         int c, Store store) {
  constexpr int N = Parts<T>::N;
  FragA<N> p[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
    if (t < nt) p[t] = frag_a<N, false>(s[t][0], s[t][2], s[t][1], s[t][3]);
  for (int d = 0; d < width; d += 8) {
    float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (t < nt) {
        const T* v0 = v + (8 * t + 2 * c) * stride + d + g;
        product<N>(o, p[t], to_float(v0[0]), to_float(v0[stride]));
      }
    }
    store(d, o);
  }
}
// bf16: P as two bf16 parts (16 bits, so that the result keeps the precision of its own rounding), V as it is.
template <int NT, typename Store>
__device__ __forceinline__ void weighted_bf16(const float (&s)[NT][4], const __nv_bfloat16* v, int stride, int nt,
                                              int width, int lane, Store store) {
  uint32_t high[NT / 2][4], low[NT / 2][4];
#pragma unroll
  for (int t = 0; t < NT; t += 2) {
    if (t < nt) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        halves(s[t][2 * u], s[t][2 * u + 1], high[t / 2][u], low[t / 2][u]);
        high[t / 2][2 + u] = low[t / 2][2 + u] = 0u;
        if (t + 1 < nt) halves(s[t + 1][2 * u], s[t + 1][2 * u + 1], high[t / 2][2 + u], low[t / 2][2 + u]);
      }
    }
  }
  const uint32_t va = tc::smem_addr(v) + 2 * ((lane & 15) * stride + (lane >> 4) * 8);
  for (int d = 0; d < width; d += 16) {
    float o[2][4] = {};
    const bool two = d + 8 < width;
#pragma unroll
    for (int t = 0; t < NT; t += 2) {
      if (t < nt) {
        uint32_t b[4];
        const uint32_t at = va + 2 * (8 * t * stride + d);
        if (two) blocks4_turned(b, at);
        else blocks2_turned(b, at);
        mma16(o[0], low[t / 2], b[0], b[1]);
        mma16(o[0], high[t / 2], b[0], b[1]);
        if (two) {
          mma16(o[1], low[t / 2], b[2], b[3]);
          mma16(o[1], high[t / 2], b[2], b[3]);
        }
      }
    }
    store(d, o[0]);
    if (two) store(d + 8, o[1]);
  }
}

template <typename T, int NT>
__global__ void __launch_bounds__(16 * NT) small_forward_kernel(const __grid_constant__ AttArgs a,
                                                                const AttSmall* __restrict__ list, int64_t n,
                                                                int stride, int shift, int vec, T* __restrict__ out,
                                                                float* __restrict__ lse) {
  constexpr int R = 8 * NT;
  extern __shared__ __align__(16) unsigned char small_smem[];
  T* s_q = reinterpret_cast<T*>(small_smem);
  T* s_k = s_q + R * stride;
  T* s_v = s_k + R * stride;
  float* s_x = reinterpret_cast<float*>(s_v + R * stride);
  float* s_y = s_x + R * 3;
  const int64_t task = blockIdx.y + int64_t(gridDim.y) * blockIdx.z;
  if (task >= n) return;
  const AttSmall it = list[task];
  const int h = int(blockIdx.x), hk = a.group == 1 ? h : h / a.group;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int width = (a.D + 7) / 8 * 8;
  const int q_rows = (it.nq + 15) / 16 * 16, k_rows = (it.nk + 15) / 16 * 16;  // what the fragments read
  load_rows<T>(s_q, stride, static_cast<const T*>(a.q) + int64_t(it.q) * a.q_row + h * a.q_head, a.q_row, it.nq,
               q_rows, a.D, shift, vec & 1);
  load_rows<T>(s_k, stride, static_cast<const T*>(a.k) + int64_t(it.k) * a.k_row + hk * a.k_head, a.k_row, it.nk,
               k_rows, a.D, shift, vec & 2);
  load_rows<T>(s_v, stride, static_cast<const T*>(a.v) + int64_t(it.k) * a.v_row + hk * a.v_head, a.v_row, it.nk,
               k_rows, a.D, shift, vec & 4);
  const bool bias = a.slopes != nullptr;
  if (bias) {
    load_places(s_x, a.x + int64_t(it.q) * 3, it.nq, q_rows);
    load_places(s_y, a.y + int64_t(it.k) * 3, it.nk, k_rows);
  }
  arrived();
  const int r0 = 16 * warp;
  if (r0 >= it.nq) return;
  const int nt = (it.nk + 7) / 8;
  float s[NT][4];
  scores<T, NT>(s, s_q + r0 * stride, s_k, stride, nt, width, g, c);
  Places<NT> at;
  if (bias) distances<NT>(at, s_x + 3 * (r0 + g), s_x + 3 * (r0 + g + 8), s_y, nt, c);
  const Softmax sm = softmax<NT>(s, nt, it.nk, c, a.scale2, bias ? a.slopes[h] * kLog2e : 0.0f, bias, at);
  const float inv[2] = {sm.l[0] == 0.0f ? 0.0f : tc::rcp_approx(sm.l[0]),
                        sm.l[1] == 0.0f ? 0.0f : tc::rcp_approx(sm.l[1])};
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int r = r0 + g + 8 * u;
    if (c == u && r < it.nq)
      lse[(int64_t(it.q) + r) * a.H + h] = inv[u] == 0.0f ? INFINITY : sm.m[u] + tc::lg2_approx(sm.l[u]);
  }
  T* const to = out + ((int64_t(it.q) + r0 + g) * a.H + h) * a.D;
  const int64_t to8 = int64_t(8) * a.H * a.D;
  const auto store = [&](int d, const float(&o)[4]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (r0 + g + 8 * u < it.nq)
        store_pair(to + u * to8, d + 2 * c, a.D, inv[u] == 0.0f ? 0.0f : o[2 * u] * inv[u],
                   inv[u] == 0.0f ? 0.0f : o[2 * u + 1] * inv[u], (vec & 16) != 0);
    }
  };
  if constexpr (sizeof(T) == 2) weighted_bf16<NT>(s, s_v, stride, nt, width, lane, store);
  else weighted<T, NT>(s, s_v, stride, nt, width, g, c, store);
}

// CTAs an SM that the registers are held to: 168 a thread where that spills little (512 molecules, 4 heads of 32, up to
// 32 atoms in fp32: 28.4 -> 27.2 us; bf16, 8 heads, up to 64 atoms: 101 -> 91 us), else as many as it takes (bf16 of up
// to 32 atoms takes 168 by itself: 115 us, held to them 122; width 64, up to 64 atoms: 105 us against 133).
template <typename T, int NT, int DT>
constexpr int backward_ctas = DT == 4 && (sizeof(T) == 4) == (NT == 4) ? 24 / NT : 1;

// The accumulators of dk and dv of 16 keys x up to 8 * DT components stay in registers over the query heads that share
// the key head.
template <typename T, int NT, int DT>
__global__ void __launch_bounds__(16 * NT, backward_ctas<T, NT, DT>) small_backward_kernel(
    const __grid_constant__ AttArgs a, const AttSmall* __restrict__ list, int64_t n, int stride, int shift, int vec,
    const T* __restrict__ grad, T* __restrict__ dq, T* __restrict__ dk, T* __restrict__ dv,
    float* __restrict__ slope_part, float* __restrict__ dx_part, float* __restrict__ dy_part) {
  constexpr int R = 8 * NT, N = Parts<T>::N, SP = R + 4;
  extern __shared__ __align__(16) unsigned char small_smem[];
  T* s_q = reinterpret_cast<T*>(small_smem);
  T* s_g = s_q + R * stride;
  T* s_k = s_g + R * stride;
  T* s_v = s_k + R * stride;
  float* s_p = reinterpret_cast<float*>(s_v + R * stride);
  float* s_d = s_p + R * SP;
  float* s_x = s_d + R * SP;
  float* s_y = s_x + R * 3;
  const int64_t task = blockIdx.y + int64_t(gridDim.y) * blockIdx.z;
  if (task >= n) return;
  const AttSmall it = list[task];
  const int hk = int(blockIdx.x);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int width = (a.D + 7) / 8 * 8, r0 = 16 * warp;
  const int nt = (it.nk + 7) / 8, qt = (it.nq + 7) / 8;
  const int q_rows = (it.nq + 15) / 16 * 16, k_rows = (it.nk + 15) / 16 * 16;  // what the fragments read
  const bool bias = a.slopes != nullptr, even = (vec & 16) != 0;
  load_rows<T>(s_k, stride, static_cast<const T*>(a.k) + int64_t(it.k) * a.k_row + hk * a.k_head, a.k_row, it.nk,
               k_rows, a.D, shift, vec & 2);
  load_rows<T>(s_v, stride, static_cast<const T*>(a.v) + int64_t(it.k) * a.v_row + hk * a.v_head, a.v_row, it.nk,
               k_rows, a.D, shift, vec & 4);
  if (bias) {
    load_places(s_x, a.x + int64_t(it.q) * 3, it.nq, q_rows);
    load_places(s_y, a.y + int64_t(it.k) * 3, it.nk, k_rows);
  }
  float ak[DT][4], av[DT][4], f[2][3];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int k = 0; k < 4; ++k) ak[t][k] = av[t][k] = 0.0f;
#pragma unroll
  for (int u = 0; u < 2; ++u) f[u][0] = f[u][1] = f[u][2] = 0.0f;

  for (int h = hk * a.group; h < (hk + 1) * a.group; ++h) {
    load_rows<T>(s_q, stride, static_cast<const T*>(a.q) + int64_t(it.q) * a.q_row + h * a.q_head, a.q_row, it.nq,
                 q_rows, a.D, shift, vec & 1);
    load_rows<T>(s_g, stride, grad + (int64_t(it.q) * a.H + h) * a.D, int64_t(a.H) * a.D, it.nq, q_rows, a.D, shift,
                 vec & 8);
    arrived();
    const float slope = bias ? a.slopes[h] : 0.0f;
    if (r0 < 8 * qt) {
      // ---- rows = queries: P, dS, dq and the row's sums
      float s[NT][4], tt[NT][4];
      scores<T, NT>(s, s_q + r0 * stride, s_k, stride, nt, width, g, c);
      scores<T, NT>(tt, s_g + r0 * stride, s_v, stride, nt, width, g, c);
      const float* x_of[2] = {s_x + 3 * (r0 + g), s_x + 3 * (r0 + g + 8)};
      Places<NT> at;
      if (bias) distances<NT>(at, x_of[0], x_of[1], s_y, nt, c);
      const Softmax sm = softmax<NT>(s, nt, it.nk, c, a.scale2, slope * kLog2e, bias, at);
      float delta[2] = {0.0f, 0.0f};
      const float inv[2] = {sm.l[0] == 0.0f ? 0.0f : 1.0f / sm.l[0], sm.l[1] == 0.0f ? 0.0f : 1.0f / sm.l[1]};
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (t < nt) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            s[t][k] *= inv[k >> 1];
            delta[k >> 1] = fmaf(s[t][k], tt[t][k], delta[k >> 1]);
          }
        }
      }
      delta[0] = quad_sum(delta[0]);
      delta[1] = quad_sum(delta[1]);
      float sd[2] = {0.0f, 0.0f}, fx[2][3] = {{0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f}};
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (t < nt) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int u = k >> 1, col = 8 * t + 2 * c + (k & 1);
            const float ds = s[t][k] * (tt[t][k] - delta[u]);
            tt[t][k] = ds;
            if (bias) {
              const Apart3 v = apart3(x_of[u], s_y + 3 * col);
              // 64 columns: distances formed again are cheaper than 64 registers over the softmax (95 -> 87 us)
              const float q = NT == 4 ? 0.0f : square(v), r = NT == 4 ? at.r[t][k] : tc::rsqrt_approx(q);
              const float w = ds * r;
              sd[u] = fmaf(ds, NT == 4 ? at.d[t][k] : q * r, sd[u]);
              fx[u][0] = fmaf(w, v.x, fx[u][0]);
              fx[u][1] = fmaf(w, v.y, fx[u][1]);
              fx[u][2] = fmaf(w, v.z, fx[u][2]);
            }
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int r = r0 + g + 8 * u, to = r * SP + 8 * t + 2 * c;
            const bool there = r < it.nq;  // a row past the end holds a softmax of zeros
            *reinterpret_cast<float2*>(s_p + to) =
                there ? make_float2(s[t][2 * u], s[t][2 * u + 1]) : make_float2(0.0f, 0.0f);
            *reinterpret_cast<float2*>(s_d + to) =
                there ? make_float2(tt[t][2 * u], tt[t][2 * u + 1]) : make_float2(0.0f, 0.0f);
          }
        }
      }
      T* const to = dq + ((int64_t(it.q) + r0 + g) * a.H + h) * a.D;
      const int64_t to8 = int64_t(8) * a.H * a.D;
      const auto store = [&](int d, const float(&o)[4]) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if (r0 + g + 8 * u < it.nq)
            store_pair(to + u * to8, d + 2 * c, a.D, o[2 * u] * a.scale, o[2 * u + 1] * a.scale, even);
        }
      };
      if constexpr (sizeof(T) == 2) weighted_bf16<NT>(tt, s_k, stride, nt, width, lane, store);
      else weighted<T, NT>(tt, s_k, stride, nt, width, g, c, store);
      if (bias) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int r = r0 + g + 8 * u;
          const int64_t at_row = (int64_t(it.q) + r) * a.H + h;
          sd[u] = quad_sum(sd[u]);
#pragma unroll
          for (int k = 0; k < 3; ++k) fx[u][k] = quad_sum(fx[u][k]);
          if (c == 0 && r < it.nq) {
            slope_part[at_row] = -sd[u];
#pragma unroll
            for (int k = 0; k < 3; ++k) dx_part[at_row * 3 + k] = -slope * fx[u][k];
          }
        }
      }
    }
    __syncthreads();
    if (r0 < 8 * nt) {
      // ---- rows = keys: dv += P^T G, dk += dS^T Q and the key's force
      for (int t = 0; t < qt; ++t) {
        const int q0 = 8 * t + 2 * c;
        const float* p0 = s_p + q0 * SP + r0 + g;
        const float* d0 = s_d + q0 * SP + r0 + g;
        const float w[4] = {d0[0], d0[8], d0[SP], d0[SP + 8]};
        // keys past the last block of 8 were not written by any row
        const bool hi = r0 + 8 < 8 * nt;
        const FragA<N> fp = frag_a<N, false>(p0[0], hi ? p0[8] : 0.0f, p0[SP], hi ? p0[SP + 8] : 0.0f);
        const FragA<N> fd = frag_a<N, false>(w[0], hi ? w[1] : 0.0f, w[2], hi ? w[3] : 0.0f);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          if (8 * d < width) {
            const T* g0 = s_g + q0 * stride + 8 * d + g;
            const T* x0 = s_q + q0 * stride + 8 * d + g;
            product<N>(av[d], fp, to_float(g0[0]), to_float(g0[stride]));
            product<N>(ak[d], fd, to_float(x0[0]), to_float(x0[stride]));
          }
        }
        if (bias) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int u = k & 1, q = q0 + (k >> 1);  // key g + 8 u, query q
            if (u == 1 && !hi) continue;
            const Apart3 v = apart3(s_x + 3 * q, s_y + 3 * (r0 + g + 8 * u));
            const float e = slope * w[k] * tc::rsqrt_approx(square(v));
            f[u][0] = fmaf(e, v.x, f[u][0]);
            f[u][1] = fmaf(e, v.y, f[u][1]);
            f[u][2] = fmaf(e, v.z, f[u][2]);
          }
        }
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int r = r0 + g + 8 * u;
    const int64_t at = (int64_t(it.k) + r) * a.Hk + hk;
#pragma unroll
    for (int k = 0; k < 3; ++k) f[u][k] = quad_sum(f[u][k]);
    if (r < it.nk) {
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        if (8 * d < width) {
          store_pair(dk + at * a.D, 8 * d + 2 * c, a.D, ak[d][2 * u] * a.scale, ak[d][2 * u + 1] * a.scale, even);
          store_pair(dv + at * a.D, 8 * d + 2 * c, a.D, av[d][2 * u], av[d][2 * u + 1], even);
        }
      }
      if (bias && c == 0) {
#pragma unroll
        for (int k = 0; k < 3; ++k) dy_part[at * 3 + k] = f[u][k];
      }
    }
  }
}

// Values a row in shared memory: a multiple of 16 bytes whose words are an odd multiple of 4, so that the
// fragments' reads meet every bank once.
template <typename T>
int row_stride(int D) {
  const int width = (D + 7) / 8 * 8;
  if (sizeof(T) == 4) return width + 4;
  return width + (width / 8 % 2 == 0 ? 8 : 0);
}

// log2 of the threads that take a row's 16-byte parts.
template <typename T>
int part_shift(int D) {
  const int parts = (D + 7) / 8 * 8 * int(sizeof(T)) / 16;
  int shift = 0;
  while ((1 << shift) < parts) ++shift;
  return shift;
}

// A CTA a head (x) and structure (y and z): no division in the kernel.
dim3 by_structure(int heads, int64_t n) {
  const int64_t y = std::min<int64_t>(n, 65535);
  return dim3(unsigned(heads), unsigned(y), unsigned((n + y - 1) / y));
}

template <typename T, int NT>
int forward_smem(int D) {
  return 3 * 8 * NT * row_stride<T>(D) * int(sizeof(T)) + 6 * 8 * NT * 4;
}
template <typename T, int NT>
int backward_smem(int D) {
  constexpr int R = 8 * NT;
  return 4 * R * row_stride<T>(D) * int(sizeof(T)) + 2 * R * (R + 4) * 4 + 6 * R * 4;
}

// A kernel may have what its widest head needs, whatever this call does: the limit is the kernel's, and another thread's
// call of fewer components must not lower it between the setting and the launch.
template <typename T, int NT>
int forward_class(const AttArgs& a, const AttSmall* list, int64_t n, int vec, T* out, float* lse, cudaStream_t s) {
  const auto kernel = small_forward_kernel<T, NT>;
  Y3B_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    forward_smem<T, NT>(kAttMaxWidth)));
  kernel<<<by_structure(a.H, n), 16 * NT, forward_smem<T, NT>(a.D), s>>>(a, list, n, row_stride<T>(a.D),
                                                                         part_shift<T>(a.D), vec, out, lse);
  Y3B_LAUNCH_CHECK();
  return Y3B_OK;
}

template <typename T, int NT, int DT>
int backward_class(const AttArgs& a, const AttSmall* list, int64_t n, int vec, const T* grad, T* dq, T* dk, T* dv,
                   float* slope_part, float* dx_part, float* dy_part, cudaStream_t s) {
  const auto kernel = small_backward_kernel<T, NT, DT>;
  Y3B_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    backward_smem<T, NT>(8 * DT)));
  kernel<<<by_structure(a.Hk, n), 16 * NT, backward_smem<T, NT>(a.D), s>>>(
      a, list, n, row_stride<T>(a.D), part_shift<T>(a.D), vec, grad, dq, dk, dv, slope_part, dx_part, dy_part);
  Y3B_LAUNCH_CHECK();
  return Y3B_OK;
}

bool on16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Bits: 16-byte loads of q, k, v and grad, paired stores.
template <typename T>
int vector_bits(const AttArgs& a, const void* grad, const void* o0, const void* o1, const void* o2) {
  constexpr int W = 16 / int(sizeof(T));
  const auto fits = [&](const void* p, int64_t row, int64_t head) {
    return a.D % 8 == 0 && row % W == 0 && head % W == 0 && on16(p);
  };
  const auto pairs = [&](const void* p) { return !p || reinterpret_cast<uintptr_t>(p) % (2 * sizeof(T)) == 0; };
  return (fits(a.q, a.q_row, a.q_head) ? 1 : 0) | (fits(a.k, a.k_row, a.k_head) ? 2 : 0) |
         (fits(a.v, a.v_row, a.v_head) ? 4 : 0) | (grad && fits(grad, int64_t(a.H) * a.D, a.D) ? 8 : 0) |
         (a.D % 2 == 0 && pairs(o0) && pairs(o1) && pairs(o2) ? 16 : 0);
}

}  // namespace

template <typename T>
int attention_small_forward(const AttArgs& a, const AttSmall* list, int64_t up_to_32, int64_t up_to_64, T* out,
                            float* lse, cudaStream_t s) {
  const int vec = vector_bits<T>(a, nullptr, out, nullptr, nullptr);
  if ((up_to_32 + up_to_64) * a.H > INT32_MAX) return fail(Y3B_ERR_UNSUPPORTED, "structure_attention: too many tiles");
  if (up_to_32 > 0) {
    const int rc = forward_class<T, 4>(a, list, up_to_32, vec, out, lse, s);
    if (rc) return rc;
  }
  return up_to_64 > 0 ? forward_class<T, 8>(a, list + up_to_32, up_to_64, vec, out, lse, s) : Y3B_OK;
}

template <typename T>
int attention_small_backward(const AttArgs& a, const AttSmall* list, int64_t up_to_32, int64_t up_to_64, const T* grad,
                             T* dq, T* dk, T* dv, float* slope_part, float* dx_part, float* dy_part, cudaStream_t s) {
  const int vec = vector_bits<T>(a, grad, dq, dk, dv);
  if ((up_to_32 + up_to_64) * a.Hk > INT32_MAX) return fail(Y3B_ERR_UNSUPPORTED, "structure_attention: too many tiles");
#define Y3B_SMALL(NT, n, first)                                                                                       \
  if (n > 0) {                                                                                                        \
    const int rc =                                                                                                    \
        a.D <= 32   ? backward_class<T, NT, 4>(a, list + first, n, vec, grad, dq, dk, dv, slope_part, dx_part,        \
                                               dy_part, s)                                                            \
        : a.D <= 64 ? backward_class<T, NT, 8>(a, list + first, n, vec, grad, dq, dk, dv, slope_part, dx_part,        \
                                               dy_part, s)                                                            \
                    : backward_class<T, NT, 16>(a, list + first, n, vec, grad, dq, dk, dv, slope_part, dx_part,       \
                                                dy_part, s);                                                          \
    if (rc) return rc;                                                                                                \
  }
  Y3B_SMALL(4, up_to_32, 0)
  Y3B_SMALL(8, up_to_64, up_to_32)
#undef Y3B_SMALL
  return Y3B_OK;
}

template int attention_small_forward<float>(const AttArgs&, const AttSmall*, int64_t, int64_t, float*, float*,
                                            cudaStream_t);
template int attention_small_forward<__nv_bfloat16>(const AttArgs&, const AttSmall*, int64_t, int64_t, __nv_bfloat16*,
                                                    float*, cudaStream_t);
template int attention_small_backward<float>(const AttArgs&, const AttSmall*, int64_t, int64_t, const float*, float*,
                                             float*, float*, float*, float*, float*, cudaStream_t);
template int attention_small_backward<__nv_bfloat16>(const AttArgs&, const AttSmall*, int64_t, int64_t,
                                                     const __nv_bfloat16*, __nv_bfloat16*, __nv_bfloat16*,
                                                     __nv_bfloat16*, float*, float*, float*, cudaStream_t);

}  // namespace y3b
