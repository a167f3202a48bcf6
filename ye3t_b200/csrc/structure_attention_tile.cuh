// Structure attention on the tensor cores: one kernel body for the forward and the two sides
// of the backward.
//
// A CTA takes an item: up to 128 rows of one structure, a range of its columns, one head.
//   forward    rows = queries, columns = keys     S = Q K^T            O  += P V
//   query side rows = queries, columns = keys     S = Q K^T, T = G V^T dQ += dS K
//   key side   rows = keys,    columns = queries  S = K Q^T, T = V G^T dV += P G, dK += dS Q
// (G = gradient of the output.)  Per tile of BN columns: tcgen05.mma forms the score products in
// tensor memory; thread r of the four score warps reads row r, does the softmax arithmetic in fp32 and
// writes P or dS back to tensor memory in bf16 pieces, where it is the A operand of the accumulating product
// (B: the same shared-memory column tile, read MN-major).  One warp issues the MMAs, one
// warp brings the column tiles (TMA; a tile cut by the structure's end with cp.async and zeros), so that
// nothing of another structure enters a product.
//
// What bounds it: the score warps.  A score takes one exp2 and one reciprocal square root on the special-function unit
// (16 lanes a cycle and SM, so 8 scores a cycle and SM) and 12 to 28 operations (forward with shared distances, key
// side 22, query side 28), a packed fp32 pair of which takes two issue cycles; the products of a score at D = 64 take 3/64
// of a cycle (forward).  The warps issue in 52 to 60 % of the cycles, packed pairs counted once.  Two CTAs share an SM, or
// two score groups, so that one's MMAs and waits lie under another's arithmetic; more warps an SM gained nothing.  16,384
// atoms, 8 heads of 64, bf16: forward 1.40 ms (393 TFLOP/s); 8,192 atoms: forward 406, query side 721, key side 684 us.
//
// fp32 data is carried as three bf16 pieces (8 + 8 + 8 bits): six products of pieces give each
// product to about 2^-24, and P and dS are split likewise.  With bf16 data P and dS are two pieces, 2^-17: results are then
// as far from 64 bits as their own rounding (8,192 atoms, 8 heads of 64: 1.66e-3 of the norm, the result and all
// gradients; with one piece 2.16e-3 and 2.35e-3).  The second piece costs the forward 382 -> 411 us, the query side 697 ->
// 730, the key side 571 -> 687.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "structure_attention.cuh"
#include "tcgen05.cuh"

namespace y3b {

enum AttMode { kForward = 0, kQuerySide = 1, kKeySide = 2 };

constexpr int kTileRows = 128;
constexpr int kLoadThreads = 32;

struct AttItem {
  int row, rows, col, cols, slot, pad[3];
};
struct AttJoin {
  int row, rows, first, count;
};

// A bf16 operand: element (piece, row, head, d) at piece * piece_stride + row * row_stride + head * head_stride + d.
struct AttOperand {
  const __nv_bfloat16* p;
  int64_t row, head, piece;
};

struct AttTileArgs {
  CUtensorMap cols[2];  // the column operands (K, V or Q, G) in boxes of 64 values x 1 head x BN rows
  AttOperand q, k, v, g;
  int64_t nq, nk;
  int H, Hk, D, group, chunks;  // chunks: 16-byte pieces of a row of an operand
  const float* x;
  const float* y;
  const float* slopes;
  float scale, scale2;
  const AttItem* items;
  const void* out_in;   // forward result, query side
  const void* grad_in;  // gradient of it, query side
  float* lse;           // written by the forward
  float* delta;         // written by the query side
  float* slope_part;    // [nq, H]
  float* place_part;    // [nq, H, 3] or [nk, Hk, 3]
  void* out0;           // O, dQ or dV
  void* out1;           // dK
  float* part;          // partial results of split items
  int32_t* status;
  int vec;              // 16-byte stores to out0 / out1 and loads of out_in / grad_in
};

// HP: heads of a CTA.  Two heads see the same distances, so that the forward in bf16 shares the differences, squares and
// reciprocal square roots of a pair of atoms among two: 8,192 atoms, 8 heads of 64: 384 us against 459.  The backward
// gains nothing by it: its accumulators then fill the tensor memory, one CTA an SM is left (775 against 777 us, 649
// against 638).
template <int MODE, int DP, int NP, int HP>
struct AttCfg {
  static constexpr bool KEY_BF16 = MODE == kKeySide && NP == 1 && DP == 64;
  // Columns a tile: as many as tensor and shared memory hold.  Twice the columns are 23 and 26 % faster on the
  // backward of 128-wide heads in bf16 and 14 % on the fp32 query side (4,096 atoms, 4 heads).
  static constexpr int BN = HP == 2   ? 32
                            : NP == 1 ? (MODE == kQuerySide && DP == 64 ? 32 : 64)
                            : DP == 64 ? (MODE == kQuerySide ? 64 : 32)
                                       : (MODE == kForward ? 32 : 16);
  static constexpr int STAGES = NP == 3 ? (DP == 128 && MODE != kForward ? 1 : 2) : DP == 128 ? 2 : 4;
  // Score groups of four warps; with two, each takes every other column tile: for what leaves an SM a single CTA.
  // Two CTAs of one group with 64 columns a tile and one buffer (key side), or 32 and two (query side), are 6 and 7 %
  // faster than two of two groups (8,192 atoms, 8 heads of 64, one piece of P and dS: 636 against 677 us, 777 against 837).
  static constexpr int GROUPS = MODE != kForward && STAGES > 1 && (NP == 3 || DP == 128) ? 2 : 1;
  static constexpr int MMA_WARP = 4 * GROUPS, LOAD_WARP = MMA_WARP + 1;
  static constexpr int THREADS = 32 * (LOAD_WARP + 1);
  static constexpr int ROWOPS = MODE == kForward ? 1 : 2;
  static constexpr int PANELS = DP / 64;
  static constexpr int ROW_PIECE = kTileRows * DP * 2;
  static constexpr int COL_PIECE = BN * DP * 2;
  static constexpr int COL_HEAD = 2 * NP * COL_PIECE;
  static constexpr int COL_STAGE = HP * COL_HEAD;
  static constexpr int EXTRA = 5 * BN;  // floats a stage: x, y, z, lse, delta of the columns
  // Three pieces: the row operands lie in tensor memory where they fit.  A product of 128 rows and 32 columns reads
  // 4 KB of rows from shared memory for 1 KB of columns, and six products of pieces make that the bound
  // (4,096 atoms, 4 heads of 64, rows in shared memory: query side 578 us, key side 650, without the products 189 and
  // 207; rows in tensor memory and the MMA loop entered by the whole warp: 263 and 350).
  static constexpr bool ROWS_TMEM = NP == 3 && (DP == 64 || MODE == kForward);
  static constexpr int ROW_BYTES = ROWS_TMEM ? 0 : HP * ROWOPS * NP * ROW_PIECE;
  // Tensor memory columns.  P and dS, in AP pieces of BN / 2 columns each, take the place of the scores they come from.
  // Two pieces lie by turns, so that those of 16 columns fill these columns and no others.
  static constexpr int AP = NP == 1 ? 2 : 3;
  __device__ static constexpr int piece_at(int piece, int step) {
    return AP == 2 ? step * 16 + piece * 8 : piece * (BN / 2) + step * 8;
  }
  // Score buffers: with two, the products of tile j + 1 run under the arithmetic of tile j (a single
  // stage of columns allows one).
  static constexpr int BUFS = STAGES > 1 && !KEY_BF16 ? 2 : 1;
  static constexpr int T = BN;  // T within a buffer
  static constexpr int A0 = 0;
  static constexpr int A1 = NP == 1 ? BN : NP * BN / 2;
  static constexpr int BUF = MODE == kForward ? (NP == 1 ? BN : NP * BN / 2)
                             : MODE == kKeySide ? (NP == 1 ? 2 * BN : NP * BN)
                                                : 2 * BN;  // of one head
  static constexpr int ACC = BUFS * HP * BUF;
  // Accumulators: OPS results (dV and dK on the key side).  The tensor cores truncate when they accumulate; three
  // pieces are six products, each of which truncates the long sum.  The score warps therefore add the accumulator
  // to a total in fp32 every FLUSH tiles, and it starts again.  With one piece the
  // query side also accumulates P K, to correct dQ for the rounding of delta.
  static constexpr int OPS = MODE == kKeySide ? 2 : 1;
  static constexpr int FLUSH = 2;  // 4,096 atoms: errors of 3 to 5e-7 against 64 bits; 8 tiles 9e-7, never 2e-6
  static constexpr int TOTALS = NP == 3 ? OPS : 0;
  static constexpr bool FIX = MODE == kQuerySide && NP == 1;
  static constexpr int HALVES = MODE == kKeySide && NP == 3 && DP == 128 ? 2 : 1;  // CTAs that share a width
  static constexpr int W = DP / HALVES;  // columns of one accumulator
  // the totals lie in shared memory, [component][row], where the row operands leave it free
  static constexpr bool TOTALS_SMEM = ROWS_TMEM;
  static constexpr int NACC = OPS + (TOTALS_SMEM ? 0 : TOTALS) + (FIX ? 1 : 0);  // accumulators of one head
  static constexpr int ROWS = ACC + HP * NACC * W;                                // row operands
  static constexpr int NEED = ROWS + (ROWS_TMEM ? ROWOPS * NP * DP / 2 : 0);
  static constexpr int SMEM = 1024 + ROW_BYTES + STAGES * (COL_STAGE + EXTRA * 4) +
                              (TOTALS_SMEM ? TOTALS * W * kTileRows * 4 : 0);
  static constexpr int COLUMNS = NEED <= 128 ? 128 : NEED <= 256 ? 256 : 512;
  static_assert(NEED <= 512 && SMEM <= 227 * 1024 && ACC % 16 == 0 && FLUSH % GROUPS == 0, "tile shape");
  static constexpr int PER_SM_TMEM = 512 / COLUMNS;
  static constexpr int PER_SM_SMEM = (227 * 1024) / (SMEM + 2048);
  static constexpr int PER_SM_MIN = PER_SM_TMEM < PER_SM_SMEM ? PER_SM_TMEM : PER_SM_SMEM;
  static constexpr int PER_SM = PER_SM_MIN > 2 ? 2 : PER_SM_MIN;
  // floats of one row of a split item's partial result
  static constexpr int PART = (MODE == kKeySide || FIX ? 2 : 1) * DP + 16;
};

// Two-operand piece products, smallest first.
template <int NP> struct Pieces;
template <> struct Pieces<1> {
  static constexpr int N = 1;
  __device__ static constexpr int a(int) { return 0; }
  __device__ static constexpr int b(int) { return 0; }
};
template <> struct Pieces<3> {
  static constexpr int N = 6;
  __device__ static constexpr int a(int n) { return n == 0 ? 2 : n == 2 ? 1 : n == 3 ? 1 : 0; }
  __device__ static constexpr int b(int n) { return n == 1 ? 2 : n == 2 ? 1 : n == 4 ? 1 : 0; }
};
// The same of the accumulating products, whose A operand has two pieces where the data has one.
template <int NP> struct AccPieces : Pieces<NP> {};
template <> struct AccPieces<1> {
  static constexpr int N = 2;
  __device__ static constexpr int a(int n) { return 1 - n; }
  __device__ static constexpr int b(int) { return 0; }
};

// Rows [0, valid) of an operand into a tile of ROWS x DP in the 128-byte swizzle, zeros elsewhere.
template <int ROWS, int DP, int NP>
__device__ __forceinline__ void load_tile(uint32_t dst, const AttOperand& o, int64_t row0, int head, int valid,
                                          int chunks, int t, int threads) {
  constexpr int CH = DP / 8;
  const __nv_bfloat16* base = o.p + row0 * o.row + head * o.head;
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    for (int u = t; u < ROWS * CH; u += threads) {
      const int r = u / CH, c = u % CH;
      const uint32_t at = dst + p * (ROWS * DP * 2) + (c >> 3) * (ROWS * 128) + (r >> 3) * 1024 + (r & 7) * 128 +
                          (((c & 7) ^ (r & 7)) << 4);
      const bool there = r < valid && c < chunks;
      const __nv_bfloat16* src = there ? base + p * o.piece + int64_t(r) * o.row + c * 8 : o.p;
      tc::cp16(at, src, there);
    }
  }
}

// Values (2k, 2k + 1) as NP packed bf16 pieces.
template <int NP>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&r)[NP]) {
  r[0] = tc::bf16x2(a, b);
#pragma unroll
  for (int p = 1; p < NP; ++p) {
    a -= __uint_as_float(r[p - 1] << 16);
    b -= __uint_as_float(r[p - 1] & 0xffff0000u);
    r[p] = tc::bf16x2(a, b);
  }
}

template <typename T>
__device__ __forceinline__ void store_row16(T* dst, const float* v, int d0, int D, bool vec) {
  if (vec && d0 + 16 <= D) {
    if constexpr (sizeof(T) == 2) {
      uint32_t r[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) r[k] = tc::bf16x2(v[2 * k], v[2 * k + 1]);
      reinterpret_cast<uint4*>(dst + d0)[0] = make_uint4(r[0], r[1], r[2], r[3]);
      reinterpret_cast<uint4*>(dst + d0)[1] = make_uint4(r[4], r[5], r[6], r[7]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        reinterpret_cast<float4*>(dst + d0)[k] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 16; ++k)
      if (d0 + k < D) dst[d0 + k] = from_float<T>(v[k]);
  }
}

// Distances of a pair of columns and their reciprocals from the squares.  The squares come with a
// tiny term, so that 1/d stays finite and (x - y) / d is zero at distance zero.  Every mode forms its
// scores by the same operations: the backward then sees the forward's scores bit for bit.
struct Distance {
  tc::f2 d, r;
};
__device__ __forceinline__ Distance distance(tc::f2 squares) {
  float u0, u1;
  tc::unpack(squares, u0, u1);
  Distance x;
  x.r = tc::pack(tc::rsqrt_approx(u0), tc::rsqrt_approx(u1));
  x.d = tc::mul2(squares, x.r);
  return x;
}

template <int MODE, int DP, int NP, int HP, bool BIAS>
__global__ void __launch_bounds__(AttCfg<MODE, DP, NP, HP>::THREADS, AttCfg<MODE, DP, NP, HP>::PER_SM)
    attention_tile_kernel(const __grid_constant__ AttTileArgs a) {
  using C = AttCfg<MODE, DP, NP, HP>;
  using T = typename std::conditional<NP == 1, __nv_bfloat16, float>::type;
  constexpr int BN = C::BN;
  extern __shared__ __align__(1024) unsigned char tile_smem[];
  __shared__ __align__(8) uint64_t bars[2 * C::STAGES + 2 * C::BUFS + 1];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int heads = MODE == kKeySide ? a.Hk : a.H;
  const int half = C::HALVES == 1 ? 0 : int(blockIdx.x % C::HALVES);
  const unsigned task = blockIdx.x / C::HALVES;
  const unsigned head_blocks = unsigned(heads) / HP;
  const int head0 = int(task % head_blocks) * HP;  // heads head0 .. head0 + HP
  const AttItem item = a.items[task / head_blocks];
  const int d_first = half * C::W;                                            // accumulated components: d_first ..
  const int d_count = C::HALVES == 1 ? a.D : min(a.D - d_first, int(C::W));   // .. d_first + d_count (D > 64 with halves)
  const int acc_n = (d_count + 15) / 16 * 16;
  const int ntiles = (item.cols + BN - 1) / BN;
  const int total = MODE == kKeySide ? ntiles * a.group : ntiles;

  const uint32_t smem = (tc::smem_addr(tile_smem) + 1023u) & ~1023u;
  const uint32_t rows_at = smem;  // (head, operand) one after the other
  const uint32_t cols = smem + C::ROW_BYTES;
  float* extra = reinterpret_cast<float*>(tile_smem + (cols - tc::smem_addr(tile_smem)) + C::STAGES * C::COL_STAGE);
  [[maybe_unused]] float* totals = extra + C::STAGES * C::EXTRA;
  const uint32_t bar0 = tc::smem_addr(bars);
  const auto full = [&](int s) { return bar0 + 8 * s; };
  const auto empty = [&](int s) { return bar0 + 8 * (C::STAGES + s); };
  const auto s_ready = [&](int j) { return bar0 + 8 * (2 * C::STAGES + j % C::BUFS); };
  const auto p_ready = [&](int j) { return bar0 + 8 * (2 * C::STAGES + C::BUFS + j % C::BUFS); };
  const uint32_t drain = bar0 + 8 * (2 * C::STAGES + 2 * C::BUFS);

  if (warp == C::MMA_WARP) tc::alloc(tc::smem_addr(&s_tmem), C::COLUMNS);
  if (tid == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      tc::mbar_init(full(s), kLoadThreads);
      tc::mbar_init(empty(s), 1);
    }
    for (int k = 0; k < C::BUFS; ++k) {
      tc::mbar_init(s_ready(k), 1);
      tc::mbar_init(p_ready(k), 4);
    }
    tc::mbar_init(drain, 1);
    tc::mbar_init_fence();
    s_abort = 0;
  }
  // row operands, by all threads
  if constexpr (!C::ROWS_TMEM) {
#pragma unroll
    for (int u = 0; u < HP * C::ROWOPS; ++u) {
      const int h = u / C::ROWOPS, op = u % C::ROWOPS;
      load_tile<kTileRows, DP, NP>(rows_at + u * NP * C::ROW_PIECE, MODE == kKeySide ? (op ? a.v : a.k) : op ? a.g : a.q,
                                   item.row, head0 + h, item.rows, a.chunks, tid, C::THREADS);
    }
    tc::cp_commit();
    tc::cp_wait<0>();
    tc::fence_async_smem();
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = s_tmem;
  if constexpr (C::ROWS_TMEM) {
    // or into tensor memory, a thread its row: two values a column, DP / 2 columns a piece
    if (warp < C::MMA_WARP) {
      const int r = tid & (kTileRows - 1);
      const uint32_t dst = tmem + (uint32_t(32 * (warp & 3)) << 16) + C::ROWS;
#pragma unroll 1
      for (int u = tid / kTileRows; u < C::ROWOPS * NP; u += C::GROUPS) {
        const int op = u / NP, piece = u - op * NP;
        const AttOperand& o = MODE == kKeySide ? (op ? a.v : a.k) : op ? a.g : a.q;
        const __nv_bfloat16* src = o.p + piece * o.piece + (int64_t(item.row) + r) * o.row + head0 * o.head;
#pragma unroll
        for (int c = 0; c < DP / 8; c += 4) {
          uint32_t w[16];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint4 x = make_uint4(0u, 0u, 0u, 0u);
            if (r < item.rows && c + k < a.chunks) x = *reinterpret_cast<const uint4*>(src + (c + k) * 8);
            w[4 * k] = x.x;
            w[4 * k + 1] = x.y;
            w[4 * k + 2] = x.z;
            w[4 * k + 3] = x.w;
          }
          tc::st16(dst + u * (DP / 2) + c * 4, w);
        }
      }
      tc::wait_st();
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
  }

  if (warp == C::LOAD_WARP) {
    // ---- loading warp.  A full column tile comes by TMA; one cut short by the structure's end by
    // cp.async, with zeros past it: rows of the next structure, whatever they hold, stay out.
    const int t = lane;
    bool ok = true;
    int j = 0;
    for (; j < total; ++j) {
      const int s = j % C::STAGES;
      if (j >= C::STAGES) ok = tc::mbar_wait(empty(s), ((j / C::STAGES) - 1) & 1);
      if (!ok) break;
      const int sub = MODE == kKeySide ? j / ntiles : 0, jt = MODE == kKeySide ? j - sub * ntiles : j;
      const int c0 = jt * BN, n = item.cols - c0 < BN ? item.cols - c0 : BN;
      const int64_t col = int64_t(item.col) + c0;
      const uint32_t dst = cols + s * C::COL_STAGE;
      const auto head_of = [&](int h) { return MODE == kKeySide ? (head0 + h) * a.group + sub : (head0 + h) / a.group; };
      if (n == BN) {
        if (t == 0) {
          tc::mbar_expect(full(s), C::COL_STAGE);
#pragma unroll
          for (int u = 0; u < HP * 2 * NP; ++u) {
            const int h = u / (2 * NP), op = u / NP % 2, p = u % NP;
#pragma unroll
            for (int q = 0; q < C::PANELS; ++q)
              tc::tma_load4(dst + u * C::COL_PIECE + q * (BN * 128), &a.cols[op], full(s), q * 64, head_of(h), int(col),
                            p);
          }
        }
      } else {
#pragma unroll
        for (int u = 0; u < HP * 2; ++u) {
          load_tile<BN, DP, NP>(dst + u * NP * C::COL_PIECE, MODE == kKeySide ? (u % 2 ? a.g : a.q) : u % 2 ? a.v : a.k,
                                col, head_of(u / 2), n, a.chunks, t, kLoadThreads);
        }
      }
      const uint32_t ex = tc::smem_addr(extra + s * C::EXTRA);
      if constexpr (BIAS) {
        const float* pos = MODE == kKeySide ? a.x : a.y;
        for (int u = t; u < 3 * BN; u += kLoadThreads) {
          const int r = u / 3, c = u - 3 * r;
          tc::cp4(ex + (c * BN + r) * 4, r < n ? pos + 3 * (col + r) + c : pos, r < n);
        }
      }
      if constexpr (MODE == kKeySide) {
        for (int u = t; u < 2 * BN; u += kLoadThreads) {
          const int c = u / BN, r = u % BN;
          const float* src = c ? a.delta : a.lse;
          tc::cp4(ex + (3 * BN + u) * 4, r < n ? src + (col + r) * a.H + head_of(0) : src, r < n);
        }
      }
      tc::cp_commit();
      tc::cp_wait<0>();
      tc::fence_async_smem();
      tc::mbar_arrive(full(s));
    }
    if (!ok) s_abort = 1;
    // no copy is in flight when the CTA ends, also where a warp gave up before it came
    for (int k = j > C::STAGES ? j - C::STAGES : 0; k < j; ++k) tc::mbar_wait(full(k % C::STAGES), (k / C::STAGES) & 1);
  } else if (warp == C::MMA_WARP) {
    // ---- MMA issue: scores of tile j, then (when P is back) its accumulating product
    {
      const bool lead = tc::elect();
      const int ksteps = (a.D + 15) / 16;
      const uint32_t id_s = tc::idesc_bf16(kTileRows, BN, false), id_a = tc::idesc_bf16(kTileRows, acc_n, true);
      // every lane waits, one issues
      const auto wait = [&](uint32_t bar, uint32_t parity) {
        const bool done = __all_sync(0xffffffffu, tc::mbar_wait(bar, parity));
        tc::fence_after();
        return done;
      };
      // Descriptors are formed once, and each MMA adds a constant to their address field (16-byte units).
      [[maybe_unused]] const uint64_t rows_desc = tc::desc_sw128(rows_at, 16, 1024);
      const uint64_t cols_k = tc::desc_sw128(cols, 16, 1024), cols_mn = tc::desc_sw128(cols, BN * 128, 1024);
      const auto issue_scores = [&](int j) {
        const int s = j % C::STAGES;
        if (!wait(full(s), (j / C::STAGES) & 1)) return false;
        const uint64_t b0 = cols_k + uint64_t(s * (C::COL_STAGE / 16));
        const uint32_t buf = tmem + (j % C::BUFS) * (HP * C::BUF);
        if (lead) {
#pragma unroll
          for (int n = 0; n < Pieces<NP>::N; ++n) {
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) {
              if (ks >= ksteps) continue;
#pragma unroll
              for (int u = 0; u < HP * C::ROWOPS; ++u) {
                const int h = u / C::ROWOPS, op = u % C::ROWOPS, off = (ks & 3) * 32;
                const uint64_t b = b0 + uint64_t((h * C::COL_HEAD + (op * NP + Pieces<NP>::b(n)) * C::COL_PIECE +
                                                  (ks >> 2) * (BN * 128) + off) / 16);
                const uint32_t d = buf + h * C::BUF + (op ? C::T : 0);
                if constexpr (C::ROWS_TMEM) {
                  tc::mma_ts(d, tmem + C::ROWS + (op * NP + Pieces<NP>::a(n)) * (DP / 2) + ks * 8, b, id_s,
                             n > 0 || ks > 0);
                } else {
                  const uint64_t r = rows_desc + uint64_t(((u * NP + Pieces<NP>::a(n)) * C::ROW_PIECE +
                                                           (ks >> 2) * (kTileRows * 128) + off) / 16);
                  tc::mma_ss(d, r, b, id_s, n > 0 || ks > 0);
                }
              }
            }
          }
          tc::commit(s_ready(j));
        }
        __syncwarp();
        return true;
      };
      bool ok = total == 0 || issue_scores(0);
      for (int j = 0; ok && j < total; ++j) {
        const int s = j % C::STAGES;
        if (C::BUFS == 2 && j + 1 < total) ok = issue_scores(j + 1);
        if (!ok) break;
        ok = wait(p_ready(j), (j / C::BUFS) & 1);
        if (!ok) break;
        // forward: P x V; query side: dS x K (and P x K); key side: P x G and dS x Q
        const uint64_t b0 = cols_mn + uint64_t(s * (C::COL_STAGE / 16) + half * (BN * 128 / 16));
        const uint32_t buf = tmem + (j % C::BUFS) * (HP * C::BUF);
        const uint32_t go_on = C::TOTALS ? j % C::FLUSH > 0 : j > 0;
        if (lead) {
          constexpr int kOps = C::OPS + (C::FIX ? 1 : 0);
#pragma unroll
          for (int n = 0; n < AccPieces<NP>::N; ++n) {
#pragma unroll
            for (int ks = 0; ks < BN / 16; ++ks) {
#pragma unroll
              for (int u = 0; u < HP * kOps; ++u) {
                const int h = u / kOps, op = u % kOps;
                const bool one = C::FIX && op == 1;  // P K, the small correction's factor, has one piece
                if (one && AccPieces<NP>::a(n) > 0) continue;
                const int second = MODE == kForward || (MODE == kKeySide && op == 0) ? 1 : 0;  // V or G
                tc::mma_ts(tmem + C::ACC + (h * C::NACC + op) * C::W,
                           buf + h * C::BUF + (op == 0 ? C::A0 : C::A1) + C::piece_at(AccPieces<NP>::a(n), ks),
                           b0 + uint64_t((h * C::COL_HEAD + (second * NP + AccPieces<NP>::b(n)) * C::COL_PIECE +
                                          ks * 2048) / 16),
                           id_a, ks > 0 || (n > 0 && !one) ? 1u : go_on);
              }
            }
          }
          tc::commit(empty(s));
        }
        __syncwarp();
        if (C::BUFS == 1 && j + 1 < total) ok = issue_scores(j + 1);
      }
      if (!ok) s_abort = 1;
      if (lead) tc::commit(drain);
      __syncwarp();
      tc::mbar_wait(drain, 0);  // no product either
    }
    __syncwarp();
  } else {
    // ---- score warps: thread = row, in each group
    const int r_tile = tid & (kTileRows - 1), group = C::GROUPS == 1 ? 0 : tid / kTileRows;
    const bool valid = r_tile < item.rows;
    const int64_t row = int64_t(item.row) + (valid ? r_tile : 0);
    const uint32_t lane_base = tmem + (uint32_t(32 * (warp & 3)) << 16);
    float px = 0.0f, py = 0.0f, pz = 0.0f, slope[HP];
    tc::f2 nslope2[HP];
    const auto set_slopes = [&](int sub) {
#pragma unroll
      for (int h = 0; h < HP; ++h) {
        slope[h] = 0.0f;
        if (BIAS) slope[h] = a.slopes[MODE == kKeySide ? (head0 + h) * a.group + sub : head0 + h];
        nslope2[h] = tc::pack(-slope[h] * kLog2e, -slope[h] * kLog2e);
      }
    };
    set_slopes(0);
    if constexpr (BIAS) {
      const float* pos = (MODE == kKeySide ? a.y : a.x) + 3 * row;
      px = pos[0];
      py = pos[1];
      pz = pos[2];
    }
    const tc::f2 px2 = tc::pack(px, px), py2 = tc::pack(py, py), pz2 = tc::pack(pz, pz);
    const tc::f2 scale2 = tc::pack(a.scale2, a.scale2), tiny2 = tc::pack(1e-30f, 1e-30f);
    bool ok = true;

    // state of the forward: each head's reference maximum and sum; of the query side: the ten sums; of the key side: the
    // force
    float m[HP], l[HP];
#pragma unroll
    for (int h = 0; h < HP; ++h) {
      m[h] = -INFINITY;
      l[h] = 0.0f;
    }
    float nL = 0.0f, delta0 = 0.0f;
    constexpr int SUMS = MODE == kQuerySide ? 10 : 3;
    float sum[SUMS];
    tc::f2 acc[SUMS];
#pragma unroll
    for (int k = 0; k < SUMS; ++k) {
      sum[k] = 0.0f;
      acc[k] = tc::pack(0.0f, 0.0f);
    }
    if constexpr (MODE == kQuerySide) {
      if (valid) {
        const int64_t at = row * a.H + head0;
        nL = -a.lse[at];
        const T* o = static_cast<const T*>(a.out_in) + at * a.D;
        const T* g = static_cast<const T*>(a.grad_in) + at * a.D;
        constexpr int W = 16 / int(sizeof(T));
        int d = 0;
        if (a.vec) {
          for (; d + W <= a.D; d += W) {
            const uint4 ou = *reinterpret_cast<const uint4*>(o + d), gu = *reinterpret_cast<const uint4*>(g + d);
            const T* ov = reinterpret_cast<const T*>(&ou);
            const T* gv = reinterpret_cast<const T*>(&gu);
#pragma unroll
            for (int k = 0; k < W; ++k) delta0 = fmaf(to_float(ov[k]), to_float(gv[k]), delta0);
          }
        }
        for (; d < a.D; ++d) delta0 = fmaf(to_float(o[d]), to_float(g[d]), delta0);
      }
    }
    const tc::f2 nL2 = tc::pack(nL, nL), delta02 = tc::pack(delta0, delta0);

    // row sums go from pairs within a few tiles to the row's: two levels keep the rounding of long rows small
    const auto fold = [&] {
#pragma unroll
      for (int k = 0; k < SUMS; ++k) {
        float s0, s1;
        tc::unpack(acc[k], s0, s1);
        if constexpr (MODE == kKeySide) sum[k] = fmaf(slope[0], s0 + s1, sum[k]);
        else sum[k] += s0 + s1;
        acc[k] = tc::pack(0.0f, 0.0f);
      }
    };

    // The accumulators of the tiles before j into the totals.
    const auto flush = [&](int j) {
      const bool first = j == C::FLUSH;
      for (int d = 0; d < C::OPS * C::W; d += 16) {
        float o[16], e[16];
        tc::ld16(lane_base + C::ACC + d, o);
        if (!C::TOTALS_SMEM && !first) tc::ld16(lane_base + C::ACC + C::OPS * C::W + d, e);
        if (C::TOTALS_SMEM && !first) {
#pragma unroll
          for (int k = 0; k < 16; ++k) e[k] = totals[(d + k) * kTileRows + r_tile];
        }
        tc::wait_ld();
#pragma unroll
        for (int k = 0; k < 16; ++k) o[k] = first ? o[k] : e[k] + o[k];
        if constexpr (C::TOTALS_SMEM) {
#pragma unroll
          for (int k = 0; k < 16; ++k) totals[(d + k) * kTileRows + r_tile] = o[k];
        } else {
          uint32_t r[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) r[k] = __float_as_uint(o[k]);
          tc::st16(lane_base + C::ACC + C::OPS * C::W + d, r);
        }
      }
      if constexpr (!C::TOTALS_SMEM) tc::wait_st();
    };

    // One tile's arithmetic; n < BN columns where CUT, all of them otherwise.
    const auto forward_tile = [&](auto cut, int j, int n, const float* ex, uint32_t buf) {
      constexpr bool CUT = decltype(cut)::value;
      float v[HP][BN];
#pragma unroll
      for (int h = 0; h < HP; ++h)
#pragma unroll
        for (int c = 0; c < BN; c += 16) tc::ld16(buf + h * C::BUF + c, v[h] + c);
      tc::wait_ld();
      float top[HP];
#pragma unroll
      for (int h = 0; h < HP; ++h) top[h] = -INFINITY;
#pragma unroll
      for (int c = 0; c < BN; c += 4) {
        [[maybe_unused]] tc::f2 d0, d1;
        if constexpr (BIAS) {
          const ulonglong2 xx = *reinterpret_cast<const ulonglong2*>(ex + c);
          const ulonglong2 yy = *reinterpret_cast<const ulonglong2*>(ex + BN + c);
          const ulonglong2 zz = *reinterpret_cast<const ulonglong2*>(ex + 2 * BN + c);
          const tc::f2 dx0 = tc::sub2(px2, xx.x), dx1 = tc::sub2(px2, xx.y);
          const tc::f2 dy0 = tc::sub2(py2, yy.x), dy1 = tc::sub2(py2, yy.y);
          const tc::f2 dz0 = tc::sub2(pz2, zz.x), dz1 = tc::sub2(pz2, zz.y);
          d0 = distance(tc::fma2(dz0, dz0, tc::fma2(dy0, dy0, tc::fma2(dx0, dx0, tiny2)))).d;
          d1 = distance(tc::fma2(dz1, dz1, tc::fma2(dy1, dy1, tc::fma2(dx1, dx1, tiny2)))).d;
        }
#pragma unroll
        for (int h = 0; h < HP; ++h) {
          float* w = v[h] + c;
          tc::f2 s0 = tc::mul2(tc::pack(w[0], w[1]), scale2), s1 = tc::mul2(tc::pack(w[2], w[3]), scale2);
          if constexpr (BIAS) {
            s0 = tc::fma2(d0, nslope2[h], s0);
            s1 = tc::fma2(d1, nslope2[h], s1);
          }
          tc::unpack(s0, w[0], w[1]);
          tc::unpack(s1, w[2], w[3]);
          if constexpr (CUT) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (c + k >= n) w[k] = -INFINITY;
          }
          top[h] = tc::max3(tc::max3(top[h], w[0], w[1]), w[2], w[3]);
        }
      }
      // the reference maximum moves only when a row would pass 2^8 times it: P stays within 2^8
      // and the accumulated rows are rescaled seldom
      if (j == 0) {
#pragma unroll
        for (int h = 0; h < HP; ++h) m[h] = top[h];
      } else {
        bool move[HP], any = false;
#pragma unroll
        for (int h = 0; h < HP; ++h) {
          move[h] = top[h] > m[h] + 8.0f || (m[h] == -INFINITY && top[h] > m[h]);
          any = any || move[h];
        }
        if (__any_sync(0xffffffffu, any)) {
          if (!__all_sync(0xffffffffu, tc::mbar_wait(empty((j - 1) % C::STAGES), ((j - 1) / C::STAGES) & 1)))
            return false;
          tc::fence_after();
#pragma unroll
          for (int h = 0; h < HP; ++h) {
            const float f = move[h] ? tc::ex2(m[h] - top[h]) : 1.0f;
            if (move[h]) m[h] = top[h];
            l[h] *= f;
#pragma unroll
            for (int u = 0; u < C::NACC; ++u) {
              for (int d = 0; d < acc_n; d += 16) {
                float o[16];
                tc::ld16(lane_base + C::ACC + (h * C::NACC + u) * C::W + d, o);
                tc::wait_ld();
                uint32_t r[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) r[k] = __float_as_uint(o[k] * f);
                tc::st16(lane_base + C::ACC + (h * C::NACC + u) * C::W + d, r);
              }
            }
            if constexpr (C::TOTALS_SMEM) {
              if (j > C::FLUSH) {
                for (int d = 0; d < acc_n; ++d) totals[d * kTileRows + r_tile] *= f;
              }
            }
          }
          tc::wait_st();
        }
      }
#pragma unroll
      for (int h = 0; h < HP; ++h) {
        const float ref = m[h] == -INFINITY ? 0.0f : m[h];
        const tc::f2 nref = tc::pack(-ref, -ref);
        tc::f2 l0 = tc::pack(0.0f, 0.0f), l1 = l0;
        const uint32_t dst = lane_base + C::A0 + ((j % C::BUFS) * HP + h) * C::BUF;
#pragma unroll
        for (int c0 = 0; c0 < BN; c0 += 16) {
          uint32_t pr[C::AP][8];
#pragma unroll
          for (int c = 0; c < 16; c += 2) {
            float e0, e1;
            tc::unpack(tc::add2(tc::pack(v[h][c0 + c], v[h][c0 + c + 1]), nref), e0, e1);
            e0 = tc::ex2(e0);
            e1 = tc::ex2(e1);
            if (c & 2) l1 = tc::add2(l1, tc::pack(e0, e1));
            else l0 = tc::add2(l0, tc::pack(e0, e1));
            uint32_t r[C::AP];
            split_pair<C::AP>(e0, e1, r);
#pragma unroll
            for (int p = 0; p < C::AP; ++p) pr[p][c / 2] = r[p];
          }
#pragma unroll
          for (int p = 0; p < C::AP; ++p) tc::st8(dst + C::piece_at(p, c0 / 16), pr[p]);
        }
        float s0, s1;
        tc::unpack(tc::add2(l0, l1), s0, s1);
        l[h] += s0 + s1;
      }
      return true;
    };

    const auto backward_tile = [&](auto cut, int j, int n, const float* ex, uint32_t buf) {
      constexpr bool CUT = decltype(cut)::value;
      const uint32_t dst = lane_base + (j % C::BUFS) * C::BUF;
      // bf16 data: the next 16 columns load under these; P and dS of columns c0 .. take the columns that were read.  Three
      // pieces take more than that: all scores come to registers first.
      constexpr int HOLD = NP == 1 ? 2 : BN / 16;
      float sv[HOLD][16], tv[HOLD][16];
#pragma unroll
      for (int k = 0; k < (NP == 1 ? 1 : HOLD); ++k) {
        tc::ld16(buf + 16 * k, sv[k]);
        tc::ld16(buf + C::T + 16 * k, tv[k]);
      }
#pragma unroll
      for (int c0 = 0; c0 < BN; c0 += 16) {
        constexpr int kLast = BN - 16;
        const int cur = (c0 / 16) % HOLD;
        if (NP == 1 || c0 == 0) tc::wait_ld();
        if (NP == 1 && c0 < kLast) {
          tc::ld16(buf + c0 + 16, sv[cur ^ 1]);
          tc::ld16(buf + C::T + c0 + 16, tv[cur ^ 1]);
        }
        constexpr int PP = MODE == kKeySide ? C::AP : 1;  // pieces of P
        [[maybe_unused]] uint32_t pr[PP][8];
        uint32_t dr[C::AP][8];
#pragma unroll
        for (int c = 0; c < 16; c += 2) {
          const int cc = c0 + c;
          [[maybe_unused]] tc::f2 dx, dy, dz, d, r;
          tc::f2 score = tc::mul2(tc::pack(sv[cur][c], sv[cur][c + 1]), scale2);
          if constexpr (BIAS) {
            dx = tc::sub2(px2, *reinterpret_cast<const tc::f2*>(ex + cc));
            dy = tc::sub2(py2, *reinterpret_cast<const tc::f2*>(ex + BN + cc));
            dz = tc::sub2(pz2, *reinterpret_cast<const tc::f2*>(ex + 2 * BN + cc));
            const Distance x = distance(tc::fma2(dz, dz, tc::fma2(dy, dy, tc::fma2(dx, dx, tiny2))));
            d = x.d;
            r = x.r;
            score = tc::fma2(d, nslope2[0], score);
          }
          float p0, p1;
          if constexpr (MODE == kQuerySide) tc::unpack(tc::add2(score, nL2), p0, p1);
          else tc::unpack(tc::sub2(score, *reinterpret_cast<const tc::f2*>(ex + 3 * BN + cc)), p0, p1);
          p0 = tc::ex2(p0);
          p1 = tc::ex2(p1);
          if constexpr (CUT) {
            if (cc >= n) p0 = 0.0f;
            if (cc + 1 >= n) p1 = 0.0f;
          }
          const tc::f2 p = tc::pack(p0, p1), tt = tc::pack(tv[cur][c], tv[cur][c + 1]);
          float g0, g1;
          if constexpr (MODE == kQuerySide) {
            // with delta from the rounded result; what delta is off by follows from the sums
            const tc::f2 ds = tc::mul2(p, tc::sub2(tt, delta02));
            tc::unpack(ds, g0, g1);
            acc[0] = tc::add2(acc[0], ds);
            acc[9] = tc::add2(acc[9], p);
            if constexpr (BIAS) {
              acc[1] = tc::fma2(d, ds, acc[1]);
              acc[2] = tc::fma2(d, p, acc[2]);
              const tc::f2 u = tc::mul2(ds, r), w = tc::mul2(p, r);
              acc[3] = tc::fma2(u, dx, acc[3]);
              acc[4] = tc::fma2(u, dy, acc[4]);
              acc[5] = tc::fma2(u, dz, acc[5]);
              acc[6] = tc::fma2(w, dx, acc[6]);
              acc[7] = tc::fma2(w, dy, acc[7]);
              acc[8] = tc::fma2(w, dz, acc[8]);
            }
          } else {
            const tc::f2 ds = tc::mul2(p, tc::sub2(tt, *reinterpret_cast<const tc::f2*>(ex + 4 * BN + cc)));
            tc::unpack(ds, g0, g1);
            if constexpr (BIAS) {
              const tc::f2 u = tc::mul2(ds, r);
              acc[0] = tc::fma2(u, dx, acc[0]);
              acc[1] = tc::fma2(u, dy, acc[1]);
              acc[2] = tc::fma2(u, dz, acc[2]);
            }
          }
          if constexpr (MODE == kKeySide || C::FIX) {
            uint32_t q[PP];
            split_pair<PP>(p0, p1, q);
#pragma unroll
            for (int k = 0; k < PP; ++k) pr[k][c / 2] = q[k];
          }
          uint32_t q[C::AP];
          split_pair<C::AP>(g0, g1, q);
#pragma unroll
          for (int k = 0; k < C::AP; ++k) dr[k][c / 2] = q[k];
        }
        // key side: P first, then dS, stored by turns (8,192 atoms, 8 heads: 687 us, one after the other 723); query side:
        // dS first
#pragma unroll
        for (int k = 0; k < C::AP; ++k) {
          tc::st8(dst + (MODE == kKeySide ? C::A1 : C::A0) + C::piece_at(k, c0 / 16), dr[k]);
          if constexpr (MODE == kKeySide) tc::st8(dst + C::A0 + C::piece_at(k, c0 / 16), pr[k]);
        }
        if constexpr (C::FIX) tc::st8(dst + C::A1 + C::piece_at(0, c0 / 16), pr[0]);
      }
      return true;
    };

    [[maybe_unused]] int last_sub = -1;
    for (int j = group; j < total; j += C::GROUPS) {
      const int s = j % C::STAGES;
      const int sub = MODE == kKeySide ? j / ntiles : 0, jt = MODE == kKeySide ? j - sub * ntiles : j;
      const int n = item.cols - jt * BN;  // columns there are, BN or more in a full tile
      ok = tc::mbar_wait(full(s), (j / C::STAGES) & 1) && tc::mbar_wait(s_ready(j), (j / C::BUFS) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc::fence_after();
      const float* ex = extra + s * C::EXTRA;
      const uint32_t buf = lane_base + (j % C::BUFS) * (HP * C::BUF);
      // a warp without a row of the item only keeps the barriers going: its lanes of P reach no result
      if (32 * (warp & 3) < item.rows) {
        if constexpr (MODE == kForward) {
          ok = n >= BN ? forward_tile(std::false_type{}, j, n, ex, buf) : forward_tile(std::true_type{}, j, n, ex, buf);
          if (!ok) break;
        } else {
          if constexpr (MODE == kKeySide && BIAS) {
            if (sub != last_sub) {
              fold();
              last_sub = sub;
              set_slopes(sub);
            }
          }
          if (((j / C::GROUPS) & 3) == 3) fold();
          if (n >= BN) backward_tile(std::false_type{}, j, n, ex, buf);
          else backward_tile(std::true_type{}, j, n, ex, buf);
        }
      }
      tc::wait_st();
      if constexpr (C::TOTALS > 0) {
        // the product of this tile starts the accumulators again: what they hold goes to the totals
        if (j > 0 && j % C::FLUSH == 0) {
          ok = __all_sync(0xffffffffu, tc::mbar_wait(empty((j - 1) % C::STAGES), ((j - 1) / C::STAGES) & 1));
          if (!ok) break;
          tc::fence_after();
          flush(j);
        }
      }
      tc::fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(p_ready(j));
    }
    if constexpr (MODE != kForward) fold();

    // ---- results
    if (ok && total > 0) {
      ok = tc::mbar_wait(empty((total - 1) % C::STAGES), ((total - 1) / C::STAGES) & 1);
      ok = __all_sync(0xffffffffu, ok);
    }
    // the groups' sums: every thread gets the other group's of its row, through the stages' memory
    if constexpr (C::GROUPS == 2) {
      float* shared = reinterpret_cast<float*>(tile_smem + (cols - tc::smem_addr(tile_smem)));
      if (!ok) s_abort = 1;
      asm volatile("bar.sync 1, 256;\n" ::: "memory");
      if (ok) {
#pragma unroll
        for (int k = 0; k < SUMS; ++k) shared[(group * SUMS + k) * kTileRows + r_tile] = sum[k];
      }
      asm volatile("bar.sync 1, 256;\n" ::: "memory");
      ok = ok && *static_cast<volatile int*>(&s_abort) == 0;  // a row needs both groups
      if (ok) {
        const float* other = shared + (1 - group) * SUMS * kTileRows + r_tile;
#pragma unroll
        for (int k = 0; k < SUMS; ++k) sum[k] += other[k * kTileRows];
      }
    }
    if (ok) {
      tc::fence_after();
      const bool split = item.slot >= 0;
#pragma unroll
      for (int h = 0; h < HP; ++h) {
        const int64_t at = row * heads + head0 + h;
        float* part =
            split ? a.part + ((int64_t(item.slot) * heads + head0 + h) * kTileRows + r_tile) * C::PART : nullptr;
          float f0 = 1.0f;
        bool none = total == 0;
        if constexpr (MODE == kForward) {
          none = none || (m[h] == -INFINITY && l[h] == 0.0f);
          f0 = split ? 1.0f : none ? 0.0f : 1.0f / l[h];
        } else if constexpr (MODE == kQuerySide) {
          f0 = split ? 1.0f : a.scale;
        }
        // query side: delta = delta0 + off; the sum of P is 1 up to the rounding of lse, which dividing by it takes out.
        // It is 0 for a row without a score above -inf, whose lse is +inf.
        float inv = 0.0f, off = 0.0f;
        if constexpr (MODE == kQuerySide) {
          inv = none || sum[9] == 0.0f ? 0.0f : 1.0f / sum[9];
          off = sum[0] * inv;
        }
#pragma unroll
        for (int op = 0; op < C::OPS; ++op) {
          const float f = MODE == kKeySide && op == 1 && !split ? a.scale : f0;
          T* dst = static_cast<T*>(op ? a.out1 : a.out0) + at * a.D;
          for (int d = 16 * group; d < acc_n; d += 16 * C::GROUPS) {
            float o[16];
            tc::ld16(lane_base + C::ACC + (h * C::NACC + op) * C::W + d, o);
            if constexpr (C::TOTALS > 0 || C::FIX) {
              float e[16];
              if constexpr (C::TOTALS_SMEM) {
#pragma unroll
                for (int k = 0; k < 16; ++k) e[k] = totals[(op * C::W + d + k) * kTileRows + r_tile];
              } else {
                tc::ld16(lane_base + C::ACC + (h * C::NACC + C::OPS + op) * C::W + d, e);
              }
              tc::wait_ld();
              const bool whole = C::TOTALS > 0 && total <= C::FLUSH;  // nothing went into the total
              if (whole) {
#pragma unroll
                for (int k = 0; k < 16; ++k) e[k] = 0.0f;
              }
              const float fe = !C::FIX ? 1.0f : split ? 0.0f : -off;
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                if constexpr (C::FIX) {
                  if (split && valid) part[DP + 16 + d + k] = none ? 0.0f : e[k];
                }
                o[k] = fmaf(fe, e[k], o[k]);
              }
            } else {
              tc::wait_ld();
            }
            if (valid) {
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = none ? 0.0f : o[k] * f;
              if (split) {
#pragma unroll
                for (int k = 0; k < 16; k += 4)
                  *reinterpret_cast<float4*>(part + op * DP + d_first + d + k) =
                      make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
              } else {
                store_row16<T>(dst, o, d_first + d, a.D, a.vec != 0);
              }
            }
          }
        }
        if (valid && group == 0) {
          if constexpr (MODE == kForward) {
            if (split) {
              part[DP] = none ? -INFINITY : m[h];
              part[DP + 1] = l[h];
            } else {
              a.lse[at] = none ? INFINITY : m[h] + log2f(l[h]);
            }
          } else if constexpr (MODE == kQuerySide) {
            if (split) {
#pragma unroll
              for (int k = 0; k < 10; ++k) part[DP + k] = sum[k];
              part[DP + 10] = delta0;
            } else {
              a.delta[at] = delta0 + off;
              if constexpr (BIAS) {
                a.slope_part[at] = -inv * (sum[1] - off * sum[2]);
#pragma unroll
                for (int k = 0; k < 3; ++k) a.place_part[at * 3 + k] = -slope[0] * inv * (sum[3 + k] - off * sum[6 + k]);
              }
            }
          } else if (BIAS && half == 0) {
#pragma unroll
            for (int k = 0; k < 3; ++k) {
              if (split) part[2 * DP + k] = sum[k];
              else a.place_part[at * 3 + k] = -sum[k];
            }
          }
        }
      }
    } else {
      s_abort = 1;
      // a wait ran out: NaN, so that what is missing cannot pass as a result where no status is read
      if (valid) {
        const float nan = __int_as_float(0x7fffffff);
#pragma unroll 1
        for (int h = 0; h < HP; ++h) {
          const int64_t at = row * heads + head0 + h;
          if (item.slot >= 0) {
            float* part = a.part + ((int64_t(item.slot) * heads + head0 + h) * kTileRows + r_tile) * C::PART;
#pragma unroll 1
            for (int k = group; k < C::PART; k += C::GROUPS) part[k] = nan;
            continue;
          }
#pragma unroll 1
          for (int d = d_first + group; d < d_first + d_count; d += C::GROUPS) {
            static_cast<T*>(a.out0)[at * a.D + d] = from_float<T>(nan);
            if constexpr (C::OPS == 2) static_cast<T*>(a.out1)[at * a.D + d] = from_float<T>(nan);
          }
          if constexpr (MODE == kForward) a.lse[at] = nan;
          if constexpr (MODE == kQuerySide) a.delta[at] = nan;
          if constexpr (MODE == kQuerySide && BIAS) a.slope_part[at] = nan;
          if constexpr (MODE != kForward && BIAS)
            for (int k = 0; k < 3; ++k) a.place_part[at * 3 + k] = nan;
        }
      }
    }
  }
  tc::fence_before();
  __syncthreads();
  if (warp == C::MMA_WARP) {
    tc::fence_after();
    tc::dealloc(tmem, C::COLUMNS);
  }
  if (tid == 0 && s_abort && a.status) atomicOr(a.status, Y3B_STATUS_TIMEOUT);
}

// Encodes the tensor map of a column operand; its strides are positive multiples of 16 bytes.
int encode_columns(CUtensorMap* map, const AttOperand& o, int D, int heads, int64_t rows, int pieces, int box_rows);

template <int MODE, int DP, int NP, int HP, bool BIAS>
int launch_attention_tile(AttTileArgs& a, int64_t items, cudaStream_t s) {
  using C = AttCfg<MODE, DP, NP, HP>;
  int rc = encode_columns(&a.cols[0], MODE == kKeySide ? a.q : a.k, a.D, MODE == kKeySide ? a.H : a.Hk,
                          MODE == kKeySide ? a.nq : a.nk, NP, C::BN);
  if (!rc)
    rc = encode_columns(&a.cols[1], MODE == kKeySide ? a.g : a.v, a.D, MODE == kKeySide ? a.H : a.Hk,
                        MODE == kKeySide ? a.nq : a.nk, NP, C::BN);
  if (rc) return rc;
  const auto kernel = attention_tile_kernel<MODE, DP, NP, HP, BIAS>;
  Y3B_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
  const int64_t grid = items * ((MODE == kKeySide ? a.Hk : a.H) / HP) * C::HALVES;
  if (grid > INT32_MAX) return fail(Y3B_ERR_UNSUPPORTED, "structure_attention: %lld tiles", (long long)grid);
  kernel<<<unsigned(grid), C::THREADS, C::SMEM, s>>>(a);
  Y3B_LAUNCH_CHECK();
  return Y3B_OK;
}

template <int MODE>
int dispatch_attention_tile(int pieces, AttTileArgs& a, int64_t items, cudaStream_t s) {
  if (items == 0) return Y3B_OK;
  const bool bias = a.slopes != nullptr, wide = a.D > 64;
#define Y3B_TILE(DP, NP)                                                       \
  return bias ? launch_attention_tile<MODE, DP, NP, 1, true>(a, items, s)      \
              : launch_attention_tile<MODE, DP, NP, 1, false>(a, items, s)
  if (pieces == 1) {
    if constexpr (MODE == kForward) {
      if (bias && !wide && a.H % 2 == 0) return launch_attention_tile<MODE, 64, 1, 2, true>(a, items, s);
    }
    if (wide) { Y3B_TILE(128, 1); }
    Y3B_TILE(64, 1);
  }
  if (wide) { Y3B_TILE(128, 3); }
  Y3B_TILE(64, 3);
#undef Y3B_TILE
}

// One mode a translation unit.
int attention_forward_tiles(int pieces, AttTileArgs& a, int64_t items, cudaStream_t s);
int attention_query_tiles(int pieces, AttTileArgs& a, int64_t items, cudaStream_t s);
int attention_key_tiles(int pieces, AttTileArgs& a, int64_t items, cudaStream_t s);

}  // namespace y3b

