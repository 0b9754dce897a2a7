// Matrix products grouped by expert in 16-bit floats, with their gradients, and
// in 8-bit integers with a scale for each row and column, grouped or dense.
//
// The slots are grouped by moe_align_block_size, whose blocks the kernels walk;
// rows are gathered from and written to their slots' places, so nothing is
// permuted in memory:
//   product     y[s, n]  = sum_k x[row(s), k] w[e(s), n, k]
//   by rows     dxs[s, k] = sum_n dy[s, n] w[e(s), n, k]
//   by weights  dw[e, n, k] = sum over the slots s of e of dy[s, n] x[row(s), k]
//   int8        y[s, n]  = (sum_k a[row, k] b[e, n, k]) * as[row] * bs[e, n] (+ bias[n]) (* w[s])
// Sums are held in fp32 (int8: exactly, in 32-bit integers) and rounded once.
#include "grouped_launch.hpp"

namespace moe {

// ---- any sizes, strides and alignment --------------------------------------
// 64 x 64 tiles in four waves of 32 x 32; a step of 64 bytes of the contraction
// is staged through registers one element at a time.  Bound by those loads; it
// serves the widths whose rows are not 16-byte runs.
constexpr int kAnyTile = 64;
constexpr int kAnyRow = 64 + 16;  // bytes of an LDS row, padded: 16 rows start in distinct bank groups

template <class OP, bool FP16, bool WEIGHTS>
__global__ __launch_bounds__(256) void any_mm_kernel(MmArgs g) {
  constexpr int EB = OP::BYTES;
  constexpr int KE = 64 / EB;  // elements of a step
  __shared__ __attribute__((aligned(16))) uint8_t sA[kAnyTile * kAnyRow], sB[kAnyTile * kAnyRow];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t jt = (int64_t)blockIdx.x % g.n_jt, it = (int64_t)blockIdx.x / g.n_jt;
  const int64_t j0 = jt * kAnyTile;
  int64_t pos0, i0 = 0, length;
  int rows, e = 0;
  if constexpr (WEIGHTS) {
    const int64_t nt = (g.Cn + kAnyTile - 1) / kAnyTile;
    e = (int)(it / nt);
    i0 = it % nt * kAnyTile;
    rows = (int)(g.Cn - i0 < kAnyTile ? g.Cn - i0 : kAnyTile);
    const Run r = run_of(g, e);
    pos0 = r.pos0;
    length = r.count;
  } else {
    const int per = (g.bm + kAnyTile - 1) / kAnyTile;  // tiles of a block
    const int64_t b = it / per;
    if (b >= live_blocks(g)) return;
    const int sub = (int)(it % per) * kAnyTile;
    pos0 = b * g.bm + sub;
    rows = g.bm - sub < kAnyTile ? g.bm - sub : kAnyTile;
    length = g.Cn;
    if (g.eids) e = g.eids[b];
    else if (pos0 + rows > g.S) rows = (int)(g.S - pos0);
  }
  const bool none = e < 0 || e >= g.E;
  auto slot_at = [&](int64_t pos) -> int64_t { return g.sorted ? (int64_t)(uint32_t)g.sorted[pos] : pos; };

  // This thread's part of each operand's tile: 64 bytes a row by 64 rows, 16
  // bytes a thread, along whichever direction is contiguous in memory.
  const bool b_by_j = WEIGHTS || g.sbc != 1;
  const int run_r = tid >> 2, run_c = (tid & 3) * (KE / 4);  // contiguous along the contraction
  const int col_r = tid & 63, col_c = (tid >> 6) * (KE / 4); // contiguous along the rows
  const uint8_t* a_row = nullptr;
  const uint8_t* b_row = nullptr;
  if constexpr (!WEIGHTS) {
    if (run_r < rows) {
      const int64_t slot = slot_at(pos0 + run_r);
      if (slot < g.S) a_row = g.A + (g.a_by_pos ? pos0 + run_r : (int64_t)slot_row(g, (uint32_t)slot)) * g.lda * EB;
    }
    const int64_t j = j0 + (b_by_j ? col_r : run_r);
    if (j < g.J && !none) b_row = g.B + ((int64_t)e * g.b_es + j * g.sbj) * EB;
  }
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32, fr = lane & 15, kseg = lane >> 4;
  typename OP::Acc acc[2][2] = {};
  typedef typename std::conditional<EB == 2, uint16_t, uint8_t>::type E;
  if (none) length = 0;
  for (int64_t c0 = 0; c0 < length; c0 += KE) {
    E a[KE / 4], b[KE / 4];
#pragma unroll
    for (int q = 0; q < KE / 4; ++q) {
      if constexpr (WEIGHTS) {
        const int64_t c = c0 + col_c + q;
        const int64_t slot = c < length ? slot_at(pos0 + c) : g.S;
        const bool on = slot < g.S;
        a[q] = on && col_r < rows ? reinterpret_cast<const E*>(g.A)[slot * g.lda + i0 + col_r] : (E)0;
        b[q] = on && j0 + col_r < g.J ? reinterpret_cast<const E*>(g.B)[(int64_t)slot_row(g, (uint32_t)slot) * g.sbc + j0 + col_r] : (E)0;
      } else {
        const int64_t ca = c0 + run_c + q, cb = c0 + (b_by_j ? col_c : run_c) + q;
        a[q] = a_row && ca < length ? reinterpret_cast<const E*>(a_row)[ca] : (E)0;
        b[q] = b_row && cb < length ? reinterpret_cast<const E*>(b_row)[cb * g.sbc] : (E)0;
      }
    }
    __syncthreads();  // the last step's fragments are read
#pragma unroll
    for (int q = 0; q < KE / 4; ++q) {
      const int ar = WEIGHTS ? col_r : run_r, ac = WEIGHTS ? col_c : run_c;
      const int br = b_by_j ? col_r : run_r, bc = b_by_j ? col_c : run_c;
      reinterpret_cast<E*>(sA + ar * kAnyRow)[ac + q] = a[q];
      reinterpret_cast<E*>(sB + br * kAnyRow)[bc + q] = b[q];
    }
    __syncthreads();
    v4i af[2], bf[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      af[s] = *reinterpret_cast<const v4i*>(sA + (wm + s * 16 + fr) * kAnyRow + kseg * 16);
      bf[s] = *reinterpret_cast<const v4i*>(sB + (wn + s * 16 + fr) * kAnyRow + kseg * 16);
    }
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int c = 0; c < 2; ++c) acc[r][c] = OP::mfma(bf[c], af[r], acc[r][c]);
  }
  // a lane holds four consecutive columns of one row
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = wm + r * 16 + fr;
    if (row >= rows) continue;
    int64_t orow, arow = 0;
    float w = 1.0f, sa = 1.0f;
    if constexpr (WEIGHTS) {
      orow = (int64_t)e * g.Cn + i0 + row;
    } else {
      orow = slot_at(pos0 + row);
      if (orow >= g.S) continue;
      arow = g.a_by_pos ? pos0 + row : (int64_t)slot_row(g, (uint32_t)orow);
      if (g.topk_w) w = g.topk_w[orow];
      if constexpr (EB == 1) sa = g.As[arow];
    }
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int64_t j = j0 + wn + c * 16 + 4 * kseg + v;
        if (j >= g.J) continue;
        float f = 0.0f;
        if constexpr (EB == 1) {
          if (!none)
            f = int8_out(acc[r][c][v], sa, g.Bs[(int64_t)e * g.J + j], g.bias, g.bias ? from16<FP16>(g.bias[j]) : 0.0f,
                         g.topk_w, w);
        } else {
          f = acc[r][c][v];
        }
        if (g.out32) reinterpret_cast<float*>(g.C)[orow * g.ldc + j] = f;
        else reinterpret_cast<uint16_t*>(g.C)[orow * g.ldc + j] = (uint16_t)pack2<FP16>(f, 0.0f);
      }
  }
}

template <class OP, bool FP16, bool WEIGHTS>
static int launch_any(MmArgs g, hipStream_t st) {
  g.n_jt = (g.J + kAnyTile - 1) / kAnyTile;
  const int64_t rows = WEIGHTS ? g.E * ((g.Cn + kAnyTile - 1) / kAnyTile)
                               : g.n_blocks * ((g.bm + kAnyTile - 1) / kAnyTile);
  const int64_t grid = rows * g.n_jt;
  if (!fits_launch(grid, 256)) return kErrBadShape;
  hipLaunchKernelGGL((any_mm_kernel<OP, FP16, WEIGHTS>), dim3((unsigned)grid), dim3(256), 0, st, g);
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

// What every grouped entry checks of the slots.
static int slots_ok(const int32_t* sorted, const int32_t* eids, const int32_t* ntpp, int64_t S, int32_t E, int32_t BM,
                    int64_t max_padded) {
  if (S < 0 || max_padded < 0 || S > 0x7FFFFFFE || max_padded > 0x7FFFFFFF) return kErrBadShape;
  if (E <= 0) return kErrBadExperts;
  if (!block_m_ok(BM)) return kErrBadBlockSize;
  if (max_padded > 0 && (!sorted || !eids || !ntpp)) return kErrNullPointer;
  return kOk;
}

}  // namespace moe

using namespace moe;

extern "C" int moe_grouped_mm(const void* x, int64_t ldx, const void* w, const int32_t* sorted_ids,
                              const int32_t* expert_ids, const int32_t* ntpp, const int32_t* table, int64_t S,
                              int32_t top_k, int64_t N, int64_t K, int32_t E, int32_t BM, int64_t max_padded,
                              int32_t dtype, void* y, void* stream) {
  const int rc = slots_ok(sorted_ids, expert_ids, ntpp, S, E, BM, max_padded);
  if (rc != kOk) return rc;
  if (N < 0 || K < 0 || ldx < K || (dtype != kBf16 && dtype != kFp16)) return kErrBadShape;
  if (top_k <= 0) return kErrBadTopK;
  if (S == 0 || N == 0 || max_padded == 0) return kOk;
  if (!y || (K > 0 && (!x || !w))) return kErrNullPointer;
  if (!aligned(x, 2) || !aligned(w, 2) || !aligned(y, 2)) return kErrBadShape;
  MmArgs g{};
  g.A = (const uint8_t*)x;
  g.B = (const uint8_t*)w;
  g.C = (uint8_t*)y;
  g.sorted = sorted_ids;
  g.eids = expert_ids;
  g.ntpp = ntpp;
  g.table = table;
  g.S = S;
  g.J = N;
  g.Cn = K;
  g.lda = ldx;
  g.sbj = K;
  g.sbc = 1;
  g.b_es = N * K;
  g.ldc = N;
  g.n_blocks = max_padded / BM;
  g.bm = BM;
  set_top_k(g, top_k);
  g.E = E;
  hipStream_t st = (hipStream_t)stream;
  if (K > 0 && K % 8 == 0 && chunks(x, ldx, 2) && chunks(w, K, 2) && chunks(y, N, 2))
    return tile_product(g, dtype, st);
  return dtype == kFp16 ? launch_any<Fp16, true, false>(g, st) : launch_any<Bf16, false, false>(g, st);
}

extern "C" int moe_grouped_mm_dgrad(const void* dy, const void* w, const int32_t* sorted_ids,
                                    const int32_t* expert_ids, const int32_t* ntpp, const int32_t* table, int64_t S,
                                    int64_t N, int64_t K, int32_t E, int32_t BM, int64_t max_padded, int32_t dtype,
                                    int32_t rows_f32, void* dx, void* stream) {
  const int rc = slots_ok(sorted_ids, expert_ids, ntpp, S, E, BM, max_padded);
  if (rc != kOk) return rc;
  if (N < 0 || K < 0 || (dtype != kBf16 && dtype != kFp16)) return kErrBadShape;
  if (S == 0 || K == 0 || max_padded == 0) return kOk;
  if (!dx || (N > 0 && (!dy || !w))) return kErrNullPointer;
  if (!aligned(dy, 2) || !aligned(w, 2) || !aligned(dx, rows_f32 ? 4 : 2)) return kErrBadShape;
  MmArgs g{};
  g.A = (const uint8_t*)dy;
  g.B = (const uint8_t*)w;
  g.C = (uint8_t*)dx;
  g.sorted = sorted_ids;
  g.eids = expert_ids;
  g.ntpp = ntpp;
  g.table = table;
  g.S = S;
  g.J = K;
  g.Cn = N;
  g.lda = N;
  g.sbj = 1;
  g.sbc = K;
  g.b_es = N * K;
  g.ldc = K;
  g.n_blocks = max_padded / BM;
  g.bm = BM;
  set_top_k(g, 1);
  g.out32 = rows_f32 ? 1 : 0;
  g.E = E;
  hipStream_t st = (hipStream_t)stream;
  if (N > 0 && chunks(dy, N, 2) && chunks(w, K, 2) && chunks(dx, K, 2))
    return tile_dgrad(g, dtype, st);
  return dtype == kFp16 ? launch_any<Fp16, true, false>(g, st) : launch_any<Bf16, false, false>(g, st);
}

extern "C" int moe_grouped_mm_wgrad(const void* dy, const void* x, int64_t ldx, const int32_t* sorted_ids,
                                    const int32_t* expert_ids, const int32_t* ntpp, const int32_t* table, int64_t S,
                                    int32_t top_k, int64_t N, int64_t K, int32_t E, int32_t BM, int64_t max_padded,
                                    int32_t dtype, void* dw, void* stream) {
  const int rc = slots_ok(sorted_ids, expert_ids, ntpp, S, E, BM, max_padded);
  if (rc != kOk) return rc;
  if (N < 0 || K < 0 || ldx < K || (dtype != kBf16 && dtype != kFp16)) return kErrBadShape;
  if (top_k <= 0) return kErrBadTopK;
  if (N == 0 || K == 0) return kOk;
  if (!dw || (S > 0 && (!dy || !x))) return kErrNullPointer;
  if (!aligned(dy, 2) || !aligned(x, 2) || !aligned(dw, 2)) return kErrBadShape;
  MmArgs g{};
  g.A = (const uint8_t*)dy;
  g.B = (const uint8_t*)x;
  g.C = (uint8_t*)dw;
  g.sorted = sorted_ids;
  g.eids = expert_ids;
  g.ntpp = max_padded > 0 ? ntpp : nullptr;  // without positions: no blocks
  g.table = max_padded > 0 ? table : nullptr;
  g.S = S;
  g.J = K;
  g.Cn = N;
  g.lda = N;
  g.sbc = ldx;
  g.ldc = K;
  g.n_blocks = max_padded / BM;
  g.bm = BM;
  set_top_k(g, top_k);
  g.E = E;
  hipStream_t st = (hipStream_t)stream;
  if (S > 0 && chunks(dy, N, 2) && chunks(x, ldx, 2) && chunks(dw, K, 2) && N < (1 << 30) && ldx < (1 << 30))
    return launch_weights<kWgrad>(g, dtype, st);
  return dtype == kFp16 ? launch_any<Fp16, true, true>(g, st) : launch_any<Bf16, false, true>(g, st);
}

// For rows of whole chunks that the caller has checked (gated.hip).
int moe::tile_product(const MmArgs& g, int32_t dtype, hipStream_t st) {
  return dtype == kFp16 ? launch_rows<Fp16, true, kProduct>(g, st) : launch_rows<Bf16, false, kProduct>(g, st);
}
int moe::tile_dgrad(const MmArgs& g, int32_t dtype, hipStream_t st) {
  return dtype == kFp16 ? launch_rows<Fp16, true, kDgrad>(g, st) : launch_rows<Bf16, false, kDgrad>(g, st);
}
int moe::tile_wgrad(const MmArgs& g, int32_t dtype, hipStream_t st) { return launch_weights<kWgrad>(g, dtype, st); }

// a [rows, K] and b [E, N, K] int8 with their scales, y in the output type.
static int int8_product(MmArgs g, int32_t dtype, hipStream_t st) {
  if (g.Cn > 0 && g.Cn % 16 == 0 && g.J % 8 == 0 && chunks(g.A, g.lda, 1) && chunks(g.B, g.sbj, 1) && chunks(g.C, g.ldc, 2))
    return dtype == kFp16 ? launch_rows<Int8, true, kProduct>(g, st) : launch_rows<Int8, false, kProduct>(g, st);
  return dtype == kFp16 ? launch_any<Int8, true, false>(g, st) : launch_any<Int8, false, false>(g, st);
}

constexpr int64_t kInt8MaxK = (1 << 17) - 1;

extern "C" int moe_grouped_gemm_int8(const void* a, const float* a_scale, const void* b, const float* b_scale,
                                     const int32_t* sorted_ids, const int32_t* expert_ids, const int32_t* ntpp,
                                     const float* topk_weights, int64_t S, int32_t top_k, int32_t a_by_pos, int64_t N,
                                     int64_t K, int32_t E, int32_t BM, int64_t max_padded, int32_t dtype, void* y,
                                     void* stream) {
  const int rc = slots_ok(sorted_ids, expert_ids, ntpp, S, E, BM, max_padded);
  if (rc != kOk) return rc;
  if (N < 0 || K < 0 || K > kInt8MaxK || (dtype != kBf16 && dtype != kFp16)) return kErrBadShape;
  if (top_k <= 0) return kErrBadTopK;
  if (S == 0 || N == 0 || max_padded == 0) return kOk;
  if (!y || !a_scale || !b_scale || (K > 0 && (!a || !b))) return kErrNullPointer;
  if (!aligned(y, 2) || !aligned(a_scale, 4) || !aligned(b_scale, 4) || !aligned(topk_weights, 4)) return kErrBadShape;
  MmArgs g{};
  g.A = (const uint8_t*)a;
  g.B = (const uint8_t*)b;
  g.C = (uint8_t*)y;
  g.sorted = sorted_ids;
  g.eids = expert_ids;
  g.ntpp = ntpp;
  g.As = a_scale;
  g.Bs = b_scale;
  g.topk_w = topk_weights;
  g.S = S;
  g.J = N;
  g.Cn = K;
  g.lda = K;
  g.sbj = K;
  g.sbc = 1;
  g.b_es = N * K;
  g.ldc = N;
  g.n_blocks = max_padded / BM;
  g.bm = BM;
  set_top_k(g, top_k);
  g.a_by_pos = a_by_pos ? 1 : 0;
  g.E = E;
  return int8_product(g, dtype, (hipStream_t)stream);
}

extern "C" int moe_int8_scaled_mm(const void* a, int64_t lda, const float* a_scale, const void* b, int64_t ldb,
                                  const float* b_scale, const void* bias, int64_t M, int64_t N, int64_t K,
                                  int32_t dtype, void* y, int64_t ldy, void* stream) {
  if (M < 0 || N < 0 || K < 0 || K > kInt8MaxK || lda < K || ldb < K || ldy < N || M > 0x7FFFFF00) return kErrBadShape;
  if (dtype != kBf16 && dtype != kFp16) return kErrBadShape;
  if (M == 0 || N == 0) return kOk;
  if (!y || !a_scale || !b_scale || (K > 0 && (!a || !b))) return kErrNullPointer;
  if (!aligned(y, 2) || !aligned(bias, 2) || !aligned(a_scale, 4) || !aligned(b_scale, 4)) return kErrBadShape;
  MmArgs g{};
  g.Cn = K;
  g.lda = lda;
  g.sbj = ldb;
  g.sbc = 1;
  g.ldc = ldy;
  g.bm = dense_rows(M, N);
  set_top_k(g, 1);
  g.E = 1;
  // In parts that one launch has the threads for, up to 512 of them for 16 columns of a
  // block of up to 32 rows or 64 x 64 of another: up to 2^26 columns, and whole blocks.
  const int64_t cols = N < (1 << 26) ? N : 1 << 26;
  const int64_t tiles = g.bm <= 32 ? (cols + 15) / 16 : g.bm / 64 * ((cols + 63) / 64);
  const int64_t rows = (0xFFFFFFFFll / 512 - 8) / tiles * g.bm;
  for (int64_t m = 0; m < M; m += rows) {
    for (int64_t n = 0; n < N; n += cols) {
      g.A = (const uint8_t*)a + m * lda;
      g.As = a_scale + m;
      g.B = (const uint8_t*)b + n * ldb;
      g.Bs = b_scale + n;
      g.bias = bias ? (const uint16_t*)bias + n : nullptr;
      g.C = (uint8_t*)y + 2 * (m * ldy + n);
      g.S = M - m < rows ? M - m : rows;
      g.J = N - n < cols ? N - n : cols;
      g.n_blocks = (g.S + g.bm - 1) / g.bm;
      const int rc = int8_product(g, dtype, (hipStream_t)stream);
      if (rc != kOk) return rc;
    }
  }
  return kOk;
}
