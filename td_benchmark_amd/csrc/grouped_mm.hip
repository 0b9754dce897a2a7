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
#include "grouped_tile.hpp"

namespace moe {

// A launch has fewer than 2^32 threads.
static bool fits_launch(int64_t workgroups, int threads) { return workgroups <= 0xFFFFFFFFll / threads; }

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

// ---- whole, aligned chunks ---------------------------------------------------
template <class OP, bool FP16, int FORM, class T>
static int launch_tile(MmArgs g, hipStream_t st) {
  g.n_jt = (g.J + T::TN - 1) / T::TN;
  int64_t tiles = (FORM == kWgrad ? g.E * ((g.Cn + T::TM - 1) / T::TM) : g.n_blocks) * g.n_jt, more = 0;
  if (FORM != kWgrad) {
    // The short last tiles apart from the whole ones: even rounds, but an expert's
    // weights are read once more for its short tile, about 250 / rows of its time.
    // It pays where the launch has few rounds and the runs are long (8 experts of
    // 1024 rows, 28672 to 4096 columns, 2.3 rounds: 2200 us by blocks, 1802 so; to
    // 28672 columns, 16 rounds: 1800 and 1890; 64 of 512 rows 465 and 510; 128 of 256
    // 311 and 376).
    const int64_t used = g.S < g.E ? g.S : g.E;
    if (T::TM != 256 || g.S < 768 * (int64_t)g.E || g.S / 256 * g.n_jt > 1024) g.table = nullptr;
    if (g.table) {  // whole tiles: at most S / 256 and one more an expert; then the short ones
      tiles = (g.S / 256 + used + 1) * g.n_jt;
      if (T::TN == 256) {
        g.short_parts = used * g.n_jt <= 256 && g.Cn * OP::BYTES >= 64 * 128 ? 4 : 1;
        more = used * g.n_jt * g.short_parts;
      }
    }
  }
  const int64_t deal = FORM == kWgrad ? 8 * kWgradChunk : 8;
  g.shorts = (tiles + deal - 1) / deal * deal;
  const int64_t grid = g.shorts + more;
  if (!fits_launch(grid, T::THREADS)) return kErrBadShape;
  static const hipError_t attr =
      hipFuncSetAttribute((const void*)tile_mm_kernel<OP, FP16, FORM, T>, hipFuncAttributeMaxDynamicSharedMemorySize,
                          T::LDS_BYTES);
  if (attr != hipSuccess) return kErrLaunch;
  hipLaunchKernelGGL((tile_mm_kernel<OP, FP16, FORM, T>), dim3((unsigned)grid), dim3(T::THREADS), T::LDS_BYTES, st, g);
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

// ---- few rows: the weights' stream, split along the contraction ---------------
// Sixteen columns of one block of up to 16 RT rows a workgroup.  Its waves take the
// contraction's 128-byte chunks in turn, operands straight to registers (lane fr,
// kseg: 32 bytes of row fr), U chunks' loads in flight each, and their sums are
// added in wave order through LDS: several times the workgroups of the narrowest
// staged tile, where those are too few to draw on the memory.  A CU draws 50-60
// GB/s of data that is in no cache.
constexpr int kFewWaves = 8;

template <class OP, bool FP16, int RT>
__global__ __launch_bounds__(64 * kFewWaves) void few_mm_kernel(MmArgs g) {
  constexpr int EB = OP::BYTES, TM = 16 * RT, U = 4;
  __shared__ typename OP::Acc part[kFewWaves][RT][64];
  __shared__ int32_t smSlot[TM];
  const int tid = threadIdx.x, lane = tid & 63, fr = lane & 15, kseg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int64_t b, j;
  if (!rows_tile<false>(g, b, j)) return;
  const int64_t j0 = j * 16, pos0 = b * g.bm;
  const int e = g.eids ? g.eids[b] : 0;
  bool valid = false;
  if (tid < TM) {
    const uint32_t slot = g.sorted ? (uint32_t)g.sorted[pos0 + tid] : (uint32_t)(pos0 + tid);
    valid = slot < g.S;
    smSlot[tid] = valid ? (int)slot : -1;
  }
  const int nvalid = end_of<TM>(valid);  // rows up to the last slot
  if (nvalid == 0) return;
  const bool none = e < 0 || e >= g.E;
  const uint8_t* a_row[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int slot = smSlot[16 * r + fr];
    const int64_t ar = slot < 0 ? 0 : g.a_by_pos ? pos0 + 16 * r + fr : (int64_t)slot_row(g, (uint32_t)slot);
    a_row[r] = g.A + ar * g.lda * EB + kseg * 32;
  }
  const int64_t jb = j0 + fr < g.J ? j0 + fr : g.J - 1;
  const uint8_t* b_row = g.B + ((int64_t)e * g.b_es + jb * g.sbj) * EB + kseg * 32;
  typename OP::Acc acc[RT] = {};
  const int64_t bytes = g.Cn * EB;
  const int chunks = none ? 0 : (int)((bytes + 127) / 128);
  auto load = [&](const uint8_t* p, int64_t at) -> v4i {  // 16 bytes at `at` + kseg * 32 of a row, zeros past its end
    return at + kseg * 32 < bytes ? *reinterpret_cast<const v4i*>(p + at) : (v4i){0, 0, 0, 0};
  };
  const bool second = nvalid > 16;  // whether the second 16 rows hold slots
  for (int c0 = wave; c0 < chunks; c0 += kFewWaves * U) {
    v4i bf[U][2], af[U][RT][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = (int64_t)(c0 + u * kFewWaves) * 128;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        bf[u][h] = load(b_row, at + 16 * h);
#pragma unroll
        for (int r = 0; r < RT; ++r) af[u][r][h] = r == 0 || second ? load(a_row[r], at + 16 * h) : (v4i){0, 0, 0, 0};
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[r] = OP::mfma(bf[u][h], af[u][r][h], acc[r]);
  }
#pragma unroll
  for (int r = 0; r < RT; ++r) part[wave][r][lane] = acc[r];
  __syncthreads();
  // a lane's four columns of one row again, 64 lanes a 16 x 16 part
  if (tid < RT * 64) {
    const int l = tid & 63, r = tid / 64, row = 16 * r + (l & 15);
    const int64_t jj = j0 + 4 * (l >> 4);
    if (row >= nvalid || jj >= g.J) return;  // J is a multiple of 8
    typename OP::Acc sum = part[0][r][l];
#pragma unroll
    for (int w = 1; w < kFewWaves; ++w) sum = sum + part[w][r][l];
    const int slot = smSlot[row];
    if (slot < 0) return;  // padding before a slot
    float f[4];
    if constexpr (EB == 1) {
      const float sa = none ? 0.0f : g.As[g.a_by_pos ? pos0 + row : (int64_t)slot_row(g, (uint32_t)slot)];
      const float w = g.topk_w ? g.topk_w[slot] : 1.0f;
#pragma unroll
      for (int v = 0; v < 4; ++v)
        f[v] = none ? 0.0f
                    : int8_out(sum[v], sa, g.Bs[(int64_t)e * g.J + jj + v], g.bias,
                               g.bias ? from16<FP16>(g.bias[jj + v]) : 0.0f, g.topk_w, w);
    } else {
#pragma unroll
      for (int v = 0; v < 4; ++v) f[v] = sum[v];
    }
    const v2u pk = {pack2<FP16>(f[0], f[1]), pack2<FP16>(f[2], f[3])};
    *reinterpret_cast<v2u*>(g.C + ((int64_t)slot * g.ldc + jj) * 2) = pk;
  }
}

template <class OP, bool FP16, int RT>
static int launch_few(MmArgs g, hipStream_t st) {
  g.n_jt = (g.J + 15) / 16;
  const int64_t grid = (g.n_blocks * g.n_jt + 7) / 8 * 8;
  if (!fits_launch(grid, 64 * kFewWaves)) return kErrBadShape;
  hipLaunchKernelGGL((few_mm_kernel<OP, FP16, RT>), dim3((unsigned)grid), dim3(64 * kFewWaves), 0, st, g);
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

// The rows form by the align block's rows.  The 256 columns of a wide tile cost
// the fewest loads, narrower ones give more tiles where there are few: `rounds`
// weighs the rounds that a width's tiles take on 256 CUs with what one of them
// costs (a tile of 128 columns about 0.65 and of 64 about 0.5 of one of 256, which
// measured 118 / 74 / 68 us at 8 experts of 128 rows, 4096 x 2048).  Up to 32 rows
// the product only streams its weights, which 64 columns and two workgroups a CU
// with deep rings do best at every count (4 rows an expert of 128: 189 us against
// 197; one token: 24 against 37); its gradient by rows reads them transposed and
// stays with wide tiles where they fill the chip (183 against 187, 9 rows of 8
// experts 221 against 241).
static double rounds(double blocks, int64_t J, int TN, double cost) {
  const double r = blocks * (double)((J + TN - 1) / TN) / 256.0;
  return cost * (r < 1.0 ? 1.0 : (double)(int64_t)(r + 0.999));
}

// The blocks that hold slots, as far as the host knows: near one an expert where
// they are short, and half a block over where they are long.
static double live_blocks_guess(const MmArgs& g) {
  if (!g.eids) return (double)g.n_blocks;
  const double used = g.S < g.E ? (double)g.S : (double)g.E;
  const double b = 2.0 * g.S <= used * g.bm ? used : (double)g.S / g.bm + 0.5 * used;
  return b < (double)g.n_blocks ? b : (double)g.n_blocks;
}

template <class OP, bool FP16, int FORM>
static int launch_rows(const MmArgs& g, hipStream_t st) {
  const double blocks = live_blocks_guess(g);
  const double wide = rounds(blocks, g.J, 256, 1.0), half = rounds(blocks, g.J, 128, 0.65),
               slim = rounds(blocks, g.J, 64, 0.5);
  // Few rows on long rows of weights: few tiles, or one or two slots a block (more
  // rows make it draw as much of A as of the weights).  int8, one row, 7168 x 4096:
  // 16.3 us, staged 24.5; 16 tokens on 128 experts 126 and 148; 9 slots a block of
  // 14336 272 and 226; rows of 768 bytes 123 and 79.
  if constexpr (FORM == kProduct) {
    if (g.bm <= 32 && g.Cn * OP::BYTES >= 2048 && (blocks * ((g.J + 63) / 64) <= 128.0 || g.S <= 2.0 * blocks))
      return g.bm == 16 ? launch_few<OP, FP16, 1>(g, st) : launch_few<OP, FP16, 2>(g, st);
  }
  if (g.bm <= 32) {
    const bool stream = FORM == kProduct || wide <= 1.0;
    if (g.bm == 16)
      return stream ? launch_tile<OP, FP16, FORM, MmTile<16, 64, 2, 1, 4, 2>>(g, st)
                    : launch_tile<OP, FP16, FORM, MmTile<16, 256, 8, 1, 3, 1>>(g, st);
    return stream ? launch_tile<OP, FP16, FORM, MmTile<32, 64, 4, 2, 6, 2>>(g, st)
                  : launch_tile<OP, FP16, FORM, MmTile<32, 256, 8, 1, 3, 1>>(g, st);
  }
  if (g.bm == 64) {
    if (FORM == kProduct || half < wide) {
      if (slim < half) return launch_tile<OP, FP16, FORM, MmTile<64, 64, 4, 2, 4, 2>>(g, st);
      return launch_tile<OP, FP16, FORM, MmTile<64, 128, 4, 1, 3, 2>>(g, st);
    }
    return launch_tile<OP, FP16, FORM, MmTile<64, 256, 8, 2, 3, 1>>(g, st);
  }
  if (g.bm == 128) {
    if (slim < half && slim < wide) return launch_tile<OP, FP16, FORM, MmTile<128, 64, 8, 4, 3, 2>>(g, st);
    if (half < wide) return launch_tile<OP, FP16, FORM, MmTile<128, 128, 8, 4, 4, 1>>(g, st);
    return launch_tile<OP, FP16, FORM, MmTile<128, 256, 8, 2, 3, 1>>(g, st);
  }
  if (slim < half && slim < wide) return launch_tile<OP, FP16, FORM, MmTile<256, 64, 8, 4, 3, 1>>(g, st);
  if (half < wide) return launch_tile<OP, FP16, FORM, MmTile<256, 128, 8, 4, 3, 1>>(g, st);
  return launch_tile<OP, FP16, FORM, MmTile<256, 256, 8, 4, 2, 1>>(g, st);
}

static bool aligned(const void* p, int n) { return ((uintptr_t)p & (n - 1)) == 0; }
// Whether rows at p with a stride of ld elements of `bytes` are whole 16-byte chunks.
static bool chunks(const void* p, int64_t ld, int bytes) { return aligned(p, 16) && ld * bytes % 16 == 0; }

constexpr int kBf16 = MOE_BF16, kFp16 = MOE_FP16;

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
    return dtype == kFp16 ? launch_rows<Fp16, true, kProduct>(g, st) : launch_rows<Bf16, false, kProduct>(g, st);
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
    return dtype == kFp16 ? launch_rows<Fp16, true, kDgrad>(g, st) : launch_rows<Bf16, false, kDgrad>(g, st);
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
  if (S > 0 && chunks(dy, N, 2) && chunks(x, ldx, 2) && chunks(dw, K, 2) &&
      N < (1 << 30) && ldx < (1 << 30)) {
    // Steps of 32 slots in rings of three or four: rows of a column-staged step are
    // whole lines at any length, so the finer ring costs nothing (256 slots an expert
    // of 128: 381 us, 403 with steps of 64 in a ring of two; 1024 of 8 even).  The rows
    // forms lose with it, whose row-staged lines it reads in halves.
    //
    // Two workgroups a CU with tiles of 128 rows: one writes its tile while the other
    // sums, where runs are short and most of the time is the gradient's own bytes, or
    // where square tiles would take more rounds (never fewer) or leave CUs idle in one.
    // They read half as much again, which long runs lose.  Over 1471 calls of 16 shapes
    // (384 to 28672 columns, 4 to 128 experts of 1 to 1024 slots on average) the time is
    // 1.2 % over the better tile's by this rule, 3.8 % with square tiles only, 1.3 % with
    // the others only; limits of 192 to 640 slots are alike within 0.3 %.  By rounds, 128
    // and 256 rows, us: one, 8 experts of 1024 x 1024, 700 slots 27 and 30; 2 and 3, 20 of
    // 384 x 3584, 600 slots 55 and 70; alike, 64 of 2048 x 4096, 24 slots 228 and 264; 24 of
    // 4096 x 2048, 100 slots 143 and 130, 300 slots 206 and 198; 8 of 28672 x 4096, 1024
    // slots 2039 and 1988.
    const int64_t cols = (K + 255) / 256;
    const int64_t half = (E * ((N + 127) / 128) * cols + 511) / 512, square = (E * ((N + 255) / 256) * cols + 255) / 256;
    if (half < square || half == 1 || S <= 224 * (int64_t)E) {
      using T = MmTile<128, 256, 4, 2, 3, 2, 64>;
      return dtype == kFp16 ? launch_tile<Fp16, true, kWgrad, T>(g, st) : launch_tile<Bf16, false, kWgrad, T>(g, st);
    }
    using T = MmTile<256, 256, 8, 4, 4, 1, 64>;
    return dtype == kFp16 ? launch_tile<Fp16, true, kWgrad, T>(g, st) : launch_tile<Bf16, false, kWgrad, T>(g, st);
  }
  return dtype == kFp16 ? launch_any<Fp16, true, true>(g, st) : launch_any<Bf16, false, true>(g, st);
}

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
  // The rows of a tile are free here: as many as there are up to 256, or fewer where
  // tiles of 64 columns do not fill the 256 CUs (us by 16, 32, 64, 128, 256 rows: 1463 x
  // 10640 to 168 columns 29, 23, 29, 39, 61; 256 x 7168 to 4096 66, 37, 22, 24, 33; 512 x
  // 7168 to 512 18, 23, 21, 24, 33; 200 x 1024 to 8192 26, 16, 11, 8.7, 9.9).
  g.bm = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : M <= 128 ? 128 : 256;
  while (M > 32 && g.bm > 16 && (M + g.bm / 2 - 1) / (g.bm / 2) * ((N + 63) / 64) <= 256) g.bm /= 2;
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
