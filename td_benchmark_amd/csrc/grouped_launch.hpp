// Launches of the products' kernels for rows of whole, aligned 16-byte chunks
// (grouped_mm.hip; gated.hip).
#pragma once

#include "grouped_tile.hpp"

namespace moe {

// A launch has fewer than 2^32 threads.
static bool fits_launch(int64_t workgroups, int threads) { return workgroups <= 0xFFFFFFFFll / threads; }

// ---- whole, aligned chunks ---------------------------------------------------
// Whether tiles of 256 rows are dealt by the experts' counts, and among how many
// workgroups an expert's short last tile is shared (launch_tile).
static bool by_counts(int64_t S, int64_t E, int64_t n_jt) { return S >= 768 * E && S / 256 * n_jt <= 1024; }
static int short_parts(int64_t S, int64_t E, int64_t n_jt, int64_t row_bytes) {
  return (S < E ? S : E) * n_jt <= 256 && row_bytes >= 64 * 128 ? 4 : 1;
}

template <class OP, bool FP16, int FORM, class T>
static int launch_tile(MmArgs g, hipStream_t st) {
  constexpr int kColumns = out_columns(FORM, T::TN);
  g.n_jt = (g.J + kColumns - 1) / kColumns;
  int64_t tiles = (by_weights(FORM) ? g.E * ((g.Cn + T::TM - 1) / T::TM) : g.n_blocks) * g.n_jt, more = 0;
  if (!by_weights(FORM)) {
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
  const int64_t deal = by_weights(FORM) ? 8 * kWgradChunk : 8;
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

template <class OP, bool FP16, int RT, int FORM>
__global__ __launch_bounds__(64 * kFewWaves) void few_mm_kernel(MmArgs g) {
  constexpr int EB = OP::BYTES, TM = 16 * RT, U = 4;
  __shared__ typename OP::Acc part[kFewWaves][RT][64];
  __shared__ int32_t smSlot[TM];
  const int tid = threadIdx.x, lane = tid & 63, fr = lane & 15, kseg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int64_t b, j;
  if (!rows_tile<false>(g, b, j)) return;
  constexpr int kCols = out_columns(FORM, 16);
  const int64_t j0 = j * kCols, pos0 = b * g.bm;
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
  // kGated: rows of 8 gate and the 8 up columns
  const int64_t jc = FORM == kGated ? j0 + (fr & 7) : j0 + fr;
  const int64_t jb = (jc < g.J ? jc : g.J - 1) + (FORM == kGated && fr >= 8 ? g.J : 0);
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
    const int64_t jj = j0 + (FORM == kGated ? 4 * (l >> 4 & 1) : 4 * (l >> 4));
    if (row >= nvalid || jj >= g.J) return;  // J is a multiple of 8
    typename OP::Acc sum = part[0][r][l];
#pragma unroll
    for (int w = 1; w < kFewWaves; ++w) sum = sum + part[w][r][l];
    if constexpr (FORM == kGated) {
      // lanes 0 to 31 hold the gate's, 32 to 63 the up projection's four columns of the row
      const int slot = smSlot[row];
      if (slot < 0 || none) return;
      if (g.gu) *reinterpret_cast<v4f*>(g.gu + (int64_t)slot * 2 * g.J + (l & 32 ? g.J : 0) + jj) = sum;
      if (l & 32) return;
      typename OP::Acc up = part[0][r][l + 32];
#pragma unroll
      for (int w = 1; w < kFewWaves; ++w) up = up + part[w][r][l + 32];
      const float w = g.topk_w ? g.topk_w[slot] : 1.0f;
      float h[4];
#pragma unroll
      for (int v = 0; v < 4; ++v) h[v] = jj + v < g.J_used ? gated(sum[v], up[v], w) : 0.0f;
      const v2u pk = {pack2<FP16>(h[0], h[1]), pack2<FP16>(h[2], h[3])};
      *reinterpret_cast<v2u*>(g.C + ((int64_t)slot * g.ldc + jj) * 2) = pk;
      return;
    }
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
    if constexpr (FORM == kRows32) {
      *reinterpret_cast<v4f*>(g.C + ((int64_t)slot * g.ldc + jj) * 4) = (v4f){f[0], f[1], f[2], f[3]};
    } else {
      const v2u pk = {pack2<FP16>(f[0], f[1]), pack2<FP16>(f[2], f[3])};
      *reinterpret_cast<v2u*>(g.C + ((int64_t)slot * g.ldc + jj) * 2) = pk;
    }
  }
}

template <class OP, bool FP16, int RT, int FORM>
static int launch_few(MmArgs g, hipStream_t st) {
  g.n_jt = (g.J + out_columns(FORM, 16) - 1) / out_columns(FORM, 16);
  const int64_t grid = (g.n_blocks * g.n_jt + 7) / 8 * 8;
  if (!fits_launch(grid, 64 * kFewWaves)) return kErrBadShape;
  hipLaunchKernelGGL((few_mm_kernel<OP, FP16, RT, FORM>), dim3((unsigned)grid), dim3(64 * kFewWaves), 0, st, g);
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

// Rows and columns of a tile; few: few_mm_kernel's split of the contraction.
struct TileChoice {
  int rows, columns;
  bool few;
};
// The tile of the rows form: `blocks` blocks of bm rows that hold S slots, J columns of
// B, whose rows (those along the contraction) have row_bytes.
static TileChoice rows_choice(bool columns, double blocks, int64_t S, int bm, int64_t J, int64_t row_bytes) {
  const double wide = rounds(blocks, J, 256, 1.0), half = rounds(blocks, J, 128, 0.65), slim = rounds(blocks, J, 64, 0.5);
  // Few rows on long rows of weights: few tiles, or one or two slots a block (more
  // rows make it draw as much of A as of the weights).  int8, one row, 7168 x 4096:
  // 16.3 us, staged 24.5; 16 tokens on 128 experts 126 and 148; 9 slots a block of
  // 14336 272 and 226; rows of 768 bytes 123 and 79.
  if (!columns && bm <= 32 && row_bytes >= 2048 && (blocks * ((J + 63) / 64) <= 128.0 || S <= 2.0 * blocks)) return {bm, 16, true};
  if (bm <= 32) return {bm, !columns || wide <= 1.0 ? 64 : 256, false};
  if (bm == 64) return {64, columns && half >= wide ? 256 : slim < half ? 64 : 128, false};
  if (slim < half && slim < wide) return {bm, 64, false};
  return {bm, half < wide ? 128 : 256, false};
}

template <class OP, bool FP16, int FORM>
static int launch_rows(const MmArgs& g, hipStream_t st) {
  const int64_t J = FORM == kGated ? 2 * g.J : g.J;  // columns of B
  const TileChoice t = rows_choice(by_columns(FORM), live_blocks_guess(g), g.S, g.bm, J, g.Cn * OP::BYTES);
  if constexpr (!by_columns(FORM)) {
    if (t.few) return g.bm == 16 ? launch_few<OP, FP16, 1, FORM>(g, st) : launch_few<OP, FP16, 2, FORM>(g, st);
  }
  if (g.bm == 16) {
    if (t.columns == 64) return launch_tile<OP, FP16, FORM, MmTile<16, 64, 2, 1, 4, 2>>(g, st);
    return launch_tile<OP, FP16, FORM, MmTile<16, 256, 8, 1, 3, 1>>(g, st);
  }
  if (g.bm == 32) {
    if (t.columns == 64) return launch_tile<OP, FP16, FORM, MmTile<32, 64, 4, 2, 6, 2>>(g, st);
    return launch_tile<OP, FP16, FORM, MmTile<32, 256, 8, 1, 3, 1>>(g, st);
  }
  if (g.bm == 64) {
    if (t.columns == 64) return launch_tile<OP, FP16, FORM, MmTile<64, 64, 4, 2, 4, 2>>(g, st);
    if (t.columns == 128) return launch_tile<OP, FP16, FORM, MmTile<64, 128, 4, 1, 3, 2>>(g, st);
    return launch_tile<OP, FP16, FORM, MmTile<64, 256, 8, 2, 3, 1>>(g, st);
  }
  if (g.bm == 128) {
    if (t.columns == 64) return launch_tile<OP, FP16, FORM, MmTile<128, 64, 8, 4, 3, 2>>(g, st);
    if (t.columns == 128) return launch_tile<OP, FP16, FORM, MmTile<128, 128, 8, 4, 4, 1>>(g, st);
    return launch_tile<OP, FP16, FORM, MmTile<128, 256, 8, 2, 3, 1>>(g, st);
  }
  if (t.columns == 64) return launch_tile<OP, FP16, FORM, MmTile<256, 64, 8, 4, 3, 1>>(g, st);
  if (t.columns == 128) return launch_tile<OP, FP16, FORM, MmTile<256, 128, 8, 4, 3, 1>>(g, st);
  return launch_tile<OP, FP16, FORM, MmTile<256, 256, 8, 4, 2, 1>>(g, st);
}

// The rows of a dense product's tile are free: as many as there are up to 256, or
// fewer where tiles of 64 columns do not fill the 256 CUs (int8, us by 16, 32, 64,
// 128, 256 rows: 1463 x 10640 to 168 columns 29, 23, 29, 39, 61; 256 x 7168 to 4096 66,
// 37, 22, 24, 33; 512 x 7168 to 512 18, 23, 21, 24, 33; 200 x 1024 to 8192 26, 16, 11,
// 8.7, 9.9).
static int dense_rows(int64_t M, int64_t N) {
  int bm = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : M <= 128 ? 128 : 256;
  while (M > 32 && bm > 16 && (M + bm / 2 - 1) / (bm / 2) * ((N + 63) / 64) <= 256) bm /= 2;
  return bm;
}

// The dense FP8 product's tile for M x N outputs from rows of K codes, by the rules above,
// whose weights fit its steps too: over 176 calls of 7 shapes (512 to 36864 columns from
// 1024 to 7168, 1 to 8192 rows, weights from HBM) the time is 3.0 % over the best of all
// tiles'.  Few rows, split and staged, us: one, to 4096 from 7168 8.2 and 19.2, to 14344
// from 4096 15.7 and 17.3, to 36864 from 7168 59.5 and 68.8; two 9.1 and 19.2, 15.0 and
// 15.7, 57.1 and 64.8; eight 10.3 and 19.2, 18.7 and 15.6, 70.1 and 65.8.  Where it is
// farthest off: 24 and 32 rows to 7168 from 2048, split, 10.9 and 12.3, staged 8.1; 300 to
// 36864 from 7168, 256 x 256, 183, by 128 x 256 139.
static TileChoice fp8_choice(int64_t M, int64_t N, int64_t K, int bm) {
  const double blocks = (double)((M + bm - 1) / bm);
  const double wide = rounds(blocks, N, 256, 1.0), half = rounds(blocks, N, 128, 0.65), slim = rounds(blocks, N, 64, 0.5);
  if (bm <= 32 && K >= 2048 && (blocks * ((N + 63) / 64) <= 128.0 || M <= 2.0 * blocks)) return {bm, 16, true};
  if (bm <= 32) return {bm, 64, false};
  if (bm == 64) return {64, slim < half ? 64 : 128, false};
  if (slim < half && slim < wide) return {bm, 64, false};
  return {bm, half < wide ? 128 : 256, false};
}

// The gradient by weights.  Whether its tiles are square:
//
// Square tiles take steps of 64 slots in a ring of two that is handed over in parts,
// 8 experts of 28672 x 4096, 1024 slots 1970 us, with steps of 32 in a ring of four
// 2130; those of 128 rows, whose stages have no halves, steps of 32 in a ring of three.
// Rows of a column-staged step are whole lines at any length; the rows forms lose with
// steps of 32, whose row-staged lines they read in halves.
//
// Two workgroups a CU with tiles of 128 rows: one writes its tile while the other
// sums, where runs are short and most of the time is the gradient's own bytes, or
// where square tiles would take more rounds (never fewer) or leave CUs idle in one.
// They read half as much again, which long runs lose.  Over 243 calls of 16 shapes
// (384 to 28672 columns, 1 to 256 experts of 1 to 4096 slots on average, each call on the
// buffers of the one before) the time is 1.6 % over the better tile's by this rule, 2.9 %
// by the limit without the rounds, 13.5 % with square tiles only, 1.5 % with the others
// only; limits of 384 to 640 slots make it 0.7 to 0.8 %.  Whole training steps on buffers
// in turn hold them back, 128 rows and 256, us: 16 experts of 4096 x 2048, 256 slots 1042
// and 1074, 384 alike, 640 1743 and 1721; 60 of 2048 x 1408, 267 slots 1418 and 1437; 128
// of 2048 x 768, 256 slots alike, 384 2054 and 2028, 512 2568 and 2517.  By rounds, 128 and
// 256 rows, us: one, 4 experts of 1024 x 1024, 640 slots 18 and 22; 2 and 3, 20 of 384 x
// 3584, 640 slots 47 and 62; by the limit, 24 of 4096 x 2048, 128 slots 107 and 125, 320
// 159 and 182, 1024 427 and 393; 8 of 28672 x 4096, 320 slots 731 and 794, 1024 1910 and
// 1795.
static bool square_choice(int64_t E, int64_t Cn, int64_t J, int64_t S) {
  const int64_t cols = (J + 255) / 256;
  const int64_t half = (E * ((Cn + 127) / 128) * cols + 511) / 512, square = (E * ((Cn + 255) / 256) * cols + 255) / 256;
  return !(half < square || half == 1 || S <= 300 * E);
}

template <int FORM>
static int launch_weights(const MmArgs& g, int32_t dtype, hipStream_t st) {
  if (!square_choice(g.E, g.Cn, g.J, g.S)) {
    using T = MmTile<128, 256, 4, 2, 3, 2, 64>;
    return dtype == MOE_FP16 ? launch_tile<Fp16, true, FORM, T>(g, st) : launch_tile<Bf16, false, FORM, T>(g, st);
  }
  using T = MmTile<256, 256, 8, 4, 2, 1>;
  return dtype == MOE_FP16 ? launch_tile<Fp16, true, FORM, T>(g, st) : launch_tile<Bf16, false, FORM, T>(g, st);
}

static bool aligned(const void* p, int n) { return ((uintptr_t)p & (n - 1)) == 0; }
// Whether rows at p with a stride of ld elements of `bytes` are whole 16-byte chunks.
static bool chunks(const void* p, int64_t ld, int bytes) { return aligned(p, 16) && ld * bytes % 16 == 0; }

constexpr int kBf16 = MOE_BF16, kFp16 = MOE_FP16;

}  // namespace moe
