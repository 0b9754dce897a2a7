// Operand types and the arguments of the grouped products (grouped_mm.hip).
#pragma once

#include "common.hpp"
#include "internal.hpp"
#include "mfma_frag.hpp"

#include <type_traits>

namespace moe {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v2f32 __attribute__((ext_vector_type(2)));

// Operand element types.  A fragment is 16 bytes a lane: lane (fr = lane mod 16,
// kseg = lane / 16) holds row fr's 16 bytes at kseg * 16 of a 64-byte run of the
// contraction, 32 values of 16 bits or 64 of 8, for one 16x16 instruction.  The
// two operands place the contraction alike, so its order inside the instruction
// does not matter.
struct Bf16 {
  static constexpr int BYTES = 2;
  typedef v4f Acc;
  static MOE_DEVICE Acc mfma(v4i a, v4i b, Acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  }
};
struct Fp16 {
  static constexpr int BYTES = 2;
  typedef v4f Acc;
  static MOE_DEVICE Acc mfma(v4i a, v4i b, Acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  }
};
// Sums of 8-bit products in 32 bits are exact: |sum| <= 2^14 K < 2^31 for K < 2^17.
struct Int8 {
  static constexpr int BYTES = 1;
  typedef v4i Acc;
  static MOE_DEVICE Acc mfma(v4i a, v4i b, Acc c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
};

// Two fp32 -> a packed pair of the output type, round to nearest even.
template <bool FP16>
MOE_DEVICE uint32_t pack2(float a, float b) {
  if constexpr (FP16) {
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f32){a, b}, v2h));
  } else {
    return pack_bf16x2(a, b);
  }
}
// A 16-bit output value as fp32.
template <bool FP16>
MOE_DEVICE float from16(uint16_t v) {
  if constexpr (FP16) return (float)__builtin_bit_cast(_Float16, v);
  else return bf16_to_f32(v);
}

// An int8 output before its rounding: each operation rounded in fp32 by itself,
// so that every kernel gives the same bits for the same operands.
MOE_DEVICE float int8_out(int acc, float sa, float sb, bool with_bias, float bias, bool weighted, float w) {
#pragma clang fp contract(off)
  float f = (float)acc * sa;
  f = f * sb;
  if (with_bias) f = f + bias;
  if (weighted) f = f * w;
  return f;
}

// One launch of a product.  With sorted, eids and ntpp (as moe_align_block_size
// writes them): position p of block p / bm belongs to expert eids[p / bm] and
// slot sorted[p] (S or more: none).  Without: S rows of one expert, slot p.
//
// Rows form: out[slot][j] = sum_c A[row][c] * B[e][j][c], row = the position with
// a_by_pos, else slot / top_k.  Blocks of an expert outside [0, E) get zero rows.
// Weights form (wgrad): out[e][n][j] = sum over the slots of e of
// A[slot][n] * B[slot / top_k][j].
// Lengths and strides are in elements.
struct MmArgs {
  const uint8_t* A;
  const uint8_t* B;
  uint8_t* C;
  const int32_t* sorted;
  const int32_t* eids;
  const int32_t* ntpp;
  const float* As;      // int8: a scale for each row of A
  const float* Bs;      // int8: a scale for each column of each expert, [E, J]
  const uint16_t* bias; // [J] in the output type, or null
  const float* topk_w;  // a factor for each slot, or null
  int64_t S;
  int64_t J;            // columns of the output
  int64_t Cn;           // rows form: length of the contraction; weights form: rows of an expert's output
  int64_t lda;          // row stride of A
  int64_t sbj, sbc;     // rows form: B's strides along j and c; weights form: sbc is B's row stride
  int64_t b_es;         // B's expert stride
  int64_t ldc;          // row stride of the output
  int64_t n_jt;         // column tiles
  int64_t n_blocks;     // blocks that fit in max_padded
  // [E + 2] first positions and [E + 1] slots of the experts and of the slots
  // without one, or null
  const int32_t* table;
  int64_t shorts;       // rows form with a table: workgroups from this one on take the experts' short last tiles,
  int short_parts;      // so many of them each
  int out32;            // kDgrad: rows of fp32, which are summed over a token's slots before they are rounded
  int bm, top_k, a_by_pos, E;
  // slot / top_k = slot * div_mul >> div_shift for slots below 2^31
  uint32_t div_mul;
  int div_shift;
};

// Sets top_k and its division: with l = ceil(log2 k) and m = floor(2^(31+l) / k) + 1
// the error m k - 2^(31+l) is at most k <= 2^l, so the quotient is exact.
inline void set_top_k(MmArgs& g, int32_t k) {
  int l = 0;
  while (((int64_t)1 << l) < k) ++l;
  g.top_k = k;
  g.div_mul = (uint32_t)(((uint64_t)1 << (31 + l)) / (uint64_t)k + 1);
  g.div_shift = 31 + l;
}
// The row of A (weights form: of B) that a slot reads.
MOE_DEVICE uint32_t slot_row(const MmArgs& g, uint32_t slot) {
  return (uint32_t)((uint64_t)slot * g.div_mul >> g.div_shift);
}

// Blocks that hold slots (ntpp is the device's word: kept to what was allocated).
MOE_DEVICE int64_t live_blocks(const MmArgs& g) {
  if (!g.ntpp) return g.n_blocks;
  const int64_t n = (int64_t)*g.ntpp / g.bm;
  return n < 0 ? 0 : (n < g.n_blocks ? n : g.n_blocks);
}

// One past the last of the workgroup's first N threads with `on`; a barrier.  Rows of
// a block up to its last slot count, for padding may stand between them in sorted
// ids that align did not write.
template <int N>
MOE_DEVICE int end_of(bool on) {
  constexpr int WAVES = (N + 63) / 64;
  __shared__ int ends[WAVES];
  const int wave = threadIdx.x >> 6;
  const uint64_t m = __ballot(on);
  if (wave < WAVES && (threadIdx.x & 63) == 0) ends[wave] = m ? 64 * wave + 64 - __clzll((long long)m) : 0;
  __syncthreads();
  int end = ends[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) end = ends[w] > end ? ends[w] : end;
  return __builtin_amdgcn_readfirstlane(end);
}

// One round of a search in ascending words by the calling wave: [lo, hi] holds the
// place of the first word that is at least v; 64 probes narrow it to a 64th.
MOE_DEVICE void narrow(const int32_t* a, int32_t v, int64_t& lo, int64_t& hi) {
  const int lane = threadIdx.x & 63;
  const int64_t step = (hi - lo + 63) / 64;
  const int64_t i = lo + step * (lane + 1) - 1;  // the lane's probe: the last of its step words
  const uint64_t ge = __ballot(i >= hi || a[i < hi ? i : hi - 1] >= v);
  // words before the first lane's run that reaches v are all smaller
  const int first = ge ? __ffsll((unsigned long long)ge) - 1 : 64;
  const int64_t nlo = lo + step * first, nhi = nlo + step - 1;
  lo = nlo < hi ? nlo : hi;
  hi = nhi < hi ? nhi : hi;
}

// Positions [pos0, pos0 + count) of the slots of expert e: its blocks are
// consecutive and ascending in e, and only the last of them has padding.
struct Run {
  int64_t pos0, count;
};
MOE_DEVICE Run run_of(const MmArgs& g, int e) {
  if (g.table) return {g.table[e], g.table[g.E + 2 + e]};
  const int64_t nb = live_blocks(g);
  int64_t b0 = 0, h0 = nb, b1 = 0, h1 = nb;
  while (b0 < h0 || b1 < h1) {  // both ends in the same rounds: two up to 4096 blocks
    if (b0 < h0) narrow(g.eids, e, b0, h0);
    if (b1 < h1) narrow(g.eids, e + 1, b1, h1);
  }
  Run r = {b0 * g.bm, 0};
  if (b1 <= b0) return r;
  const int lane = threadIdx.x & 63;
  const int32_t* tail = g.sorted + (b1 - 1) * g.bm;
  uint32_t slot[4];  // blocks have up to 256 positions
#pragma unroll
  for (int i = 0; i < 4; ++i) slot[i] = 64 * i + lane < g.bm ? (uint32_t)tail[64 * i + lane] : 0xFFFFFFFFu;
  r.count = (b1 - b0 - 1) * g.bm;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.count += __popcll(__ballot((int64_t)slot[i] < g.S));
  return r;
}

}  // namespace moe
