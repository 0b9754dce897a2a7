// The LDS-tiled kernel of the grouped products (grouped_mm.hip): operands whose
// rows are whole, aligned 16-byte chunks.
//
// A workgroup computes TM x TN outputs.  An operand is staged by rows, R rows of
// 128 bytes of the contraction, where it is contiguous along the contraction (the
// product's x and w, the int8 operands, dy by rows), or by columns, 64 contraction
// rows of R columns, where it is contiguous along the output (w in the gradient by
// rows; dy and x in the gradient by weights, in steps of 32).  Both take R * 128
// (64) bytes of a stage and are filled by direct-to-LDS loads, 16 bytes a lane from
// the lane's own address, so rows are gathered for nothing.  Fragments of a
// row-staged operand are one ds_read_b128; of a column-staged one two
// ds_read_b64_tr_b16, which hand each lane four consecutive contraction values of
// its column.
//
// LDS rows hold their 16-byte chunks at index XOR a function of the row
// (row_place; col_swz), applied on the global side, so that the lanes read
// together fall into distinct banks.
#pragma once

#include "grouped_mm.hpp"

namespace moe {

// The product and its two gradients; then, for the feed-forward block (gated.hip),
// the product into fp32 rows, the product of both projections with the activation,
// the gradient by rows with the activation's gradient, and the gradient by weights
// with a row of A for each token and of B for each slot, or of S rows of one expert
// without a list of slots.
enum Form { kProduct, kDgrad, kWgrad, kRows32, kGated, kActGrad, kWgradTok, kWgradDense };
constexpr bool by_weights(int form) { return form == kWgrad || form == kWgradTok || form == kWgradDense; }
// Whether the rows form reads B along its columns.
constexpr bool by_columns(int form) { return form == kDgrad || form == kActGrad; }
// Output columns of a tile of TN columns of B: kGated pairs 16 of the gate with 16 of
// the up projection, so that a lane holds both of an element.
constexpr int out_columns(int form, int TN) { return form == kGated ? TN / 2 : TN; }

// Tiles of the weights' gradient that go to an XCD together.  Zipf routing (4093
// tokens, 64 experts): 1573 us with an even contiguous range of the experts a XCD,
// 609 so; even routing loses 2 % (8 to 32 are alike, 4 loses 6 % at 32 experts).
constexpr int kWgradChunk = 16;

// TM x TN outputs by NW waves, WM of them along the rows, from a ring of KS
// stages of SB bytes a row, WGS workgroups a CU.
template <int TM_, int TN_, int NW_, int WM_, int KS_, int WGS_, int SB_ = 128>
struct MmTile {
  static constexpr int TM = TM_, TN = TN_, NW = NW_, WM = WM_, KS = KS_, WGS = WGS_, SB = SB_;
  static constexpr int H = SB / 64;  // matrix instructions along the contraction in a step
  static_assert(SB == 64 || SB == 128, "one or two instructions");
  static constexpr int THREADS = 64 * NW, WN = NW / WM, WPE = NW * WGS < 4 ? 1 : NW * WGS / 4;
  static constexpr int RS = TM / WM / 16, CS = TN / WN / 16;  // 16-row and 16-column subtiles of a wave
  static constexpr int A_BYTES = TM * SB, B_BYTES = TN * SB, STAGE = A_BYTES + B_BYTES;
  static constexpr int NA = A_BYTES / 1024, NB = B_BYTES / 1024;  // 1 KiB loads of a stage
  static constexpr int NA_W = (NA + NW - 1) / NW, NB_W = (NB + NW - 1) / NW;
  // loads of a stage that every wave issues at least: what may stay in flight of each younger stage
  static constexpr int VM = NA / NW + NB / NW;
  // LDS: the rows' table (slot, scale, factor) and the columns' (scale, bias), or
  // kWgrad's ring of slots of eight steps; then the ring of stages, whose addresses
  // are formed by XOR below 1 KiB.
  static constexpr int TABLE = (12 * TM + 8 * TN + 1023) / 1024 * 1024;
  static constexpr int LDS_BYTES = TABLE + KS * STAGE;
  static_assert(RS >= 1 && CS >= 1 && TM * TN * 2 <= KS * STAGE && (LDS_BYTES + 1024) * WGS <= 160 * 1024 && TABLE >= 1024, "tile");
  static_assert(VM * (KS - 1) < 64, "vmcnt immediate");
};

// Where a row-staged stage has logical 16-byte chunk c of a row, and its inverse
// (an involution).  A step of 128 bytes is split between its two instructions by
// chunks: lane (fr, kseg) takes chunk 2 kseg of its row for the first and 2 kseg + 1
// for the second, of one of 64 bytes chunk kseg.  With these places the lanes that
// a ds_read_b128 serves together hit distinct banks (chunk 4 h + kseg of a 128-byte
// row gave two-way conflicts, half of the LDS cycles).
template <int SB>
MOE_DEVICE int row_place(int c, int row) {
  return SB == 128 ? slot_of(c, row) : (c ^ (-(row >> 2) & 3));
}
// Chunk rotation of a column-staged row, of which an instruction takes rows
// 16 kseg + 8 h to + 7, or 8 kseg to + 7: the four rows that a group of 16 lanes
// reads together differ in their two low bits, the groups in bit 4 or 3.
template <int SB>
MOE_DEVICE int col_swz(int row) {
  return ((row & 3) << 1) | ((SB == 128 ? row >> 1 : row) & 8);
}

// A barrier, behind which all but the wave's last LGKM reads of LDS have arrived (15: any).
template <int LGKM = 0>
MOE_DEVICE void mm_barrier() { asm volatile("s_waitcnt lgkmcnt(%0)\n\ts_barrier" ::"n"(LGKM) : "memory"); }
template <int N>
MOE_DEVICE void mm_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
// Waits for the oldest stage in flight: of the `younger` ones behind it, at most
// MAX, every wave has at least VM loads each.
template <int MAX, int VM>
MOE_DEVICE void mm_wait_stages(int younger) {
  if constexpr (MAX <= 0) {
    mm_wait<0>();
  } else {
    if (younger >= MAX) mm_wait<MAX * VM>();
    else mm_wait_stages<MAX - 1, VM>(younger);
  }
}

// 16 (or 4) bytes a lane from the lane's address to LDS at a uniform base, lanes
// in order.  The kernel waits for them itself; M0 is written here only.  Not a
// clobber of memory: the fragments' reads may be moved across, which never reads
// the stage being filled; the barriers, which are, keep both in their step.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
MOE_DEVICE void lds_load16(const void* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(lds) : "m0");
}
MOE_DEVICE void lds_load4(const void* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(p), "s"(lds) : "m0");
}
#pragma clang diagnostic pop

// Read in the place of chunks past the contraction's end.
__device__ const v4i kZeroChunk = {0, 0, 0, 0};

typedef __attribute__((address_space(3))) uint8_t* lds_ptr;
MOE_DEVICE v4i lds_frag(uint32_t at) { return *reinterpret_cast<__attribute__((address_space(3))) v4i*>((lds_ptr)(uintptr_t)at); }
typedef short v4s __attribute__((ext_vector_type(4)));
MOE_DEVICE v4i lds_frag_t(uint32_t at, int row_bytes) {
  typedef __attribute__((address_space(3))) v4s* p4;
  const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<p4>((lds_ptr)(uintptr_t)at));
  const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<p4>((lds_ptr)(uintptr_t)(at + 4 * row_bytes)));
  const v2u l = __builtin_bit_cast(v2u, lo), h = __builtin_bit_cast(v2u, hi);
  return (v4i){(int)l[0], (int)l[1], (int)h[0], (int)h[1]};
}

// The workgroup's tile: block b and column tile j of the rows form; workgroups are
// dealt to the XCDs in turn.
//
// Each XCD takes a contiguous range of the live tiles in expert order (dealt out
// in chunks of four instead, decode through W2 takes 5 % longer and 64 rows an
// expert of 64 12 %).  Long blocks (GROUPED): within an expert the column tiles go
// in groups of four with all its row tiles, so that the workgroups that share
// weights or rows run together on one XCD's L2.  Short ones stream weights that
// nobody shares, in tiles of a few microseconds: block by block, without the
// look-up of the expert's run.
template <bool GROUPED>
MOE_DEVICE bool rows_tile(const MmArgs& g, int64_t& b, int64_t& j) {
  constexpr int kXcd = 8, kGroup = 4;
  const int64_t nb = live_blocks(g);
  const int64_t total = nb * g.n_jt, per = (total + kXcd - 1) / kXcd;
  const int64_t pid = blockIdx.x;
  const int64_t t = pid % kXcd * per + pid / kXcd;
  if (pid / kXcd >= per || t >= total) return false;
  b = t / g.n_jt;
  if constexpr (!GROUPED) {
    j = t - b * g.n_jt;
    return true;
  }
  int64_t b0 = 0, n = nb;
  if (g.eids) {  // the run of blocks with b's expert
    const int lane = threadIdx.x & 63;
    const int e = g.eids[b];
    int64_t back = 0, fwd = 1;
    for (int64_t base = b - 1;; base -= 64, back += 64) {
      const int64_t i = base - lane;
      const uint64_t end = __ballot(!(i >= 0 && g.eids[i >= 0 ? i : 0] == e));
      if (end) {
        back += __ffsll((unsigned long long)end) - 1;
        break;
      }
    }
    for (int64_t base = b + 1;; base += 64, fwd += 64) {
      const int64_t i = base + lane;
      const uint64_t end = __ballot(!(i < nb && g.eids[i < nb ? i : 0] == e));
      if (end) {
        fwd += __ffsll((unsigned long long)end) - 1;
        break;
      }
    }
    b0 = b - back;
    n = back + fwd;
  }
  const int64_t in = t - b0 * g.n_jt;
  const int64_t j0 = in / (kGroup * n) * kGroup;
  const int64_t w = g.n_jt - j0 < kGroup ? g.n_jt - j0 : kGroup;
  j = j0 + (in - j0 * n) % w;
  b = b0 + (in - j0 * n) / w;
  return true;
}

// With a table, the tiles of long blocks by the experts' counts: TM rows each, an
// expert's last one of up to SHORT rows apart (`part` of the workgroups that share
// it).  The whole tiles are dealt to the XCDs evenly, as above, but by their number
// alone: a short tile counted as a whole one gives some XCDs more whole ones than
// others, which is a round more where there are few.
template <int TM, int SHORT>
MOE_DEVICE bool table_tile(const MmArgs& g, int64_t& pos0, int64_t& j, int& e, int& nvalid, int& part) {
  constexpr int kGroup = 4;
  const int lane = threadIdx.x & 63, E1 = g.E + 1, n_jt = (int)g.n_jt;
  const int32_t* cnt = g.table + E1 + 1;
  const bool last = SHORT && (int64_t)blockIdx.x >= g.shorts;
  int c, n, incl;  // of the lane's expert: slots, row tiles, and those up to it among these 64
  auto look = [&](int i) {
    c = i < E1 ? cnt[i] : 0;
    const int rest = c % TM;
    const bool is_short = rest > 0 && rest <= SHORT && i < g.E;
    n = last ? (is_short ? 1 : 0) : c / TM + (rest > 0 && !is_short ? 1 : 0);
    incl = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(incl, o);
      if (lane >= o) incl += y;
    }
  };
  int rows = 0;
  for (int i0 = 0; i0 < E1; i0 += 64) {
    look(i0 + lane);
    rows += __builtin_amdgcn_readlane(incl, 63);
  }
  const int each = last ? n_jt * g.short_parts : n_jt, total = rows * each;
  int t;
  if (last) {
    t = (int)((int64_t)blockIdx.x - g.shorts);
  } else {
    const int per = (total + 7) / 8, l = (int)(blockIdx.x / 8);
    if (l >= per) return false;
    t = (int)(blockIdx.x % 8) * per + l;
  }
  if (t >= total) return false;
  const int at = t / each;  // the row tile among all experts'
  int before = 0;
  for (int i0 = 0;; i0 += 64) {
    if (E1 > 64) look(i0 + lane);
    const uint64_t hit = __ballot(before + incl > at);
    if (hit) {
      const int src = __ffsll((unsigned long long)hit) - 1;
      e = i0 + src;
      n = __builtin_amdgcn_readlane(n, src);
      c = __builtin_amdgcn_readlane(c, src);
      before += __builtin_amdgcn_readlane(incl, src) - n;
      break;
    }
    before += __builtin_amdgcn_readlane(incl, 63);
  }
  int u;
  if (last) {
    u = c / TM;
    part = t % each % g.short_parts;
    j = t % each / g.short_parts;
  } else {
    const int in = t - before * n_jt, g0 = in / (kGroup * n) * kGroup, w = n_jt - g0 < kGroup ? n_jt - g0 : kGroup;
    part = 0;
    j = g0 + (in - g0 * n) % w;
    u = (in - g0 * n) / w;
  }
  pos0 = g.table[e] + (int64_t)u * TM;
  nvalid = c - u * TM < TM ? c - u * TM : TM;
  return true;
}

// The 16-bit halves of a pair of outputs at columns j and j + 1 that count.
MOE_DEVICE int used_pair(const MmArgs& g, int64_t j) { return j + 1 < g.J_used ? -1 : j < g.J_used ? 0xFFFF : 0; }

// One tile: rows [i0, i0 + nvalid) of the output, or the slots of the table's first
// nvalid rows, by columns j0 on (col0 on of the columns' table), over `length` of the
// contraction.  K: the tile of the launch, which T is or is a part of.
template <class OP, bool FP16, int FORM, class K, class T>
MOE_DEVICE void mm_tile(const MmArgs& g, uint8_t* smem, int64_t pos0, int64_t i0, int64_t j0, int col0, int e,
                        int nvalid, int64_t length) {
  constexpr int EB = OP::BYTES, TM = T::TM, TN = T::TN, KS = T::KS, SB = T::SB;
  constexpr bool WEIGHTS = by_weights(FORM), COLUMNS = by_columns(FORM);
  constexpr bool A_COLS = WEIGHTS, B_COLS = WEIGHTS || COLUMNS;
  constexpr int STEP = SB / EB;  // contraction elements of a step
  static_assert(EB == 2 || FORM == kProduct, "transposing reads are of 16-bit values");
  static_assert(!WEIGHTS || (KS <= 4 && 8 * STEP * 4 <= K::TABLE), "the ring of slots");
  static_assert(T::THREADS == K::THREADS && T::LDS_BYTES <= K::LDS_BYTES && T::TABLE <= K::TABLE, "a part of the launch's tile");
  const int32_t* smSlot = reinterpret_cast<const int32_t*>(smem);
  const float* smSa = reinterpret_cast<const float*>(smem) + K::TM;
  const float* smW = reinterpret_cast<const float*>(smem) + 2 * K::TM;
  const float* smSb = reinterpret_cast<const float*>(smem) + 3 * K::TM + col0;
  const float* smBias = smSb + K::TN;
  uint8_t* const ring = smem + K::TABLE;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr)ring;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int KB = (int)((length + STEP - 1) / STEP);

  // A ring of two: the stage is handed over in two parts, A with the first half of
  // every wave's columns, and their second half (below).
  constexpr bool PHASED = KS == 2;
  static_assert(!PHASED || (T::H == 2 && T::WN == 2 && T::CS == 8 && T::NW == 8 && TM == 256), "halves of a stage");

  // ---- addresses of this lane's part of the loads ----
  // Instruction i of a wave is load wave + NW i of its operand; of a phased B, load
  // wave + NW (i mod 2) of the first or second half of the columns, of which a
  // column-staged half lies by itself.
  const uint8_t* a_ptr[T::NA_W];
  const uint8_t* b_ptr[T::NB_W];
  constexpr int BW = PHASED ? TN / 2 : TN;            // columns of a column-staged part of B
  constexpr int ACPR = TM / 8, BCPR = BW / 8;         // chunks of a column-staged row
  auto b_load = [&](int i) {
    if constexpr (!PHASED) return wave + T::NW * i;
    else if constexpr (B_COLS) return wave + T::NW * (i & 1);
    else return wave + T::NW * (2 * (i & 1) + (i >> 1));
  };
  auto b_place = [&](int i) { return T::A_BYTES + (PHASED && B_COLS ? (i >> 1) * (T::B_BYTES / 2) : 0) + b_load(i) * 1024; };
  const uint8_t* b_base = g.B + (WEIGHTS ? 0 : (int64_t)e * g.b_es * EB);
  const uint8_t* zeros = reinterpret_cast<const uint8_t*>(&kZeroChunk);
  constexpr int LPR = SB / 16, RPI = 64 / LPR;  // lanes of a row, rows of a load
  auto row_chunk = [&](int gi) { return row_place<SB>(lane % LPR, RPI * gi + lane / LPR); };
  // contraction row and column chunk of a column-staged load
  auto col_row = [&](int gi, int cpr) { return gi * (64 / cpr) + lane / cpr; };
  auto col_of = [&](int gi, int cpr) { return ((lane % cpr) ^ (col_swz<SB>(col_row(gi, cpr)) & (cpr - 1))) * 8; };
  // Weights: the element of the contraction that a staged row of step kk holds.  A step
  // of two instructions takes 32 elements with each; its step 0 is the contraction's
  // last, partial run of 32 and, where the others' steps leave one over, the first run:
  // the sum's order is that of steps of 32, so tiles of either length give the same bits.
  constexpr bool PAIRS = WEIGHTS && T::H == 2;
  const int64_t last_run = (length - 1) / 32 * 32;
  const int spare = PAIRS && last_run % 64 ? 32 : 0;
  auto element = [&](int kk, int row) -> int64_t {
    const int h = PAIRS ? row >> 3 & 1 : 0, i = PAIRS ? (row >> 4) * 8 + (row & 7) : row;
    if (kk == 0) return h ? i : last_run + i;
    return (int64_t)(kk - 1) * STEP + spare + 32 * h + i;
  };
  auto in_first = [&](int row) { return PAIRS && (row >> 3 & 1) ? spare != 0 : element(0, row) < length; };
#pragma unroll
  for (int i = 0; i < T::NA_W; ++i) {
    const int gi = wave + T::NW * i;
    if constexpr (A_COLS) {
      const int64_t c = i0 + col_of(gi, ACPR);
      a_ptr[i] = g.A + (c < g.Cn ? c : 0) * EB;
    } else {
      const int row = RPI * gi + lane / LPR;
      const int slot = gi < T::NA ? smSlot[row] : -1;
      const int64_t ar = slot < 0 ? 0 : g.a_by_pos ? pos0 + row : (int64_t)slot_row(g, (uint32_t)slot);
      a_ptr[i] = g.A + ar * g.lda * EB + row_chunk(gi) * 16 - SB;
    }
  }
#pragma unroll
  for (int i = 0; i < T::NB_W; ++i) {
    const int gi = b_load(i);
    if constexpr (B_COLS) {
      int in = col_of(gi, BCPR);
      if constexpr (PHASED) in = (in / (8 * T::CS)) * (16 * T::CS) + (i >> 1) * (8 * T::CS) + in % (8 * T::CS);
      const int64_t c = j0 + in;
      b_ptr[i] = b_base + (c < g.J ? c : 0) * EB;
      if constexpr (COLUMNS) b_ptr[i] += ((int64_t)col_row(gi, BCPR) - STEP) * g.sbc * EB;
    } else {
      const int row = RPI * gi + lane / LPR;
      int64_t j;
      if constexpr (FORM == kGated) {
        j = j0 + (row >> 5) * 16 + (row & 15);
        j = (j < g.J ? j : g.J - 1) + (row & 16 ? g.J : 0);
      } else {
        j = j0 + row;
        j = j < g.J ? j : g.J - 1;
      }
      b_ptr[i] = b_base + j * g.sbj * EB + row_chunk(gi) * 16 - SB;
    }
  }
  // kWgrad: the slots of this lane's rows of a step, read ahead of its loads; square
  // tiles place both operands alike
  constexpr bool SAME = TM == BW;
  uint32_t slot_a[T::NA_W], slot_b[T::NB_W];
  auto read_slots = [&](int kk) {
    if constexpr (FORM == kWgradDense) {  // row c of the contraction is slot c
      auto at = [&](int row) {
        const uint32_t c = (uint32_t)element(kk, row), end = (uint32_t)length - 1;
        return c < end ? c : end;
      };
#pragma unroll
      for (int i = 0; i < T::NA_W; ++i) slot_a[i] = at(col_row(wave + T::NW * i, ACPR));
#pragma unroll
      for (int i = 0; i < T::NB_W; ++i) slot_b[i] = SAME ? slot_a[i < T::NA_W ? i : 0] : at(col_row(b_load(i), BCPR));
      return;
    }
#pragma unroll
    for (int i = 0; i < T::NA_W; ++i)
      slot_a[i] = (uint32_t)smSlot[(kk & 7) * STEP + col_row(wave + T::NW * i, ACPR)];
#pragma unroll
    for (int i = 0; i < T::NB_W; ++i)
      slot_b[i] = SAME ? slot_a[i < T::NA_W ? i : 0] : (uint32_t)smSlot[(kk & 7) * STEP + col_row(b_load(i), BCPR)];
  };

  // Load d of this wave's share of step kk into its stage.  Step 0 is the last,
  // partial run of the contraction, so that no other step has to look for its
  // end; the addresses of the others start a step before the contraction and advance
  // ahead of each load, in their registers (two additions a load if the compiler derives
  // them from the step's number).
  const int tail = (int)(length - (int64_t)(KB - 1) * STEP);  // elements of step 0
  const int64_t b_step = COLUMNS ? STEP * g.sbc * EB : SB;
  constexpr int ND = T::NA_W + T::NB_W;
  auto load = [&](int kk, int stage, auto dc, auto first_c) {
    constexpr int d = decltype(dc)::value;
    constexpr bool first = decltype(first_c)::value;
    const uint32_t dst = lds0 + stage * T::STAGE;
    const int left = first ? tail : STEP;
    // B before A; phased: B's first half, A, B's second half
    constexpr int first_b = PHASED ? T::NB_W / 2 : T::NB_W;
    constexpr bool is_b = d < first_b || d >= first_b + T::NA_W;
    constexpr int i = d < first_b ? d : is_b ? d - T::NA_W : d - first_b;
    const int gi = is_b ? b_load(i) : wave + T::NW * i;
    if constexpr (WEIGHTS) {
      const uint8_t* p;
      if constexpr (is_b) p = b_ptr[i] + (uint64_t)(FORM == kWgrad ? slot_row(g, slot_b[i]) : slot_b[i]) * (uint32_t)(g.sbc * EB);
      else p = a_ptr[i] + (uint64_t)(FORM == kWgradTok ? slot_row(g, slot_a[i]) : slot_a[i]) * (uint32_t)(g.lda * EB);
      if constexpr (first) p = in_first(col_row(gi, is_b ? BCPR : ACPR)) ? p : zeros;
      if ((is_b ? T::NB : T::NA) % T::NW == 0 || gi < (is_b ? T::NB : T::NA))
        lds_load16(p, dst + (is_b ? b_place(i) : gi * 1024));
    } else if constexpr (is_b) {
      const uint8_t* p;
      if constexpr (first) {
        const bool in = COLUMNS ? col_row(gi, BCPR) < left : row_chunk(gi) * 16 < left * EB;
        p = in ? b_ptr[i] + KB * b_step : zeros;
      } else {
        b_ptr[i] += b_step;
        asm volatile("" : "+v"(b_ptr[i]));
        p = b_ptr[i];
      }
      if (T::NB % T::NW == 0 || gi < T::NB) lds_load16(p, dst + b_place(i));
    } else {
      const uint8_t* p;
      if constexpr (first) {
        p = row_chunk(gi) * 16 < left * EB ? a_ptr[i] + (int64_t)KB * SB : zeros;
      } else {
        a_ptr[i] += SB;
        asm volatile("" : "+v"(a_ptr[i]));
        p = a_ptr[i];
      }
      if (T::NA % T::NW == 0 || gi < T::NA) lds_load16(p, dst + gi * 1024);
    }
  };
  // Loads [from, to) of step kk.
  auto loads = [&](int kk, int stage, auto from, auto to, auto first) {
    [&]<int... D>(std::integer_sequence<int, D...>) {
      (load(kk, stage, std::integral_constant<int, decltype(from)::value + D>{}, first), ...);
    }(std::make_integer_sequence<int, decltype(to)::value - decltype(from)::value>{});
  };
  // kWgrad: the slots of step kk into the ring (the last wave), kAhead steps before
  // its own loads are issued: by then the waits for the stages have passed it.
  constexpr int kAhead = 3;
  auto issue_ids = [&](int kk) {
    if (wave == T::NW - 1 && kk < KB && lane < STEP) {
      const int64_t c = element(kk, lane);
      lds_load4(g.sorted + pos0 + (c < length ? c : length - 1), (uint32_t)(uintptr_t)(lds_ptr)smem + (kk & 7) * STEP * 4);
    }
  };

  // ---- fragments ----
  const int fr = lane & 15, kseg = lane >> 4;
  const int wm = wave / T::WN, wn = wave % T::WN;
  const int row_base = wm * T::RS * 16, col_base = wn * T::CS * 16;
  const uint32_t by_row = fr * SB + (row_place<SB>(T::H * kseg, fr) << 4);  // the second half of the step: XOR 16
  const int t_row = 8 * T::H * kseg + (fr >> 2);                            // and 8 rows on
  // column-staged, subtile s of the operand's columns from `base`: XOR s * 32 into the chunk
  auto by_col = [&](int base, int w) {
    return (uint32_t)(t_row * w * 2 + (((base / 8 + ((fr & 3) >> 1)) ^ (col_swz<SB>(t_row) & (w / 8 - 1))) << 4) + (fr & 1) * 8);
  };
  const uint32_t a_lane = A_COLS ? by_col(row_base, TM) : row_base * SB + by_row;
  const uint32_t b_lane = T::A_BYTES + (B_COLS ? by_col(PHASED ? col_base / 2 : col_base, BW) : col_base * SB + by_row);

  typename OP::Acc acc[T::RS][T::CS] = {};
  int ra = (nvalid - row_base + 15) / 16;
  ra = ra < 0 ? 0 : (ra > T::RS ? T::RS : ra);

  if constexpr (WEIGHTS && FORM != kWgradDense) {
    if (KB > 0) {
      for (int s = 0; s < KS + kAhead; ++s) issue_ids(s);
      mm_wait<0>();
    }
    __syncthreads();
  }
  const std::integral_constant<int, 0> none;
  const std::integral_constant<int, ND> all;
  if constexpr (WEIGHTS) read_slots(0);
  if (KB > 0) loads(0, 0, none, all, std::true_type{});
#pragma unroll
  for (int s = 1; s < KS; ++s) {
    if constexpr (WEIGHTS) read_slots(s);
    if (s < KB) loads(s, s, none, all, std::false_type{});
  }

  // A step is H CS slots of RS matrix instructions, one weight fragment each, which
  // is read two slots ahead.  The barrier that hands over the next stage stands two
  // slots before the step's end, when every fragment of this stage has been read:
  // the last two slots' instructions cover the reads of the next stage's first
  // fragments, and this stage's buffer is filled again from there on, a load a slot.
  //
  // Phased: the first half of a step's slots takes the first half of the columns, both
  // instructions along the contraction, and the second half the other, with the rows'
  // fragments in registers all the step.  A second barrier, two slots before the
  // middle, hands over the second half of the columns; behind it the stage's A and
  // first half of B are filled again, behind the step's barrier its second half, so
  // that every load has one and a half steps to arrive and a stage's worth of younger
  // ones stays in flight at each wait.
  //
  // What bounds it: a step's instructions take 2048 cycles of a SIMD, the step 2940
  // (4096 x 7168 to 4096 in 182 us at the least, 1.32 PF, 200 at the median), with
  // barriers of 100-200 and none in waits for loads; LDS gives 250 bytes a cycle, of
  // which the fragments take 66.  Fewer cycles lower the clock: 3300 a step ran at 1.96
  // GHz, 2940 at 1.82, at the board's power.
  // Four waves of 128 x 128, which read a third less from LDS, took 225 us for 196: one
  // wave a SIMD has nothing to run while it waits.
  constexpr int NQ = T::H * T::CS, MID = NQ / 2 - 2;
  constexpr auto half_of = [](int q) { return PHASED ? q % (NQ / 2) / (T::CS / 2) : q / T::CS; };
  constexpr auto column_of = [](int q) { return PHASED ? q / (NQ / 2) * (T::CS / 2) + q % (T::CS / 2) : q % T::CS; };
  constexpr int DPQ = (ND + NQ - 1) / NQ;  // loads of a slot
  static_assert(NQ >= 4 && NQ % 4 == 0, "four fragment registers in turn");
  auto kloop = [&](auto ra_c) {
    constexpr int RA = decltype(ra_c)::value;
    if (KB == 0) return;
    v4i af[2][RA > 0 ? RA : 1], bf[4];
    // Phased: a stage's addresses, from which its reads have constant offsets; the
    // compiler would add up each of them by itself.
    constexpr int VA = PHASED ? (A_COLS ? T::RS : 2) : 1, VB = PHASED ? (B_COLS ? T::CS / 2 : 2) : 1;
    uint32_t a_at[VA], b_at[VB];
    auto place = [&](int stage) {
      if constexpr (PHASED) {
        const uint32_t st = lds0 + stage * T::STAGE;
#pragma unroll
        for (int v = 0; v < VA; ++v) {
          a_at[v] = st + (a_lane ^ (v * (A_COLS ? 32 : 16)));
          asm volatile("" : "+v"(a_at[v]));
        }
#pragma unroll
        for (int v = 0; v < VB; ++v) {
          b_at[v] = st + (b_lane ^ (v * (B_COLS ? 32 : 16)));
          asm volatile("" : "+v"(b_at[v]));
        }
      }
    };
    auto read_a = [&](int to, int stage, int h, int r) {
      const uint32_t st = lds0 + stage * T::STAGE;
      if constexpr (A_COLS) af[to][r] = lds_frag_t((PHASED ? a_at[r % VA] : st + (a_lane ^ (r * 32))) + h * 8 * TM * 2, TM * 2);
      else af[to][r] = lds_frag((PHASED ? a_at[h % VA] : st + (a_lane ^ (h * 16))) + r * 16 * SB);
    };
    auto read_b = [&](int stage, int q) {
      const uint32_t st = lds0 + stage * T::STAGE;
      const int h = half_of(q), c = column_of(q);
      if constexpr (B_COLS && PHASED) bf[q & 3] = lds_frag_t(b_at[c % VB] + c / VB * (T::B_BYTES / 2) + h * 8 * BW * 2, BW * 2);
      else if constexpr (B_COLS) bf[q & 3] = lds_frag_t(st + (b_lane ^ (c * 32)) + h * 8 * TN * 2, TN * 2);
      else bf[q & 3] = lds_frag((PHASED ? b_at[h % VB] : st + (b_lane ^ (h * 16))) + c * 16 * SB);
    };
    place(0);
    // stage 0; of the others every wave has at least so many loads behind it
    constexpr int VM2 = T::NB / T::NW / 2, VM1 = T::VM - VM2;  // loads of the two parts
    if constexpr (PHASED) {
      if (KB > 1) mm_wait<VM2 + T::VM>();
      else mm_wait<VM2>();
    } else {
      mm_wait_stages<KS - 1, T::VM>(KB - 1);
    }
    mm_barrier();
    if constexpr (RA > 0) {
#pragma unroll
      for (int r = 0; r < RA; ++r) read_a(0, 0, 0, r);
      read_b(0, 0);
      read_b(0, 1);
    }
    int stage = 0;
    // P: with one instruction a step, which of the two sets of row fragments it takes
    // STEADY: the steps whose loads there are, without a branch for each
    auto step = [&](int kk, auto pc, auto steady_c) {
      constexpr int P = decltype(pc)::value;
      constexpr bool STEADY = decltype(steady_c)::value;
      const int next = stage == KS - 1 ? 0 : stage + 1, prev = stage == 0 ? KS - 1 : stage - 1;
      auto slot = [&](auto qc) {
        constexpr int Q = decltype(qc)::value;
        if constexpr (Q == NQ - 2) {
          if (STEADY || kk + 1 < KB) {
            if constexpr (PHASED) {
              if (STEADY || kk + 2 < KB) mm_wait<VM2 + VM1>();
              else mm_wait<VM2>();
            } else {
              if constexpr (STEADY) mm_wait<(KS - 2) * T::VM>();
              else mm_wait_stages<KS - 2, T::VM>(KB - 2 - kk);
            }
            mm_barrier();
            if constexpr (WEIGHTS && !PHASED) {
              if (STEADY || kk + KS < KB) {
                read_slots(kk + KS);
                if constexpr (FORM != kWgradDense) issue_ids(kk + KS + kAhead);
              }
            }
          }
          // behind the last step nothing uses these: under the condition, the compiler
          // would wait for them before this slot's instructions
          place(next);
          if constexpr (RA > 0) {
#pragma unroll
            for (int r = 0; r < RA; ++r) read_a(T::H == 2 ? 0 : P ^ 1, next, 0, r);
            read_b(next, 0);
            read_b(next, 1);
          }
        }
        if constexpr (PHASED && Q == MID) {
          if (STEADY || kk + 1 < KB) mm_wait<T::VM>();
          else mm_wait<0>();
          mm_barrier();
          if constexpr (WEIGHTS) {
            if (STEADY || kk + KS < KB) {
              read_slots(kk + KS);
              if constexpr (FORM != kWgradDense) issue_ids(kk + KS + kAhead);
            }
          }
        }
        if constexpr (RA > 0 && Q < NQ - 2) {
          read_b(stage, Q + 2);
          // phased: the second half's rows in the first two slots
          if constexpr (PHASED && Q < 2) {
#pragma unroll
            for (int r = 0; r < RA; ++r)
              if ((r < 2) == (Q == 0)) read_a(1, stage, 1, r);
          }
          // the second half's rows: one a slot up to two slots ahead, or together
          if constexpr (!PHASED && T::H == 2 && T::CS > RA + 1 && Q + RA >= T::CS - 1 && Q < T::CS - 1) read_a(1, stage, 1, Q + RA - (T::CS - 1));
          if constexpr (!PHASED && T::H == 2 && T::CS <= RA + 1 && Q == 0) {
#pragma unroll
            for (int r = 0; r < RA; ++r) read_a(1, stage, 1, r);
          }
        }
        // loads of stage kk + KS in this step's last two slots, of the stage before it in the others
        constexpr int from = PHASED ? (Q >= NQ - 2 ? Q - (NQ - 2) + VM1 : Q - MID) : (Q + 2) % NQ * DPQ;
        constexpr int to = PHASED ? from + 1 : from + DPQ < ND ? from + DPQ : ND;
        if constexpr (PHASED) {  // of stage kk + KS
          if constexpr ((from >= 0 && from < VM1) || Q >= NQ - 2) {
            if (STEADY || kk + KS < KB) loads(kk + KS, stage, std::integral_constant<int, from>{}, std::integral_constant<int, to>{}, std::false_type{});
          }
        } else if constexpr (from < ND) {
          const std::integral_constant<int, from> f;
          const std::integral_constant<int, to> t;
          if constexpr (Q >= NQ - 2) {
            if (STEADY || kk + KS < KB) loads(kk + KS, stage, f, t, std::false_type{});
          } else {
            if (STEADY || (kk > 0 && kk - 1 + KS < KB)) loads(kk - 1 + KS, prev, f, t, std::false_type{});
          }
        }
        // the reads stay ahead of the instructions, which the compiler would undo
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (RA > 0) {
          constexpr int at = T::H == 2 ? half_of(Q) : P, c = column_of(Q);
#pragma unroll
          for (int r = 0; r < RA; ++r) acc[r][c] = OP::mfma(bf[Q & 3], af[at][r], acc[r][c]);
        }
        __builtin_amdgcn_sched_barrier(0);
      };
      [&]<int... Q>(std::integer_sequence<int, Q...>) {
        (slot(std::integral_constant<int, Q>{}), ...);
      }(std::make_integer_sequence<int, NQ>{});
      stage = next;
    };
    const std::integral_constant<int, 0> p0;
    const std::integral_constant<int, 1> p1;
    const std::false_type any;
    int kk = 0;
    if constexpr (T::H == 2) {
      if constexpr (RA == T::RS) {
        if constexpr (!PHASED) step(kk++, p0, any);  // which has nothing of the stage before it to load
        for (; kk + KS < KB; ++kk) step(kk, p0, std::true_type{});
      }
      for (; kk < KB; ++kk) step(kk, p0, any);
    } else {
      auto two = [&](auto steady) {
        step(kk, p0, steady);
        if (decltype(steady)::value || kk + 1 < KB) step(kk + 1, p1, steady);
        kk += 2;
      };
      if constexpr (RA == T::RS) {
        two(any);
        while (kk + 1 + KS < KB) two(std::true_type{});
      }
      while (kk < KB) two(any);
    }
  };
  switch (ra) {
    case 0: kloop(std::integral_constant<int, 0>{}); break;
    case 1: kloop(std::integral_constant<int, 1>{}); break;
    case 2: if constexpr (T::RS >= 2) kloop(std::integral_constant<int, (T::RS >= 2 ? 2 : 1)>{}); break;
    case 3: if constexpr (T::RS >= 3) kloop(std::integral_constant<int, (T::RS >= 3 ? 3 : 1)>{}); break;
    default: if constexpr (T::RS >= 4) kloop(std::integral_constant<int, (T::RS >= 4 ? 4 : 1)>{}); break;
  }
  mm_barrier();

  if constexpr (FORM == kDgrad || FORM == kRows32) {
    // fp32 rows: 16 rows of the wave's columns a time through its own part of the
    // ring, so that a row's columns leave as one run
    if (FORM == kRows32 || g.out32) {
      constexpr int CPR = 4 * T::CS;  // 16-byte chunks of a row
      static_assert(T::NW * 16 * CPR * 16 <= KS * T::STAGE, "staging of fp32 rows");
      v4f* part = reinterpret_cast<v4f*>(ring) + wave * 16 * CPR;
#pragma unroll
      for (int r = 0; r < T::RS; ++r) {
        if (row_base + r * 16 >= nvalid) break;
#pragma unroll
        for (int c = 0; c < T::CS; ++c) part[fr * CPR + ((4 * c + kseg) ^ (fr & (CPR - 1) & 15))] = acc[r][c];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int i = 0; i < CPR / 4; ++i) {
          const int row = (i * 64 + lane) / CPR, cc = (i * 64 + lane) % CPR;
          const int64_t jj = j0 + col_base + 4 * cc;
          const v4f v = part[row * CPR + (cc ^ (row & (CPR - 1) & 15))];
          const int slot = row_base + r * 16 + row < nvalid ? smSlot[row_base + r * 16 + row] : -1;
          if (slot >= 0 && jj < g.J)
            *reinterpret_cast<v4f*>(reinterpret_cast<float*>(g.C) + (int64_t)slot * g.ldc + jj) = v;
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      return;
    }
  }

  if constexpr (FORM == kGated || FORM == kActGrad) {
    // As above: 16 rows of the wave's fp32 columns a time through its part of the
    // ring, from where a lane takes 8 columns of a row.
    constexpr int CPR = 4 * T::CS;
    static_assert(T::NW * 16 * CPR * 16 <= KS * T::STAGE && T::CS % 2 == 0, "staging of fp32 rows");
    v4f* part = reinterpret_cast<v4f*>(ring) + wave * 16 * CPR;
    auto stage = [&](int r) {
#pragma unroll
      for (int c = 0; c < T::CS; ++c) part[fr * CPR + ((4 * c + kseg) ^ (fr & (CPR - 1) & 15))] = acc[r][c];
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    };
    auto chunk = [&](int row, int c) { return part[row * CPR + (c ^ (row & (CPR - 1) & 15))]; };
    constexpr int UPR = FORM == kGated ? T::CS : 2 * T::CS;  // lanes of a row
    constexpr int NI = (16 * UPR + 63) / 64;
#pragma unroll
    for (int r = 0; r < T::RS; ++r) {
      if (row_base + r * 16 >= nvalid) break;
      if constexpr (FORM == kGated) {
        stage(r);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int row = (i * 64 + lane) / UPR, u = (i * 64 + lane) % UPR;
          const int64_t jj = j0 + wn * T::CS * 8 + 8 * u;
          const int slot = row < 16 && row_base + r * 16 + row < nvalid ? smSlot[row_base + r * 16 + row] : -1;
          if (slot < 0 || jj >= g.J) continue;
          const int c = 8 * (u >> 1) + 2 * (u & 1);  // of the gate; the up projection's 4 chunks on
          const v4f gl = chunk(row, c), gh = chunk(row, c + 1), ul = chunk(row, c + 4), uh = chunk(row, c + 5);
          if (g.gu) {
            v4f* to = reinterpret_cast<v4f*>(g.gu + (int64_t)slot * 2 * g.J + jj);
            to[0] = gl;
            to[1] = gh;
            to = reinterpret_cast<v4f*>(g.gu + (int64_t)slot * 2 * g.J + g.J + jj);
            to[0] = ul;
            to[1] = uh;
          }
          const float w = g.topk_w ? g.topk_w[slot] : 1.0f;
          v4i out;
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            out[v] = (int)pack2<FP16>(gated(gl[2 * v], ul[2 * v], w), gated(gl[2 * v + 1], ul[2 * v + 1], w));
            out[2 + v] = (int)pack2<FP16>(gated(gh[2 * v], uh[2 * v], w), gated(gh[2 * v + 1], uh[2 * v + 1], w));
          }
          if (jj + 8 > g.J_used) {
#pragma unroll
            for (int v = 0; v < 4; ++v) out[v] &= used_pair(g, jj + 2 * v);
          }
          *reinterpret_cast<v4i*>(g.C + ((int64_t)slot * g.ldc + jj) * 2) = out;
        }
      } else {
        // the saved products of all of the lane's elements are on their way before the first is used
        v4f gu[NI][4];
        int slots[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int row = (i * 64 + lane) / UPR;
          const int64_t jj = j0 + col_base + 8 * (lane % UPR);
          slots[i] = row_base + r * 16 + row < nvalid && jj < g.J ? smSlot[row_base + r * 16 + row] : -1;
          const v4f* from = reinterpret_cast<const v4f*>(g.gu + (int64_t)(slots[i] < 0 ? 0 : slots[i]) * 2 * g.J + (jj < g.J ? jj : 0));
          const v4f* up = reinterpret_cast<const v4f*>(reinterpret_cast<const float*>(from) + g.J);
          gu[i][0] = from[0];
          gu[i][1] = from[1];
          gu[i][2] = up[0];
          gu[i][3] = up[1];
        }
        stage(r);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int row = (i * 64 + lane) / UPR, u = lane % UPR, slot = slots[i];
          const int64_t jj = j0 + col_base + 8 * u;
          float sum = 0.0f;
          if (slot >= 0) {
            v4f dl = chunk(row, 2 * u), dh = chunk(row, 2 * u + 1);
            if (jj + 8 > g.J_used) {
#pragma unroll
              for (int n = 0; n < 8; ++n) {
                if (jj + n < g.J_used) continue;
                (n < 4 ? dl : dh)[n & 3] = 0.0f;
                gu[i][n < 4 ? 0 : 1][n & 3] = gu[i][n < 4 ? 2 : 3][n & 3] = 0.0f;
              }
            }
            const float w = g.topk_w ? g.topk_w[slot] : 1.0f;
            v4i dg, du;
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              float a[2], b[2];
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const int n = 2 * v + x;
                sum += gated_grad(n < 4 ? dl[n & 3] : dh[n & 3], gu[i][n < 4 ? 0 : 1][n & 3], gu[i][n < 4 ? 2 : 3][n & 3], w, a[x], b[x]);
              }
              dg[v] = (int)pack2<FP16>(a[0], a[1]);
              du[v] = (int)pack2<FP16>(b[0], b[1]);
            }
            if (jj + 8 > g.J_used) {
#pragma unroll
              for (int v = 0; v < 4; ++v) {
                dg[v] &= used_pair(g, jj + 2 * v);
                du[v] &= used_pair(g, jj + 2 * v);
              }
            }
            uint8_t* to = g.C + ((int64_t)slot * g.ldc + jj) * 2;
            *reinterpret_cast<v4i*>(to) = dg;
            *reinterpret_cast<v4i*>(to + 2 * g.J) = du;
          }
          if (g.parts) {  // of 32 columns, whatever the tile
            sum += __shfl_xor(sum, 1);
            sum += __shfl_xor(sum, 2);
            if (slot >= 0 && (u & 3) == 0) g.parts[(int64_t)slot * ((g.J + 31) / 32) + jj / 32] = sum;
          }
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    return;
  }

  // ---- epilogue: rows of 16-bit outputs through LDS, chunks XOR the row ----
  uint16_t* out = reinterpret_cast<uint16_t*>(ring);
  constexpr int CH = TN / 8, ROT = CH < 16 ? CH - 1 : 15;
#pragma unroll
  for (int c = 0; c < T::CS; ++c) {
    const int col = col_base + c * 16 + 4 * kseg;
#pragma unroll
    for (int r = 0; r < T::RS; ++r) {
      const int row = row_base + r * 16 + fr;
      float f[4];
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        if constexpr (EB == 1) f[v] = int8_out(acc[r][c][v], smSa[row], smSb[col + v], g.bias, smBias[col + v], g.topk_w, smW[row]);
        else f[v] = acc[r][c][v];
      }
      v2u pk = {pack2<FP16>(f[0], f[1]), pack2<FP16>(f[2], f[3])};
      *reinterpret_cast<v2u*>(out + row * TN + (((col >> 3) ^ (row & ROT)) << 3) + (col & 7)) = pk;
    }
  }
  __syncthreads();
  for (int c = tid; c < nvalid * CH; c += T::THREADS) {
    const int row = c / CH, cc = c % CH;
    const int64_t j = j0 + cc * 8;
    if (j >= g.J) continue;
    const int64_t orow = WEIGHTS ? (int64_t)e * g.Cn + i0 + row : (int64_t)smSlot[row];
    if (!WEIGHTS && orow < 0) continue;  // padding before a slot
    const v4i v = *reinterpret_cast<const v4i*>(out + row * TN + ((cc ^ (row & ROT)) << 3));
    v4i* const to = reinterpret_cast<v4i*>(g.C + (orow * g.ldc + j) * 2);
    // nothing reads the weights' gradient soon: past the L2 it takes 3-5 % less
    if constexpr (WEIGHTS) __builtin_nontemporal_store(v, to);
    else *to = v;
  }
}

template <class OP, bool FP16, int FORM, class T>
__global__ __launch_bounds__(T::THREADS) __attribute__((amdgpu_waves_per_eu(T::WPE, T::WPE))) void tile_mm_kernel(MmArgs g) {
  constexpr int TM = T::TM, TN = T::TN;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int tid = threadIdx.x;
  if constexpr (by_weights(FORM)) {
    // The experts' tiles go in groups of four row tiles with all column tiles, and
    // in chunks to the XCDs in turn: a chunk's tiles share an L2, and an expert with
    // many slots, whose tiles are the long ones, is spread over the chip.
    constexpr int kGroup = 4, kChunk = kWgradChunk;
    const int64_t nt = (g.Cn + TM - 1) / TM, per_e = nt * g.n_jt, total = per_e * g.E;
    const int64_t x = blockIdx.x % 8, l = blockIdx.x / 8;
    const int64_t t = (l / kChunk * 8 + x) * kChunk + l % kChunk;
    if (t >= total) return;
    const int e = (int)(t / per_e);
    const int64_t in = t % per_e, ig = in / (kGroup * g.n_jt) * kGroup;
    const int64_t w = nt - ig < kGroup ? nt - ig : kGroup, at = in - ig * g.n_jt;
    const int64_t i0 = (ig + at % w) * TM, j0 = at / w * TN;
    const Run r = FORM == kWgradDense ? Run{0, g.S} : run_of(g, e);
    mm_tile<OP, FP16, FORM, T, T>(g, smem, r.pos0, i0, j0, 0, e, (int)(g.Cn - i0 < TM ? g.Cn - i0 : TM), r.count);
  } else {
    // An expert's last block of up to kShort rows takes a shorter tile with a deeper
    // ring; alone on its CU it waits for its weights (50-60 GB/s) as long as a whole
    // tile takes, so that several workgroups share it where the launch has few rounds.
    constexpr int kShort = TM == 256 && TN == 256 ? 64 : 0;
    int32_t* smSlot = reinterpret_cast<int32_t*>(smem);
    int64_t pos0, j;
    int e, nvalid = 0, part = 0;
    const bool planned = TM == 256 && g.table;
    if (planned) {
      if constexpr (TM == 256)
        if (!table_tile<TM, kShort>(g, pos0, j, e, nvalid, part)) return;
    } else {
      int64_t b;
      if (!rows_tile<TM == 256>(g, b, j)) return;
      pos0 = b * TM;
      e = g.eids ? g.eids[b] : 0;
    }
    const int64_t j0 = j * out_columns(FORM, TN);
    const int rows = planned ? nvalid : !g.eids && pos0 + TM > g.S ? (int)(g.S - pos0) : TM;
    // the rows' slots, their scales and factors, for their addresses and the results
    bool valid = false;
    static_assert(TM <= T::THREADS, "a thread a row");
    if (tid < TM) {
      const uint32_t slot = tid >= rows ? (uint32_t)g.S : g.sorted ? (uint32_t)g.sorted[pos0 + tid] : (uint32_t)(pos0 + tid);
      valid = slot < g.S;
      smSlot[tid] = valid ? (int)slot : -1;
      if constexpr (OP::BYTES == 1) {
        reinterpret_cast<float*>(smSlot)[TM + tid] = valid ? g.As[g.a_by_pos ? pos0 + tid : slot_row(g, slot)] : 0.0f;
        reinterpret_cast<float*>(smSlot)[2 * TM + tid] = valid && g.topk_w ? g.topk_w[slot] : 1.0f;
      }
    }
    if constexpr (OP::BYTES == 1) {
      float* cols = reinterpret_cast<float*>(smSlot) + 3 * TM;
      for (int c = tid; c < TN; c += T::THREADS) {
        const int64_t jj = j0 + c < g.J ? j0 + c : g.J - 1;
        cols[c] = e >= 0 && e < g.E ? g.Bs[(int64_t)e * g.J + jj] : 0.0f;
        cols[TN + c] = g.bias ? from16<FP16>(g.bias[jj]) : 0.0f;
      }
    }
    nvalid = end_of<TM>(valid);
    if (nvalid == 0) return;
    if (e < 0 || e >= g.E) {  // no expert: zero rows
      if constexpr (FORM == kGated) return;  // nothing reads the row
      if constexpr (FORM == kActGrad) {      // but the sum over the parts
        const int64_t n_parts = (g.J + 31) / 32;
        if (g.parts) {
          for (int c = tid; c < nvalid * (TN / 32); c += T::THREADS) {
            const int64_t at = j0 / 32 + c % (TN / 32);
            const int slot = smSlot[c / (TN / 32)];
            if (slot >= 0 && at < n_parts) g.parts[(int64_t)slot * n_parts + at] = 0.0f;
          }
        }
        return;
      }
      for (int c = tid; c < nvalid * (TN / 8); c += T::THREADS) {
        const int64_t jj = j0 + c % (TN / 8) * 8;
        const int slot = smSlot[c / (TN / 8)];
        if (jj >= g.J || slot < 0) continue;
        const int64_t at = (int64_t)slot * g.ldc + jj;
        if (FORM == kRows32 || (FORM == kDgrad && g.out32)) {
          v4f* to = reinterpret_cast<v4f*>(reinterpret_cast<float*>(g.C) + at);
          to[0] = to[1] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
        } else {
          *reinterpret_cast<v4i*>(g.C + at * 2) = (v4i){0, 0, 0, 0};
        }
      }
      return;
    }
    if constexpr (kShort > 0) {
      if (nvalid <= kShort) {
        if (planned && g.short_parts == 4) {
          constexpr int kPart = out_columns(FORM, 64);
          if (j0 + part * kPart < g.J)
            mm_tile<OP, FP16, FORM, T, MmTile<64, 64, 8, 4, 6, 1>>(g, smem, pos0, 0, j0 + part * kPart, part * 64, e, nvalid, g.Cn);
        } else {
          mm_tile<OP, FP16, FORM, T, MmTile<64, 256, 8, 1, 3, 1>>(g, smem, pos0, 0, j0, 0, e, nvalid, g.Cn);
        }
        return;
      }
    }
    mm_tile<OP, FP16, FORM, T, T>(g, smem, pos0, 0, j0, 0, e, nvalid, g.Cn);
  }
}

}  // namespace moe
