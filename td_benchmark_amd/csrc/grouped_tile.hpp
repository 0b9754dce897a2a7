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

enum Form { kProduct, kDgrad, kWgrad };

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

MOE_DEVICE void mm_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
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

// One tile: rows [i0, i0 + nvalid) of the output, or the slots of the table's first
// nvalid rows, by columns j0 on (col0 on of the columns' table), over `length` of the
// contraction.  K: the tile of the launch, which T is or is a part of.
template <class OP, bool FP16, int FORM, class K, class T>
MOE_DEVICE void mm_tile(const MmArgs& g, uint8_t* smem, int64_t pos0, int64_t i0, int64_t j0, int col0, int e,
                        int nvalid, int64_t length) {
  constexpr int EB = OP::BYTES, TM = T::TM, TN = T::TN, KS = T::KS, SB = T::SB;
  constexpr bool A_COLS = FORM == kWgrad, B_COLS = FORM != kProduct;
  constexpr int STEP = SB / EB;  // contraction elements of a step
  static_assert(EB == 2 || FORM == kProduct, "transposing reads are of 16-bit values");
  static_assert(FORM != kWgrad || (KS <= 4 && 8 * STEP * 4 <= K::TABLE), "the ring of slots");
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

  // ---- addresses of this lane's part of the loads ----
  // Instruction i of a wave is load wave + NW i of its operand.
  const uint8_t* a_ptr[T::NA_W];
  const uint8_t* b_ptr[T::NB_W];
  constexpr int ACPR = TM / 8, BCPR = TN / 8;  // chunks of a column-staged row
  const uint8_t* b_base = g.B + (FORM == kWgrad ? 0 : (int64_t)e * g.b_es * EB);
  const uint8_t* zeros = reinterpret_cast<const uint8_t*>(&kZeroChunk);
  constexpr int LPR = SB / 16, RPI = 64 / LPR;  // lanes of a row, rows of a load
  auto row_chunk = [&](int gi) { return row_place<SB>(lane % LPR, RPI * gi + lane / LPR); };
  // contraction row and column chunk of a column-staged load
  auto col_row = [&](int gi, int cpr) { return gi * (64 / cpr) + lane / cpr; };
  auto col_of = [&](int gi, int cpr) { return ((lane % cpr) ^ (col_swz<SB>(col_row(gi, cpr)) & (cpr - 1))) * 8; };
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
      a_ptr[i] = g.A + ar * g.lda * EB + row_chunk(gi) * 16;
    }
  }
#pragma unroll
  for (int i = 0; i < T::NB_W; ++i) {
    const int gi = wave + T::NW * i;
    if constexpr (B_COLS) {
      const int64_t c = j0 + col_of(gi, BCPR);
      b_ptr[i] = b_base + (c < g.J ? c : 0) * EB;
      if constexpr (FORM == kDgrad) b_ptr[i] += (int64_t)col_row(gi, BCPR) * g.sbc * EB;
    } else {
      const int64_t j = j0 + RPI * gi + lane / LPR;
      b_ptr[i] = b_base + (j < g.J ? j : g.J - 1) * g.sbj * EB + row_chunk(gi) * 16;
    }
  }
  // Rows of A in subtiles without a slot are not fetched where every step waits for all of its loads.
  const int a_rows = KS == 2 ? (nvalid + 15) / 16 * 16 : TM;

  // kWgrad: the slots of this lane's rows of a step, read ahead of its loads; square
  // tiles place both operands alike
  uint32_t slot_a[T::NA_W], slot_b[T::NB_W];
  auto read_slots = [&](int kk) {
#pragma unroll
    for (int i = 0; i < T::NA_W; ++i)
      slot_a[i] = (uint32_t)smSlot[(kk & 7) * STEP + col_row(wave + T::NW * i, ACPR)];
#pragma unroll
    for (int i = 0; i < T::NB_W; ++i)
      slot_b[i] = TM == TN ? slot_a[i < T::NA_W ? i : 0] : (uint32_t)smSlot[(kk & 7) * STEP + col_row(wave + T::NW * i, BCPR)];
  };

  // Load d of this wave's share of step kk into its stage.  Step 0 is the last,
  // partial run of the contraction, so that no other step has to look for its
  // end; the addresses of the others advance from load to load.
  const int tail = (int)(length - (int64_t)(KB - 1) * STEP);  // elements of step 0
  const int64_t b_step = FORM == kDgrad ? STEP * g.sbc * EB : SB;
  constexpr int ND = T::NA_W + T::NB_W;
  auto load = [&](int kk, int stage, auto dc, auto first_c) {
    constexpr int d = decltype(dc)::value;
    constexpr bool first = decltype(first_c)::value;
    const uint32_t dst = lds0 + stage * T::STAGE;
    const int left = first ? tail : STEP;
    constexpr bool is_b = d < T::NB_W;
    constexpr int i = is_b ? d : d - T::NB_W;
    const int gi = wave + T::NW * i;
    if constexpr (FORM == kWgrad) {
      const uint8_t* p;
      if constexpr (is_b) p = b_ptr[i] + (uint64_t)slot_row(g, slot_b[i]) * (uint32_t)(g.sbc * EB);
      else p = a_ptr[i] + (uint64_t)slot_a[i] * (uint32_t)(g.lda * EB);
      if constexpr (first) p = col_row(gi, is_b ? BCPR : ACPR) < left ? p : zeros;
      if ((is_b ? T::NB : T::NA) % T::NW == 0 || gi < (is_b ? T::NB : T::NA))
        lds_load16(p, dst + (is_b ? T::A_BYTES : 0) + gi * 1024);
    } else if constexpr (is_b) {
      const uint8_t* p = b_ptr[i];
      if constexpr (first) {
        p += (KB - 1) * b_step;
        const bool in = FORM == kDgrad ? col_row(gi, BCPR) < left : row_chunk(gi) * 16 < left * EB;
        p = in ? p : zeros;
      } else {
        b_ptr[i] += b_step;
      }
      if (T::NB % T::NW == 0 || gi < T::NB) lds_load16(p, dst + T::A_BYTES + gi * 1024);
    } else {
      const uint8_t* p = a_ptr[i];
      if constexpr (first) {
        p += (int64_t)(KB - 1) * SB;
        p = row_chunk(gi) * 16 < left * EB ? p : zeros;
      } else {
        a_ptr[i] += SB;
      }
      if ((T::NA % T::NW == 0 || gi < T::NA) && RPI * gi < a_rows) lds_load16(p, dst + gi * 1024);
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
      const int64_t c0 = kk == 0 ? (int64_t)(KB - 1) * STEP : (int64_t)(kk - 1) * STEP;
      const int64_t c = c0 + lane < length ? c0 + lane : length - 1;
      lds_load4(g.sorted + pos0 + c, (uint32_t)(uintptr_t)(lds_ptr)smem + (kk & 7) * STEP * 4);
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
  const uint32_t b_lane = T::A_BYTES + (B_COLS ? by_col(col_base, TN) : col_base * SB + by_row);

  typename OP::Acc acc[T::RS][T::CS] = {};
  int ra = (nvalid - row_base + 15) / 16;
  ra = ra < 0 ? 0 : (ra > T::RS ? T::RS : ra);

  if constexpr (FORM == kWgrad) {
    if (KB > 0) {
      for (int s = 0; s < KS + kAhead; ++s) issue_ids(s);
      mm_wait<0>();
    }
    __syncthreads();
  }
  const std::integral_constant<int, 0> none;
  const std::integral_constant<int, ND> all;
  if constexpr (FORM == kWgrad) read_slots(0);
  if (KB > 0) loads(0, 0, none, all, std::true_type{});
#pragma unroll
  for (int s = 1; s < KS; ++s) {
    if constexpr (FORM == kWgrad) read_slots(s);
    if (s < KB) loads(s, s, none, all, std::false_type{});
  }

  // A step is H CS slots of RS matrix instructions, one weight fragment each, which
  // is read two slots ahead.  The barrier that hands over the next stage stands two
  // slots before the step's end, when every fragment of this stage has been read:
  // the last two slots' instructions cover the reads of the next stage's first
  // fragments, and this stage's buffer is filled again from there on, a load a slot.
  constexpr int NQ = T::H * T::CS;
  constexpr int DPQ = (ND + NQ - 1) / NQ;  // loads of a slot
  static_assert(NQ >= 4 && NQ % 4 == 0, "four fragment registers in turn");
  auto kloop = [&](auto ra_c) {
    constexpr int RA = decltype(ra_c)::value;
    if (KB == 0) return;
    v4i af[2][RA > 0 ? RA : 1], bf[4];
    auto read_a = [&](int to, int stage, int h, int r) {
      const uint32_t st = lds0 + stage * T::STAGE;
      if constexpr (A_COLS) af[to][r] = lds_frag_t(st + (a_lane ^ (r * 32)) + h * 8 * TM * 2, TM * 2);
      else af[to][r] = lds_frag(st + (a_lane ^ (h * 16)) + r * 16 * SB);
    };
    auto read_b = [&](int stage, int q) {
      const uint32_t st = lds0 + stage * T::STAGE;
      const int h = q / T::CS, c = q % T::CS;
      if constexpr (B_COLS) bf[q & 3] = lds_frag_t(st + (b_lane ^ (c * 32)) + h * 8 * TN * 2, TN * 2);
      else bf[q & 3] = lds_frag(st + (b_lane ^ (h * 16)) + c * 16 * SB);
    };
    // stage 0; of the others every wave has at least so many loads behind it
    mm_wait_stages<KS - 1, KS == 2 ? T::NB / T::NW : T::VM>(KB - 1);
    mm_barrier();
    if constexpr (RA > 0) {
#pragma unroll
      for (int r = 0; r < RA; ++r) read_a(0, 0, 0, r);
      read_b(0, 0);
      read_b(0, 1);
    }
    int stage = 0;
    // P: with one instruction a step, which of the two sets of row fragments it takes
    auto step = [&](int kk, auto pc) {
      constexpr int P = decltype(pc)::value;
      const int next = stage == KS - 1 ? 0 : stage + 1, prev = stage == 0 ? KS - 1 : stage - 1;
      auto slot = [&](auto qc) {
        constexpr int Q = decltype(qc)::value;
        if constexpr (Q == NQ - 2) {
          if (kk + 1 < KB) {
            mm_wait_stages<KS - 2, T::VM>(KB - 2 - kk);
            mm_barrier();
            if constexpr (RA > 0) {
#pragma unroll
              for (int r = 0; r < RA; ++r) read_a(T::H == 2 ? 0 : P ^ 1, next, 0, r);
              read_b(next, 0);
              read_b(next, 1);
            }
            if constexpr (FORM == kWgrad) {
              if (kk + KS < KB) {
                read_slots(kk + KS);
                issue_ids(kk + KS + kAhead);
              }
            }
          }
        }
        if constexpr (RA > 0 && Q < NQ - 2) {
          read_b(stage, Q + 2);
          // the second half's rows: one a slot up to two slots ahead, or together
          if constexpr (T::H == 2 && T::CS > RA + 1 && Q + RA >= T::CS - 1 && Q < T::CS - 1) read_a(1, stage, 1, Q + RA - (T::CS - 1));
          if constexpr (T::H == 2 && T::CS <= RA + 1 && Q == 0) {
#pragma unroll
            for (int r = 0; r < RA; ++r) read_a(1, stage, 1, r);
          }
        }
        // loads of stage kk + KS in this step's last two slots, of the stage before it in the others
        constexpr int from = (Q + 2) % NQ * DPQ, to = from + DPQ < ND ? from + DPQ : ND;
        if constexpr (from < ND) {
          const std::integral_constant<int, from> f;
          const std::integral_constant<int, to> t;
          if constexpr (Q >= NQ - 2) {
            if (kk + KS < KB) loads(kk + KS, stage, f, t, std::false_type{});
          } else {
            if (kk > 0 && kk - 1 + KS < KB) loads(kk - 1 + KS, prev, f, t, std::false_type{});
          }
        }
        // the reads stay ahead of the instructions, which the compiler would undo
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (RA > 0) {
          constexpr int at = T::H == 2 ? Q / T::CS : P, c = Q % T::CS;
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
    if constexpr (T::H == 2) {
      for (int kk = 0; kk < KB; ++kk) step(kk, std::integral_constant<int, 0>{});
    } else {
      for (int kk = 0; kk < KB; kk += 2) {
        step(kk, std::integral_constant<int, 0>{});
        if (kk + 1 < KB) step(kk + 1, std::integral_constant<int, 1>{});
      }
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

  if constexpr (FORM == kDgrad) {
    // fp32 rows: 16 rows of the wave's columns a time through its own part of the
    // ring, so that a row's columns leave as one run
    if (g.out32) {
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
    const int64_t orow = FORM == kWgrad ? (int64_t)e * g.Cn + i0 + row : (int64_t)smSlot[row];
    if (FORM != kWgrad && orow < 0) continue;  // padding before a slot
    const v4i v = *reinterpret_cast<const v4i*>(out + row * TN + ((cc ^ (row & ROT)) << 3));
    v4i* const to = reinterpret_cast<v4i*>(g.C + (orow * g.ldc + j) * 2);
    // nothing reads the weights' gradient soon: past the L2 it takes 3-5 % less
    if constexpr (FORM == kWgrad) __builtin_nontemporal_store(v, to);
    else *to = v;
  }
}

template <class OP, bool FP16, int FORM, class T>
__global__ __launch_bounds__(T::THREADS) __attribute__((amdgpu_waves_per_eu(T::WPE, T::WPE))) void tile_mm_kernel(MmArgs g) {
  constexpr int TM = T::TM, TN = T::TN;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int tid = threadIdx.x;
  if constexpr (FORM == kWgrad) {
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
    const Run r = run_of(g, e);
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
    const int64_t j0 = j * TN;
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
      for (int c = tid; c < nvalid * (TN / 8); c += T::THREADS) {
        const int64_t jj = j0 + c % (TN / 8) * 8;
        const int slot = smSlot[c / (TN / 8)];
        if (jj >= g.J || slot < 0) continue;
        const int64_t at = (int64_t)slot * g.ldc + jj;
        if (FORM == kDgrad && g.out32) {
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
          if (j0 + part * 64 < g.J)
            mm_tile<OP, FP16, FORM, T, MmTile<64, 64, 8, 4, 6, 1>>(g, smem, pos0, 0, j0 + part * 64, part * 64, e, nvalid, g.Cn);
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
