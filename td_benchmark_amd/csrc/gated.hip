// The gated feed-forward block in 16-bit floats with its gradients, dense or by
// experts.  Slot s of token t(s) = s / top_k, expert e(s), router's weight w_s (1
// without):
//   G = x_t Wg_e^T, U = x_t Wu_e^T           w13_e = [Wg; Wu], fp32 sums, kept in fp32
//   h_s = round16(w_s silu(G) U)             silu(z) = z s(z), s(z) = 1 / (1 + exp(-z))
//   y_t = round16(sum_s h_s W2_e^T)          fp32 rows, fp32 sum
// and with D_s = dy_t W2_e (fp32):
//   dw_s = sum_i D silu(G) U,  dU = w_s D silu(G),  dG = w_s D U (s + silu(G) (1 - s))
//   dx_t = round16(sum_s [dG dU]_s W13_e)    [dG dU] rounded to 16 bits
//   dW13_e = sum_s [dG dU]_s^T x_t,  dW2_e = sum_s dy_t^T h_s
// The router's weight goes into h, where there is a rounding anyway: no slot's
// output row is kept for its gradient.  h and [dG dU] are rounded because the
// matrix instructions take 16 bits; G and U are kept in fp32, which costs 8 I bytes
// more a slot than in 16 bits (3 % of a training step) and leaves the gradient of
// the router's weights, an fp32 value, as exact as its sums.
//
// Launches: the product of both projections with the activation in its epilogue (the
// tile's columns pair 16 of the gate with 16 of the up projection), the product of h,
// and with several slots a token the sum of their rows; backward the product of dy with
// the activation's gradient and dw's parts in its epilogue, the product by rows, and the
// two gradients by weights.  With the activation in kernels of its own over fp32 rows a
// prompt of 4093 tokens of 8 on 64 experts took 978 us for 911.
//
// What bounds it (us, least and median of a trace): one token, 7168 x 2048, the weights'
// stream, 12.4, 12.9 and 6.9, 7.2 (4.7 and 4.3 TB/s); 4096 tokens of one expert the matrix
// cores at the board's power (1381 W of 1400), 182, 107, 121, 198, 208, 119 for the six
// products, at the median 200, 118, 132, 225, 228, 128, 0.91 to 1.32 PF; 128 experts of 240
// slots, 2048 x 768, the weights, their gradients and the fp32 rows, by the counters 4.6 GB
// read and 2.1 written a step, 4.2 TB/s of the kernels' time.
#include "grouped_launch.hpp"

namespace moe {

static int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }
static int64_t up_to_256(int64_t n) { return (n + 255) / 256 * 256; }

// ---- the gradient of the router's weights -------------------------------------------
// dweight[s] = the sum of the slot's n parts: a wave a slot at a time, lanes in order.
// A launch has fewer than 2^32 threads: past kPartSumGrid workgroups (4 million slots)
// each goes through several slots a wave.
constexpr int64_t kPartSumGrid = 1 << 20;

__global__ __launch_bounds__(256) void part_sum_kernel(const float* __restrict__ parts, int64_t S, int64_t n, float* __restrict__ dweight) {
  for (int64_t s = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); s < S; s += (int64_t)gridDim.x * 4) {
    float sum = 0.0f;
    for (int64_t i = threadIdx.x & 63; i < n; i += 64) sum += parts[s * n + i];
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if ((threadIdx.x & 63) == 0) dweight[s] = sum;
  }
}
static int launch_part_sum(const float* parts, int64_t S, int64_t n, float* dweight, hipStream_t st) {
  const int64_t groups = (S + 3) / 4;
  hipLaunchKernelGGL(part_sum_kernel, dim3((unsigned)(groups < kPartSumGrid ? groups : kPartSumGrid)), dim3(256), 0, st, parts, S, n, dweight);
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

// ---- rows that are not whole 16-byte chunks --------------------------------------
// dst [B][rows_d][cols_d] = src [B][rows_s][cols_s] with zeros past its ends, or its
// first rows and columns: widths that the products cannot take are copied to whole
// chunks and their results back, all of a pass's operands in one launch.  A wave a row,
// 8 columns a lane: the odd side goes element by element, the other in 16-byte chunks.
struct Copy {
  const uint16_t* src;
  uint16_t* dst;
  int64_t B, rows_s, cols_s, ld_s, batch_s, rows_d, cols_d, ld_d, batch_d;
};
struct Copies {
  Copy c[4];
  int64_t first[5];  // rows of the copies before each
  int n = 0;
  void add(const Copy& x) {
    if (n == 0) first[0] = 0;
    c[n] = x;
    first[n + 1] = first[n] + x.B * x.rows_d;
    ++n;
  }
};
__global__ __launch_bounds__(256) void copy_kernel(Copies all) {
  const int lane = threadIdx.x & 63;
  const int64_t rows = all.first[all.n];
  for (int64_t r0 = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); r0 < rows; r0 += (int64_t)gridDim.x * 4) {
    int i = 0;
    while (i + 1 < all.n && r0 >= all.first[i + 1]) ++i;
    const Copy& c = all.c[i];
    const int64_t r = r0 - all.first[i], b = r / c.rows_d, row = r - b * c.rows_d;
    const uint16_t* src = c.src + b * c.batch_s + row * c.ld_s;
    uint16_t* dst = c.dst + b * c.batch_d + row * c.ld_d;
    const int64_t end = row < c.rows_s ? c.cols_s : 0;  // columns of the row that there are
    const bool from16 = ((uintptr_t)src & 15) == 0, to16 = ((uintptr_t)dst & 15) == 0;
    for (int64_t col = lane * 8; col < c.cols_d; col += 512) {
      uint32_t v[4] = {};
      if (from16 && col + 8 <= end) {
        const v4i x = *reinterpret_cast<const v4i*>(src + col);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = (uint32_t)x[k];
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (col + k < end) v[k / 2] |= (uint32_t)src[col + k] << (16 * (k & 1));
      }
      if (to16 && col + 8 <= c.cols_d) {
        *reinterpret_cast<v4i*>(dst + col) = (v4i){(int)v[0], (int)v[1], (int)v[2], (int)v[3]};
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (col + k < c.cols_d) dst[col + k] = (uint16_t)(v[k / 2] >> (16 * (k & 1)));
      }
    }
  }
}
static int launch_copies(const Copies& c, hipStream_t st) {
  if (c.n == 0 || c.first[c.n] == 0) return kOk;
  const int64_t groups = (c.first[c.n] + 3) / 4;
  hipLaunchKernelGGL(copy_kernel, dim3((unsigned)(groups < 2048 ? groups : 2048)), dim3(256), 0, st, c);
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

// ---- the block ---------------------------------------------------------------------
static int check_ffn(const moe_ffn& f) {
  if (f.T < 0 || f.H < 1 || f.I < 1 || f.H > (1 << 29) || f.I > (1 << 28) || f.ldx < f.H || f.ldx > (1 << 29)) return kErrBadShape;
  if (f.dtype != kBf16 && f.dtype != kFp16) return kErrBadShape;
  if (f.top_k < 1) return kErrBadTopK;
  if (f.E < 1) return kErrBadExperts;
  if (f.T > 0x7FFFFFFE / f.top_k || f.max_padded < 0 || f.max_padded > 0x7FFFFFFF) return kErrBadShape;
  if (f.E > ((int64_t)1 << 58) / (up8(f.H) * up8(f.I))) return kErrBadShape;  // the weights' bytes, below 2^61
  if (!f.sorted_ids && !f.expert_ids && !f.ntpp) {
    if (f.E != 1 || f.top_k != 1) return kErrBadExperts;
  } else {
    if (!f.sorted_ids || !f.expert_ids || !f.ntpp) return kErrNullPointer;
    if (!block_m_ok(f.block_size_m)) return kErrBadBlockSize;
    if (f.T > 0 && f.max_padded < f.block_size_m) return kErrBadShape;  // slots, but no block for them
  }
  return kOk;
}

// Sizes and places of one pass.
struct Ffn {
  const moe_ffn& f;
  int64_t S, Hp, Ip;
  bool dense, odd;  // odd: widths that are padded
  hipStream_t st;
  explicit Ffn(const moe_ffn& l, void* stream = nullptr)
      : f(l), S(l.T * l.top_k), Hp(up8(l.H)), Ip(up8(l.I)), dense(!l.sorted_ids), odd(Hp != l.H || Ip != l.I),
        st((hipStream_t)stream) {}
  bool copy_x() const { return Hp != f.H || !chunks(f.x, f.ldx, 2); }
  bool copy_w(const void* w) const { return odd || !aligned(w, 16); }
  int64_t x_bytes() const { return up_to_256(2 * f.T * Hp); }
  int64_t w13_bytes() const { return up_to_256(4 * f.E * Ip * Hp); }
  int64_t w2_bytes() const { return up_to_256(2 * f.E * Ip * Hp); }
  int64_t rows_bytes() const { return f.top_k > 1 ? up_to_256(4 * S * Hp) : 0; }

  Copy pad_rows(const void* x, int64_t ldx, void* to) const {
    return {(const uint16_t*)x, (uint16_t*)to, 1, f.T, f.H, ldx, 0, f.T, Hp, Hp, 0};
  }
  Copy pad_w13(const void* w, void* to) const {
    return {(const uint16_t*)w, (uint16_t*)to, 2 * f.E, f.I, f.H, f.H, f.I * f.H, Ip, Hp, Hp, Ip * Hp};
  }
  Copy pad_w2(const void* w, void* to) const {
    return {(const uint16_t*)w, (uint16_t*)to, f.E, f.H, f.I, f.I, f.H * f.I, Hp, Ip, Ip, Hp * Ip};
  }
  Copy crop_rows(const void* y, void* to) const {
    return {(const uint16_t*)y, (uint16_t*)to, 1, f.T, f.H, Hp, 0, f.T, f.H, f.H, 0};
  }
  Copy crop_w13(const void* w, void* to) const {
    return {(const uint16_t*)w, (uint16_t*)to, 2 * f.E, f.I, f.H, Hp, Ip * Hp, f.I, f.H, f.H, f.I * f.H};
  }
  Copy crop_w2(const void* w, void* to) const {
    return {(const uint16_t*)w, (uint16_t*)to, f.E, f.H, f.I, Ip, Hp * Ip, f.H, f.I, f.I, f.H * f.I};
  }

  // A product over the slots, of J columns.
  MmArgs args(int64_t J) const {
    MmArgs g{};
    g.S = S;
    g.J = J;
    g.E = f.E;
    if (dense) {
      g.bm = dense_rows(S, J);
      g.n_blocks = (S + g.bm - 1) / g.bm;
    } else {
      const bool any = f.max_padded > 0;
      g.sorted = f.sorted_ids;
      g.eids = f.expert_ids;
      g.ntpp = any ? f.ntpp : nullptr;
      g.table = any ? f.expert_table : nullptr;
      g.bm = f.block_size_m;
      g.n_blocks = f.max_padded / f.block_size_m;
    }
    return g;
  }
  template <int FORM>
  int rows(const MmArgs& g) const {
    return f.dtype == kFp16 ? launch_rows<Fp16, true, FORM>(g, st) : launch_rows<Bf16, false, FORM>(g, st);
  }
  // out rows [S] = A's rows (a row for each `per` slots) times B [E][J][Cn] along its rows, or with `columns` [E][Cn][J]
  // along its columns; fp32 rows with out32.
  int product(const void* A, int64_t lda, int per, const void* B, int64_t J, int64_t Cn, bool columns, bool out32, void* out) const {
    MmArgs g = args(J);
    g.A = (const uint8_t*)A;
    g.B = (const uint8_t*)B;
    g.C = (uint8_t*)out;
    g.Cn = Cn;
    g.lda = lda;
    g.sbj = columns ? 1 : Cn;
    g.sbc = columns ? J : 1;
    g.b_es = J * Cn;
    g.ldc = J;
    set_top_k(g, per);
    g.out32 = out32 ? 1 : 0;
    if (columns) return tile_dgrad(g, f.dtype, st);
    return out32 ? rows<kRows32>(g) : tile_product(g, f.dtype, st);
  }
  // dw [E][N][J] = A^T B over each expert's slots; by_token: A has the token's row and B the slot's, else the other way.
  int weights(const void* A, int64_t lda, const void* B, int64_t ldb, int64_t N, int64_t J, bool by_token, void* dw) const {
    MmArgs g = args(J);
    g.A = (const uint8_t*)A;
    g.B = (const uint8_t*)B;
    g.C = (uint8_t*)dw;
    g.Cn = N;
    g.lda = lda;
    g.sbc = ldb;
    g.ldc = J;
    set_top_k(g, f.top_k);
    if (dense) return launch_weights<kWgradDense>(g, f.dtype, st);
    return by_token ? launch_weights<kWgradTok>(g, f.dtype, st) : tile_wgrad(g, f.dtype, st);
  }
  // Rows of the tokens from rows of the slots.
  int token_rows(const float* rows32, void* out) const { return slot_sum_rows(rows32, Hp, f.T, f.top_k, f.H, f.dtype, out, st); }
};

// Parts of a workspace in order, each of up to 2^62 bytes; past kMost together they do not fit.
struct Parts {
  static constexpr int64_t kMost = (int64_t)1 << 61;
  uint8_t* base;
  int64_t at = 0;
  void* take(int64_t bytes, bool on = true) {
    if (!on || at > kMost) return nullptr;
    uint8_t* p = base ? base + at : nullptr;
    at += up_to_256(bytes);
    return p;
  }
};

// A pass's workspace.  Last come the copies of y, or of dx and dy, for addresses or widths
// that are not of whole 16-byte chunks: where there is neither, their room is not needed.
struct Forward {
  void *x, *w13, *w2, *rows, *y;
  Forward(const Ffn& b, Parts& p, bool aligned_y) {
    x = p.take(b.x_bytes(), b.copy_x());
    w13 = p.take(b.w13_bytes(), b.copy_w(b.f.w13));
    w2 = p.take(b.w2_bytes(), b.copy_w(b.f.w2));
    rows = p.take(b.rows_bytes(), b.f.top_k > 1);
    y = p.take(b.x_bytes(), b.f.top_k == 1 && (b.Hp != b.f.H || !aligned_y));
  }
};
struct Backward {
  void *x, *w13, *w2, *parts, *dgu, *rows, *dw13, *dw2, *dx, *dy;
  Backward(const Ffn& b, Parts& p, bool aligned_dx, bool aligned_dy) {
    x = p.take(b.x_bytes(), b.copy_x());
    w13 = p.take(b.w13_bytes(), b.copy_w(b.f.w13));
    w2 = p.take(b.w2_bytes(), b.copy_w(b.f.w2));
    parts = p.take(4 * b.S * ((b.Ip + 31) / 32), b.f.topk_weights);
    dgu = p.take(4 * b.S * b.Ip);
    rows = p.take(b.rows_bytes(), b.f.top_k > 1);
    dw13 = p.take(b.w13_bytes(), b.odd);
    dw2 = p.take(b.w2_bytes(), b.odd);
    dx = p.take(b.x_bytes(), b.f.top_k == 1 && (b.Hp != b.f.H || !aligned_dx));
    dy = p.take(b.x_bytes(), b.Hp != b.f.H || !aligned_dy);
  }
};

#define MOE_TRY(call)              \
  do {                             \
    const int rc_ = (call);        \
    if (rc_ != kOk) return rc_;    \
  } while (0)

static int ffn_forward(const Ffn& b, void* y) {
  const moe_ffn& f = b.f;
  Parts parts{(uint8_t*)f.workspace};
  const Forward ws(b, parts, aligned(y, 16));
  if (!f.workspace && parts.at > 0) return kErrNullPointer;
  const void *x = f.x, *w13 = f.w13, *w2 = f.w2;
  int64_t ldx = f.ldx;
  Copies in;
  if (ws.x) {
    in.add(b.pad_rows(x, ldx, ws.x));
    x = ws.x;
    ldx = b.Hp;
  }
  if (ws.w13) {
    in.add(b.pad_w13(w13, ws.w13));
    w13 = ws.w13;
  }
  if (ws.w2) {
    in.add(b.pad_w2(w2, ws.w2));
    w2 = ws.w2;
  }
  MOE_TRY(launch_copies(in, b.st));
  MmArgs g = b.args(b.Ip);
  g.J_used = f.I;
  g.A = (const uint8_t*)x;
  g.B = (const uint8_t*)w13;
  g.C = (uint8_t*)f.h;
  g.gu = f.gu;
  g.topk_w = f.topk_weights;
  g.Cn = b.Hp;
  g.lda = ldx;
  g.sbj = b.Hp;
  g.sbc = 1;
  g.b_es = 2 * b.Ip * b.Hp;
  g.ldc = b.Ip;
  set_top_k(g, f.top_k);
  MOE_TRY(b.rows<kGated>(g));
  if (f.top_k > 1) {
    MOE_TRY(b.product(f.h, b.Ip, 1, w2, b.Hp, b.Ip, false, true, ws.rows));
    return b.token_rows((const float*)ws.rows, y);
  }
  MOE_TRY(b.product(f.h, b.Ip, 1, w2, b.Hp, b.Ip, false, false, ws.y ? ws.y : y));
  if (!ws.y) return kOk;
  Copies out;
  out.add(b.crop_rows(ws.y, y));
  return launch_copies(out, b.st);
}

static int ffn_backward(const Ffn& b, const void* dy, void* dx, void* dw13, void* dw2, float* dweight) {
  const moe_ffn& f = b.f;
  Parts parts{(uint8_t*)f.workspace};
  const Backward ws(b, parts, aligned(dx, 16), aligned(dy, 16));
  if (!f.workspace && parts.at > 0) return kErrNullPointer;
  const void *x = f.x, *w13 = f.w13, *w2 = f.w2;
  int64_t ldx = f.ldx;
  const bool rows = dx || dw13 || dweight;  // whether the gradient of the projections is needed
  Copies in, out;
  if (ws.dy) {
    in.add(b.pad_rows(dy, f.H, ws.dy));
    dy = ws.dy;
  }
  if (ws.x && dw13) {
    in.add(b.pad_rows(x, ldx, ws.x));
    x = ws.x;
    ldx = b.Hp;
  }
  if (ws.w2 && rows) {
    in.add(b.pad_w2(w2, ws.w2));
    w2 = ws.w2;
  }
  if (ws.w13 && dx) {
    in.add(b.pad_w13(w13, ws.w13));
    w13 = ws.w13;
  }
  MOE_TRY(launch_copies(in, b.st));
  if (rows) {
    if (b.S > 0) {
      MmArgs g = b.args(b.Ip);
      g.J_used = f.I;
      g.A = (const uint8_t*)dy;
      g.B = (const uint8_t*)w2;
      g.C = (uint8_t*)ws.dgu;
      g.gu = f.gu;
      g.parts = dweight ? (float*)ws.parts : nullptr;
      g.topk_w = f.topk_weights;
      g.Cn = b.Hp;
      g.lda = b.Hp;
      g.sbj = 1;
      g.sbc = b.Ip;
      g.b_es = b.Hp * b.Ip;
      g.ldc = 2 * b.Ip;
      set_top_k(g, f.top_k);
      MOE_TRY(b.rows<kActGrad>(g));
      if (dweight) MOE_TRY(launch_part_sum((const float*)ws.parts, b.S, (b.Ip + 31) / 32, dweight, b.st));
    }
  }
  if (dx && b.S > 0) {
    if (f.top_k > 1) {
      MOE_TRY(b.product(ws.dgu, 2 * b.Ip, 1, w13, b.Hp, 2 * b.Ip, true, true, ws.rows));
      MOE_TRY(b.token_rows((const float*)ws.rows, dx));
    } else {
      MOE_TRY(b.product(ws.dgu, 2 * b.Ip, 1, w13, b.Hp, 2 * b.Ip, true, false, ws.dx ? ws.dx : dx));
      if (ws.dx) out.add(b.crop_rows(ws.dx, dx));
    }
  }
  if (dw13) {
    MOE_TRY(b.weights(ws.dgu, 2 * b.Ip, x, ldx, 2 * b.Ip, b.Hp, false, b.odd ? ws.dw13 : dw13));
    if (b.odd) out.add(b.crop_w13(ws.dw13, dw13));
  }
  if (dw2) {
    MOE_TRY(b.weights(dy, b.Hp, f.h, b.Ip, b.Hp, b.Ip, true, b.odd ? ws.dw2 : dw2));
    if (b.odd) out.add(b.crop_w2(ws.dw2, dw2));
  }
  return launch_copies(out, b.st);
}

}  // namespace moe

using namespace moe;

extern "C" int64_t moe_ffn_workspace_bytes(const moe_ffn* f, int32_t pass) {
  if (!f) return kErrNullPointer;
  const int rc = check_ffn(*f);
  if (rc != kOk) return rc;
  Parts p{nullptr};
  const Ffn b(*f);
  const bool whole = pass == MOE_FFN_ALIGNED || pass == (MOE_FFN_BACKWARD | MOE_FFN_ALIGNED);
  if (pass != 0 && pass != MOE_FFN_ALIGNED) Backward(b, p, whole, whole);
  else Forward(b, p, whole);
  return p.at > Parts::kMost ? kErrBadShape : p.at;
}

static int check_pointers(const moe_ffn& f, bool backward, bool need_gu = false) {
  if (f.T == 0 && !backward) return kOk;
  if ((f.T > 0 && (!f.x || !f.h || (need_gu && !f.gu))) || !f.w13 || !f.w2) return kErrNullPointer;
  if (!aligned(f.x, 2) || !aligned(f.w13, 2) || !aligned(f.w2, 2) || !aligned(f.topk_weights, 4) || !aligned(f.h, 16) ||
      !aligned(f.gu, 16) || !aligned(f.workspace, 16))
    return kErrBadShape;
  const int64_t work = moe_ffn_workspace_bytes(&f, backward ? MOE_FFN_BACKWARD : 0);
  return work < 0 ? (int)work : kOk;
}

extern "C" int moe_ffn_forward(const moe_ffn* f, void* y, void* stream) {
  if (!f) return kErrNullPointer;
  MOE_TRY(check_ffn(*f));
  MOE_TRY(check_pointers(*f, false));
  if (f->T == 0) return kOk;
  if (!y) return kErrNullPointer;
  if (!aligned(y, 2)) return kErrBadShape;
  return ffn_forward(Ffn(*f, stream), y);
}

extern "C" int moe_ffn_backward(const moe_ffn* f, const void* dy, void* dx, void* dw13, void* dw2, float* dtopk_weights,
                                void* stream) {
  if (!f) return kErrNullPointer;
  MOE_TRY(check_ffn(*f));
  MOE_TRY(check_pointers(*f, true, dx || dw13 || dtopk_weights));
  if ((f->T > 0 && !dy) || (dtopk_weights && !f->topk_weights)) return kErrNullPointer;
  if (!aligned(dy, 2) || !aligned(dx, 2) || !aligned(dw13, 2) || !aligned(dw2, 2) || !aligned(dtopk_weights, 4)) return kErrBadShape;
  const Ffn b(*f, stream);
  if (!b.odd && (!aligned(dw13, 16) || !aligned(dw2, 16))) return kErrBadShape;  // written where they are
  return ffn_backward(b, dy, dx, dw13, dw2, dtopk_weights);
}
