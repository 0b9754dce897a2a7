// Test-only: the tiles that the products' launches choose (declared in moe_probe.h),
// by the library's own rules.  Host code alone.
#include "grouped_launch.hpp"
#include "moe_probe.h"

using namespace moe;

extern "C" void moe_probe_rows_choice(int32_t form, int32_t dense, int64_t S, int32_t E, int32_t block_m, int64_t max_padded,
                                      int64_t J, int64_t K, int32_t* out) {
  static const int32_t some = 0;
  MmArgs g{};
  g.S = S;
  g.J = J;
  g.E = E;
  g.bm = dense ? dense_rows(S, J) : block_m;
  g.n_blocks = dense ? (S + g.bm - 1) / g.bm : max_padded / block_m;
  g.eids = dense ? nullptr : &some;
  const TileChoice t = rows_choice(by_columns(form), live_blocks_guess(g), S, g.bm, form == kGated ? 2 * J : J, 2 * K);
  const int64_t columns = out_columns(form, t.columns), n_jt = (J + columns - 1) / columns;
  const bool counts = !dense && t.rows == 256 && by_counts(S, E, n_jt);
  out[0] = t.rows;
  out[1] = t.columns;
  out[2] = t.few;
  out[3] = counts && t.columns == 256 ? short_parts(S, E, n_jt, 2 * K) : counts ? -1 : 0;
}

extern "C" int32_t moe_probe_square_choice(int32_t E, int64_t N, int64_t J, int64_t S) { return square_choice(E, N, J, S); }

extern "C" void moe_probe_fp8_choice(int64_t M, int64_t N, int64_t K, int32_t* out) {
  const TileChoice t = fp8_choice(M, N, (K + 15) / 16 * 16, dense_rows(M, N));
  out[0] = t.rows;
  out[1] = t.columns;
  out[2] = t.few;
}
