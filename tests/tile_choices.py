"""The tiles that the products' launches choose, by the library's own rules compiled
into tests/libmoe_probe.so (tests/csrc/choices.hip): tests name the tile that a case is
for, and a changed rule cannot leave a tile without its case unnoticed."""
from __future__ import annotations

import ctypes

import probe_lib

FORMS = ("product", "dgrad", "wgrad", "rows32", "gated", "actgrad", "wgrad_tok", "wgrad_dense")  # enum Form of grouped_tile.hpp


def _out(name, *args, n):
    out = (ctypes.c_int32 * n)()
    getattr(probe_lib.lib(), name)(*args, out)
    return tuple(out)


def rows_tile(form, S, J, K, E=1, block_m=0, max_padded=0):
    """(rows, columns, split, parts) of a rows form; dense without block_m."""
    i32, i64 = ctypes.c_int32, ctypes.c_int64
    return _out("moe_probe_rows_choice", i32(FORMS.index(form)), i32(not block_m), i64(S), i32(E), i32(block_m), i64(max_padded),
                i64(J), i64(K), n=4)


def square_weights(E, N, J, S):
    i64 = ctypes.c_int64
    return bool(probe_lib.lib().moe_probe_square_choice(ctypes.c_int32(E), i64(N), i64(J), i64(S)))


def fp8_tile(M, N, K):
    """"rows x columns", or "rows split" where the contraction is split over the waves."""
    i64 = ctypes.c_int64
    rows, columns, few = _out("moe_probe_fp8_choice", i64(M), i64(N), i64(K), n=3)
    return f"{rows} split" if few else f"{rows}x{columns}"
