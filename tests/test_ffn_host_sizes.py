"""CPU: sizes that the C entries of the feed-forward block and of the block-scaled FP8
product refuse because their bytes do not fit 64 bits, and refusals that come before
any device work."""
from __future__ import annotations

import ctypes

import pytest

pytest.importorskip("torch")

from td_benchmark_amd import _lib  # noqa: E402


@pytest.fixture(scope="module")
def L():
    if not _lib.LIB_PATH.exists():
        pytest.skip("native library not built")
    return _lib.lib()


BY_NAME = {name: code for code, name in _lib.STATUS.items()}
BAD = BY_NAME["MOE_ERR_BAD_SHAPE"]
BUF = (ctypes.c_int32 * 256)()  # host memory: only ever passed to a rejected call
P = (ctypes.addressof(BUF) + 15) // 16 * 16
BASE = dict(T=4, H=16, I=16, ldx=16, max_padded=48, top_k=2, E=3, block_size_m=16, dtype=0, x=P, w13=P, w2=P, topk_weights=P,
            sorted_ids=P, expert_ids=P, ntpp=P, expert_table=P, h=P, gu=P, workspace=P)


@pytest.mark.parametrize("passes,sizes", [
    # slots
    ((0, 1), dict(T=1 << 62, top_k=4)), ((0, 1), dict(T=1 << 61, top_k=1 << 30)), ((0, 1), dict(T=(1 << 63) - 1, top_k=3)),
    # the weights
    ((0, 1), dict(H=1 << 29, ldx=1 << 29, I=1 << 28, E=1 << 30)), ((0, 1), dict(H=1 << 29, ldx=1 << 29, I=1 << 28, E=1 << 7)),
    # all parts of the backward pass together
    ((1,), dict(T=1 << 30, top_k=1, max_padded=1 << 30, H=1 << 29, ldx=1 << 29, I=1 << 28, E=2, dtype=1, w13=P + 2, w2=P + 2))])
def test_c_ffn_refuses_sizes_past_64_bits(L, passes, sizes):
    f = _lib.MoeFfn(**{**BASE, **sizes})
    for backward in passes:
        assert L.moe_ffn_workspace_bytes(f, backward) == BAD
        assert (L.moe_ffn_backward(f, P, P, P, P, P, None) if backward else L.moe_ffn_forward(f, P, None)) == BAD


def test_c_ffn_takes_the_longest_widths_it_documents(L):
    """2^29 and 2^28 columns of one expert, whose weights' copies have 2^60 bytes."""
    f = _lib.MoeFfn(**{**BASE, "H": 1 << 29, "ldx": 1 << 29, "I": 1 << 28, "E": 1, "w13": P + 2})
    assert L.moe_ffn_workspace_bytes(f, 0) > 1 << 59


def test_c_fp8_refuses_sizes_past_64_bits(L):
    """Rows and columns whose padded codes have more bytes than 64 bits hold; the size and the call refuse alike."""
    for M, N, K in ((1 << 62, 24, 160), (1 << 31, 24, 160), (4, 1 << 62, 160), (4, (1 << 63) - 1, 160), (4, 1 << 41, (1 << 23) - 16)):
        assert L.moe_fp8_scaled_mm_workspace_bytes(P + 1, K + 1, P + 1, K + 1, M, N, K) == BAD
        assert L.moe_fp8_scaled_mm(P + 1, K + 1, P, P + 1, K + 1, P, None, M, N, K, 0, P, N, P, None) == BAD


@pytest.mark.parametrize("which", ["dw13", "dw2"])
def test_c_ffn_refuses_unaligned_weights_gradients_first(L, which):
    """Where the widths are multiples of 8 the weights' gradients are 16-byte aligned: found before any launch (which
    fails by another code without a GPU), also where the gradients by the tokens and the router's weights are asked for."""
    f = _lib.MoeFfn(**BASE)
    dw = dict(dw13=P, dw2=P)
    dw[which] = P + 2
    assert L.moe_ffn_backward(f, P, P, dw["dw13"], dw["dw2"], P, None) == BAD


def test_c_ffn_workspace_of_aligned_rows(L):
    """Room for copies of y (one slot a token), and of dx and dy, only where their rows are not whole 16-byte chunks."""
    size = L.moe_ffn_workspace_bytes
    rows = 1000 * 16 * 2 // 256 * 256 + (256 if 1000 * 16 * 2 % 256 else 0)
    one = dict(BASE, T=1000, top_k=1, max_padded=2000, topk_weights=None)
    f = _lib.MoeFfn(**one)
    assert size(f, 256) == 0 and size(f, 0) == rows           # y
    dgu = 1000 * 2 * 16 * 2
    assert size(f, 257) == dgu and size(f, 1) == dgu + 2 * rows  # dx and dy
    f = _lib.MoeFfn(**{**one, "top_k": 2, "max_padded": 4000})
    assert size(f, 256) == size(f, 0) and size(f, 1) == size(f, 257) + rows  # dy; y and dx come from the slots' rows
    assert size(f, 2) == size(f, 3) == size(f, -1) == size(f, 1)  # any other value is the backward pass's
    odd = _lib.MoeFfn(**{**one, "H": 15, "ldx": 16})
    assert size(odd, 256) == size(odd, 0) > rows and size(odd, 257) == size(odd, 1) > 2 * rows
