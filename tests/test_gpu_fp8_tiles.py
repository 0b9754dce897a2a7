"""GPU: each tile of the dense FP8 product through its ring, against 64-bit results
element by element: contractions below, at and past the ring's stages, the chunks of
four steps of scales and their second buffer, whole and partial last blocks."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from ffn_cases import apart, exact_fp8, over  # noqa: E402
from fp8_tile_cases import CONTRACTIONS, SPLIT, SPLIT_CONTRACTIONS, STAGED  # noqa: E402
from grouped_cases import HALF  # noqa: E402
from tile_choices import fp8_tile  # noqa: E402

BF16, FP16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def make(M, N, K):
    """a, b and their scales, random throughout and made on the GPU."""
    g = torch.Generator(device="cuda").manual_seed(7 * M + 3 * N + K)
    kb, nb = -(-K // 128), -(-N // 128)
    a, b = ((torch.randn((n, K), generator=g, device="cuda") * 100).clamp(-448, 448).to(FP8) for n in (M, N))
    sa, sb = (torch.exp(torch.randn((n, kb), generator=g, device="cuda")) * s for n, s in ((M, 1e-2), (nb, 1e-3)))
    return a, b, sa, sb


def check(tile, M, N, K, dtype, with_bias):
    from td_benchmark_amd import ops
    print(f"case: {tile} M={M} N={N} K={K} {dtype}", flush=True)
    assert fp8_tile(M, N, K) == tile
    a, b, sa, sb = make(M, N, K)
    bias = torch.randn(N, device="cuda").to(dtype) if with_bias else None
    y = ops.fp8_scaled_mm(a, b, sa, sb, bias, dtype)
    want = exact_fp8(a, b, sa, sb, bias, dtype)
    assert over(y, want) <= 0
    # one rounding, and cuts of 2^-13 of the largest of 8 products, which add up as independent errors
    assert apart(y, want[0]) <= HALF[dtype] + 2.0 ** -11
    assert torch.equal(y, ops.fp8_scaled_mm(a, b, sa, sb, bias, dtype))


@pytest.mark.parametrize("K", CONTRACTIONS)
@pytest.mark.parametrize("tile", STAGED)
def test_steps_of_each_tile(tile, K):
    M, N = STAGED[tile]
    # an odd count of columns, whose rows are stored element by element, where the last block is partial
    check(tile, M, N - (1 if K % 128 else 0), K, FP16 if K % 256 else BF16, bool(K % 128))


@pytest.mark.parametrize("K", SPLIT_CONTRACTIONS)
@pytest.mark.parametrize("tile", SPLIT)
def test_the_split_of_the_contraction(tile, K):
    M, N = SPLIT[tile]
    check(tile, M, N - K % 3, K, BF16 if K % 256 else FP16, bool(K % 128))


@pytest.mark.parametrize("tile,M,N,K", [("256x256", 2000, 7168, 7168), ("64x64", 45, 14344, 4096), ("16 split", 1, 36864, 7168), ("16 split", 2, 14344, 4096), ("16x64", 3, 14344, 4096),
                                        ("128x128", 121, 16400, 4096)])
def test_long_contractions(tile, M, N, K):
    """32 and 56 blocks, as layers have them."""
    check(tile, M, N, K, BF16, False)
