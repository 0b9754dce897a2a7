"""CPU: the shapes of the tests by tile take the tiles that they are for, by the
library's own rules."""
from __future__ import annotations

import math
import random

import pytest

import probe_lib
from ffn_tile_cases import ALL_TILES, CASES, tiles_of
from fp8_tile_cases import CONTRACTIONS, SPLIT, SPLIT_CONTRACTIONS, STAGED
from tile_choices import fp8_tile

pytestmark = pytest.mark.skipif(not probe_lib.LIB_PATH.exists(), reason="native library not built")


def test_fp8_shapes_take_their_tiles():
    for cases, lengths in ((STAGED, CONTRACTIONS), (SPLIT, SPLIT_CONTRACTIONS)):
        for tile, (M, N) in cases.items():
            for K in lengths:
                for less in range(3):  # the tests take N or one or two columns less
                    assert fp8_tile(M, N - less, K) == tile, (tile, M, N - less, K)


def test_every_fp8_tile_has_its_shape():
    """Over sizes of all kinds the rule chooses no tile without a shape."""
    sizes = [1, 2, 16, 17, 33, 64, 65, 100, 128, 129, 257, 300, 511, 700, 1000, 4096, 16400, 40000, 100000]
    found = {fp8_tile(M, N, K) for M in sizes for N in sizes for K in (128, 1024, 2048, 7168)}
    assert found == set(STAGED) | set(SPLIT)


def test_ffn_cases_take_every_tile():
    """The cases' tiles are all that there are, and calls of all sizes take no other."""
    found = set()
    for case in CASES:
        found |= tiles_of(*case)
    assert found == ALL_TILES
    rng = random.Random(3)
    for _ in range(4000):
        E = rng.choice((0, 0, 1, 2, 4, 8, 16, 48, 128))
        k = min(E, rng.choice((1, 2, 4))) if E else 1
        T, H, I = (int(round(math.exp(rng.uniform(0, math.log(n))))) for n in (16384, 14336, 14336))  # noqa: E741
        assert tiles_of(T, k, E, H, I, rng.choice((None, 16, 32, 64, 128, 256)) if E else None) <= ALL_TILES


def test_the_tiles_of_large_calls_have_large_cases():
    """Two thousand slots and more on widths of 512 and more, in the tiles that large calls spend their time in."""
    long = [c for c in CASES if c[0] * c[1] >= 2048 and min(c[3], c[4]) >= 512]
    have = set().union(*(tiles_of(*c) for c in long))
    assert {"gated 256x256", "actgrad 256x128", "actgrad 256x256", "product 256x256", "rows32 256x256", "dgrad 256x256",
            "dgrad32 256x256", "wgrad_dense 256x256"} <= have, have


def test_one_or_two_rows_split_the_contraction_at_any_width():
    """As the other products: staged tiles of 16 rows took 5 to 15 % longer."""
    for M in (1, 2):
        for N, K in ((4096, 7168), (14344, 4096), (36864, 7168), (1 << 18, 2048)):
            assert fp8_tile(M, N, K) == "16 split"
        assert fp8_tile(M, 36864, 2000) == "16x64"
    assert fp8_tile(3, 14344, 4096) == "16x64"
