"""CPU: the shapes of the tests by tile take the tiles that they are for, by the
library's own rules."""
from __future__ import annotations

import pytest

import probe_lib
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
