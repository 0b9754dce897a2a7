"""Shapes of the dense FP8 product, each tile's own, and the contractions that go
through its ring: the test of the kernels and the check that each shape takes its tile."""
from __future__ import annotations

# tile -> (M, N): the last tile of rows and of columns is partial
STAGED = {"16x64": (13, 4104), "32x64": (27, 8200), "64x64": (129, 4104), "64x128": (63, 16400), "128x64": (257, 4104),
          "128x128": (121, 16400), "128x256": (100, 40000), "256x64": (511, 4104), "256x128": (700, 9000), "256x256": (511, 16400)}
# 1 to 13 blocks of 128: below and past the rings' two to four stages and the scales' chunks of four steps, whole and partial
CONTRACTIONS = (128, 100, 256, 228, 512, 484, 640, 612, 768, 740, 1024, 1008, 1152, 1041, 1664, 1636)
# the contraction split over eight waves, four blocks of each on their way at a time
SPLIT = {"16 split": (13, 1000), "32 split": (27, 1000)}
SPLIT_CONTRACTIONS = (2048, 2052, 4096, 4224, 4200, 8320, 8400)
