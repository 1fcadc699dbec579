"""Products whose rows lie in strides that are multiples of 8 elements, and the
form each runs in (sv2hip.linear_plan): what the tests of the forms run, and
what the host tests hold the choice to."""
from __future__ import annotations


def up8(n):
    return (n + 7) // 8 * 8


# (rows, k, n), (kernel, tile, first_rows, form)
TILES = [
    ((7170, 72, 1032), ("tiles", 0, 0, "256x256")),
    ((7170, 69, 1029), ("tiles", 0, 0, "256x256")),  # k and n cut inside a piece
    ((5407, 64, 648), ("tiles", 0, 0, "256x128")),
    ((5407, 67, 643), ("tiles", 0, 0, "256x128")),
    ((1352, 200, 1480), ("tiles", 0, 0, "128x128")),
    ((1352, 203, 1477), ("tiles", 0, 0, "128x128")),
    ((1217, 1280, 784), ("tiles", 0, 0, "128x128-ksplit")),
    ((1217, 1283, 781), ("tiles", 0, 0, "128x128-ksplit")),
    ((4746, 1000, 3360), ("tiles", 0, 4608, "128x128-ksplit")),  # two launches
    ((4746, 1001, 3355), ("tiles", 0, 4608, "128x128-ksplit")),
    ((8974, 1086, 3966), ("tiles", 0, 8192, "128x128")),
]
FEW = [
    ((1, 256, 640), ("few", 16, 0, None)),
    ((20, 133, 513), ("few", 16, 0, None)),
    ((60, 1001, 2050), ("few", 16, 0, None)),
    ((300, 65, 513), ("few", 16, 0, None)),      # blocks of 64 rows
    ((300, 129, 1283), ("few", 64, 0, None)),
    ((600, 133, 2050), ("few", 64, 0, None)),
]


def sizes(table):
    return [s for s, _ in table]
