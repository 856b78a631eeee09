"""Shapes of 8-bit products that take each of the kernels' forms on 256 CUs."""

import ctypes

# (rows, K, columns): tiles of 256 x 256 that go as two halves.  Several steps of 128 k, the last one short; odd rows and
# columns; a last strip of fewer than four rows of tiles.
TILES = {
    (256, 256): [
        ((2300, 1168, 13700), 0), ((1500, 1200, 6000), 0), ((1537, 656, 16500), 0), ((300, 4112, 30001), 0),
        ((4096, 2560, 13824), 96), ((4095, 656, 13800), 96), ((8190, 1040, 2565), 96),
        ((1285, 656, 12300), 38),  # the last row of tiles has 5 rows: no second half
    ],
    (128, 256): [((1025, 2576, 6920), 0), ((300, 2576, 13825), 0), ((1300, 656, 16400), 0), ((700, 3088, 9999), 0)],
    (128, 128): [((515, 2576, 3845), 0), ((900, 720, 2900), 0), ((1100, 1040, 2000), 0), ((66, 2560, 30000), 0)],
    (128, 64): [((511, 2560, 3840), 0), ((390, 2576, 3845), 0), ((128, 2560, 13824), 0), ((609, 464, 2771), 0),
                ((147, 4256, 6175), 0)],
    (64, 64): [((130, 6912, 2560), 0), ((257, 1616, 6001), 0), ((33, 2560, 640), 0)],
}
CASES = [(tile, shape, halves) for tile, shapes in TILES.items() for shape, halves in shapes]


def plan(lib, *shape):
    """(column blocks of the weight stream, rows and columns of a tile, tiles that go as halves)."""
    out = (ctypes.c_int64 * 4)()
    assert lib.btl_int8_matmul_plan(*shape, out) == 1
    return tuple(out)
