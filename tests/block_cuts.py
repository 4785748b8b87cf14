"""Sizes of block-FP8 products that stand for every kernel, tile and split, with
the cut that each of them takes on 256 CUs (test_block_cuts.py holds the table
to the library's own choice, test_gpu_block_exact.py multiplies them)."""

F32, BF16 = 0, 1

# (M, N, K, type of the result, tile edge or 0 for the few-row kernel, splits of the K blocks).  The large tiles
# have five K blocks or more, so that stages are refilled, and remainders in M, N and K.
CUTS = [
    (1, 515, 1000, BF16, 0, 1), (1, 515, 1000, F32, 0, 1), (16, 300, 4100, BF16, 0, 1), (31, 1000, 650, F32, 0, 1),
    (64, 770, 2049, BF16, 0, 1), (64, 770, 2049, F32, 0, 1),
    (300, 400, 640, BF16, 64, 1), (300, 400, 640, F32, 64, 1), (130, 4000, 2000, BF16, 64, 1), (129, 65, 1200, F32, 64, 1),
    (300, 515, 4100, BF16, 64, 8), (300, 515, 4100, F32, 64, 4), (96, 97, 20000, BF16, 64, 16), (96, 97, 20000, F32, 64, 16),
    (2000, 1900, 900, BF16, 128, 1), (4001, 4099, 700, F32, 128, 1), (9000, 2300, 1100, BF16, 128, 1),
    (700, 500, 9000, BF16, 128, 8), (700, 500, 9000, F32, 128, 8), (1001, 2040, 5000, F32, 128, 2),
    (3900, 4090, 600, BF16, 256, 1), (8190, 2047, 840, BF16, 256, 1), (65500, 250, 600, BF16, 256, 1),
    (3970, 4090, 1300, BF16, 256, 1),
]
