"""Sizes of the grouped and 8-bit products that reach every kernel (test_products_choice.py says so, test_gpu_products_tiles.py
runs them).  Rows: two in front of the first group and three behind the last."""

GAP, TAIL = 2, 3

RAGGED = [300, 0, 1, 517, 128, 129, 401, 64]

# rows, n, k of one matrix
FP8_DENSE = [(5, 40, 400), (16, 7300, 400), (60, 200, 400), (500, 1500, 400), (2650, 300, 272), (2000, 2000, 272), (4100, 4000, 400)]

# counts, n, k
FP8_GROUPED = [([3, 0, 1, 16], 200, 400), ([1, 2, 0, 3] * 16, 400, 272), ([33, 0, 57, 20], 130, 400), ([1200, 0, 700, 231], 353, 272),
               (RAGGED, 1000, 400), ([700, 0, 385, 128, 257] * 8, 1100, 272), ([700, 130, 385, 0] * 6, 4000, 400)]

# counts, n, k: result columns and contraction of the forward product, the other way round of the input gradient
ROWS = [([3, 0, 1, 16], 200, 136), ([1, 2, 0, 3] * 16, 400, 264), ([33, 0, 57, 20], 136, 264), (RAGGED, 424, 136), (RAGGED, 1000, 264),
        ([800, 0, 570, 130], 2600, 264), (RAGGED * 2, 1000, 1000), ([700, 130, 385, 0] * 6, 1304, 264), ([700, 130, 385, 0] * 6, 2600, 200)]

# counts, n, k
WGRAD = [([3, 0, 40], 40, 72), ([1218, 0, 700], 16, 24), ([3, 0, 1, 7] * 16, 16, 208), ([6176], 336, 656), ([5000, 700, 3], 264, 520),
         ([11, 0, 5] * 20, 136, 400), ([6099], 2920, 720), ([1, 0, 0, 2] * 4 + [0] * 50, 136, 400), ([9000, 40], 1608, 88), ([8000], 2048, 1000)]
