"""Sizes at which the library takes each form of its kernels.  tests/test_emu_plans.py asks the library's own rules whether it still does, so that
no form drops out of the GPU tests when a rule changes."""

# M, N, K, tile (32 w8 rows and columns), several blocks share a tile's K steps; K a multiple of 64 or not (the tail's code)
PRODUCTS = [
    (100, 300, 320, 4, False), (130, 250, 200, 4, False), (70, 130, 4096, 4, True), (60, 100, 4104, 4, True),
    (7400, 1100, 192, 6, False), (1899, 4500, 200, 6, False), (7926, 138, 6528, 6, True), (140, 7064, 6808, 6, True),
    (1250, 7400, 704, 8, False), (3710, 2361, 712, 8, False), (608, 6760, 6784, 8, True), (2350, 1802, 5872, 8, True),
]
# M, N, K of a gradient: tile of dA = dZ B, with B as it lies, and whether K steps are shared; the same of dB = dZ^T A
GRADIENTS = [
    (128, 192, 264, (4, False), (4, False)), (130, 195, 72, (4, False), (4, False)), (64, 1000, 64, (4, True), (4, False)), (883, 64, 64, (4, False), (4, True)),
    (1315, 128, 5984, (6, False), None), (3370, 130, 2312, (6, False), None), (135, 6222, 7064, (6, True), None), (6598, 6144, 144, (6, True), None),
    (2240, 704, 4088, (8, False), None), (6256, 653, 1352, (8, False), None), (5041, 5843, 848, (8, True), None),
    (64, 6080, 1288, None, (6, False)), (65, 3178, 2632, None, (6, False)), (7736, 146, 5496, None, (6, True)), (6400, 133, 7416, None, (6, True)),
    (704, 5638, 1544, None, (8, False)), (583, 1680, 5432, None, (8, False)), (6150, 832, 5056, None, (8, True)),
    (4001, 4096, 2056, (6, False), (6, False)),
]
# rows, channels, dtype, offsets (or equal sequences): enough tiles for blocks of 256 threads, forwards and backwards
SCANS = [
    (20000, 1032, "bf16", 1), (20000, 1001, "f16", 1), (20096, 1000, "bf16", 157), (20000, 640, "f32", 1), (20003, 1001, "f32", [0, 0, 1, 3000, 3000, 3129, 15000, 19990]),
    (20001, 1160, "f16", [5, 300, 301, 9000, 20001]), (140000, 24, "bf16", [0, 70000, 139999]),
]
