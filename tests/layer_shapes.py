"""Products of more than 16 rows that take every kernel, tile width and split a layer has: (M, N, K in 16-bit units,
activation, kernel, accumulator columns, split), checked on the CPU (test_layer_plan.py) and run on the GPU
(test_linear_act_gpu.py)."""
SHAPES = [
    (17, 64, 64, False, "one", 32, 1), (129, 1288, 648, True, "one", 32, 1),
    (129, 2400, 64, False, "one", 64, 1), (17, 2528, 1280, True, "one", 64, 2), (17, 64, 1280, False, "one", 64, 4),
    (33, 72, 2560, True, "one", 64, 8),
    (32, 5120, 5120, False, "one", 96, 2), (17, 2560, 10240, True, "one", 96, 4), (40, 1288, 5128, False, "one", 96, 8),
    (300, 3168, 64, False, "one", 80, 1), (300, 3936, 64, True, "one", 96, 1), (900, 1760, 64, False, "one", 112, 1),
    (900, 2048, 64, True, "one", 128, 1),
    (900, 2432, 648, False, "pair", 128, 1), (900, 2400, 320, True, "pair", 160, 1), (1700, 4032, 320, False, "pair", 192, 1),
    (3000, 2464, 64, True, "pair", 224, 1), (3000, 2816, 200, False, "pair", 256, 1),
]
