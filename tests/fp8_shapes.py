"""Products that reach every kernel of the 8-bit float product on a B200 (148 SMs), one entry per
tile and split of k; tests/test_fp8_choice_cpu.py holds the choice to this table and
tests/test_gpu_fp8_kernels.py runs it."""

SMS = 148
# (choice, split, m, n, k): choice as gq_choose.h gives it, a narrow tile's tokens or twice a wide
# tile's channels
ANY_TYPE = [
    (16, 1, 3, 333, 96), (16, 1, 3, 19100, 4256), (16, 2, 20, 8201, 2080), (16, 4, 3, 8200, 2080), (16, 8, 3, 333, 2080),
    (32, 1, 509, 1157, 2080), (32, 2, 257, 1152, 2080), (32, 4, 50, 2597, 2080), (32, 8, 100, 336, 4128),
    (64, 1, 33, 19100, 2080), (64, 1, 257, 4608, 96), (64, 2, 509, 1157, 3584), (64, 4, 257, 1152, 3584),
    (128, 1, 257, 8201, 96), (128, 1, 70, 19104, 2080), (128, 1, 1900, 1157, 96),
    (256, 1, 509, 2600, 2080), (256, 1, 509, 2597, 2080), (256, 1, 520, 8201, 96), (256, 1, 509, 4608, 3584),
    (512, 1, 1100, 2600, 2080), (512, 1, 1100, 2597, 2080), (512, 1, 1100, 8201, 96), (512, 1, 520, 4613, 2080),
]
# f32 outputs alone: k split further, or another kernel, so that no piece of a sum grows too long
F32_ONLY = [(128, 2, 100, 19100, 8480), (16, 2, 3, 19100, 32768), (32, 2, 20, 19100, 19968), (64, 2, 50, 19100, 32768),
            (16, 4, 1, 19100, 65536)]
# what the tests of repeats, graphs, streams and chains run
WIDE = [(256, 1, 600, 2600, 2080), (256, 1, 700, 2560, 2048), (512, 1, 1500, 2560, 2048), (256, 1, 1500, 1024, 1280),
        (512, 1, 1300, 2600, 2080)]
