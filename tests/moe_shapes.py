"""Sizes that together reach every variant of the grouped product's kernels: test_moe_plan_cpu.py
holds them to that, test_moe_variants_gpu.py runs them."""
import ctypes

from mxfp4_b200 import capi

# (E, M, N, K).  Scale rows are whole multiples of 16 bytes where K % 512 == 0: TMA takes them;
# others arrive line by line.  BF16 rows of N = 2600, 2568 and 1032 are not whole 32-byte sectors.
WIDE = [
    (5, 3001, 1424, 512),    # 128 weight rows a tile, several tiles a pair; TMA
    (5, 3001, 1424, 544),    #   the same, lines
    (3, 2600, 2600, 4096),   # 256 weight rows, TMA
    (3, 2600, 2600, 4128),   #   lines
    (3, 2600, 2624, 4128),   #   and columns that can be quantized
]
NARROW = [
    (16, 100, 2568, 1056),   # 16 rows a tile, one CTA a tile, several tiles a CTA
    (16, 100, 2576, 4128),   #   two CTAs share a tile's K, several tiles a pair
    (8, 9, 512, 2048),       #   more CTAs, one tile each
    (1, 1, 64, 32),
    (2, 9, 64, 4096),
    (16, 400, 2576, 1056),   # 64 rows a tile, likewise
    (16, 400, 2560, 4128),
    (1, 30, 1032, 2048),
    (1, 60, 336, 7200),
    (3, 40, 272, 96),
]


def plan(E, M, N, K, activation="none", quantized=False, aligned=None):
    """(rows of a tile, weight rows of a tile, CTAs that split K, most tiles, clusters)."""
    out = (ctypes.c_int64 * 5)()
    aligned = K % 512 == 0 if aligned is None else aligned
    capi.call("mxb_grouped_gemm_plan", M, E, N, K, capi.ACTIVATIONS[activation], int(quantized), int(aligned), out)
    return tuple(out)
