"""Sizes at which each kernel of the int8 products and of the expert layer runs on 256 compute units.  test_i8_abi holds the
sizes to the kernels that they are listed under, test_gpu_i8_kernels runs them."""
from oxidize_amd import int8
from oxidize_amd.int8 import FEW, FEW_FLOAT, FEW_WIDE, TILES

# (kernel, tile, split?, half tiles?) or (kernel, stages held, tokens in sixteens): [(tokens, rows, columns)]
MATMUL = {
    (FEW, 2, 1): [(1, 16, 64), (16, 200, 4096), (7, 4096, 1000)],
    (FEW, 4, 1): [(1, 16, 4102), (8, 40, 8192), (5, 14336, 4096)],          # the last: a gate projection under five tokens
    (FEW, 8, 1): [(1, 3057, 8209), (2, 4096, 14336), (8, 4096, 14336), (8, 3100, 16384)],      # down projections
    (FEW_WIDE, 2, 2): [(17, 16, 64), (32, 50, 4090)],
    (FEW_WIDE, 2, 3): [(34, 16, 65), (48, 70, 4096)],
    (FEW_WIDE, 2, 4): [(49, 17, 66), (64, 4096, 4000)],
    (TILES, int8.TILE_256x256, False, False): [(514, 19821, 132)],
    (TILES, int8.TILE_256x256, False, True): [(776, 23320, 386)],
    (TILES, int8.TILE_256x256, True, False): [(130, 11042, 8238)],
    (TILES, int8.TILE_128x256, False, False): [(825, 8133, 274)],
    (TILES, int8.TILE_128x256, True, False): [(3990, 130, 12785)],
    (TILES, int8.TILE_128x192, False, False): [(603, 8092, 132)],
    (TILES, int8.TILE_128x192, True, False): [(131, 5498, 5051), (333, 4096, 14336)],
    (TILES, int8.TILE_128x128, False, False): [(66, 16916, 65)],
    (TILES, int8.TILE_128x128, True, False): [(66, 2700, 7728)],
    (TILES, int8.TILE_64x64_RING, False, False): [(67, 16, 64), (70, 300, 1030)],
    (TILES, int8.TILE_64x64_RING, True, False): [(9, 16, 4230), (48, 4096, 14336)],
    (TILES, int8.TILE_64x64, False, False): [(1, 32863, 64), (33, 40000, 100)],
    (TILES, int8.TILE_64x64, True, False): [(1, 4107, 3588)],
}
# float tokens that the product's own launch quantises: {stages held: ...}
LINEAR = {2: [(1, 16, 64), (4, 300, 4095)], 4: [(1, 16, 4102), (2, 33, 8190)], 8: [(1, 16, 8201), (1, 4096, 14336), (1, 2048, 11008)]}

# (pair by pair?, pairs of a tile, stages held for gate and up, for down): [(tokens, experts, choices, hidden, ffn)]
EXPERTS = {
    (1, 1, 2, 4): [(3, 4, 2, 70, 500), (1, 128, 8, 2048, 768)],
    (1, 1, 2, 8): [(2, 4, 1, 60, 8300), (1, 20, 8, 130, 2000)],
    (1, 1, 4, 4): [(2, 4, 1, 3000, 70)],
    (1, 1, 4, 8): [(1, 4, 2, 4096, 4200)],
    (1, 1, 8, 4): [(2, 4, 2, 5120, 300), (1, 6, 2, 5120, 1536)],
    (1, 1, 8, 8): [(1, 4, 4, 4200, 2100)],
    (0, 16, 2, 2): [(8, 2, 1, 64, 64), (17, 30, 3, 300, 130)],
    (0, 16, 2, 4): [(8, 2, 1, 200, 5000)],
    (0, 16, 2, 8): [(8, 2, 1, 130, 8200), (9, 4, 2, 70, 14336)],
    (0, 16, 4, 2): [(8, 2, 1, 2500, 100)],
    (0, 16, 4, 4): [(8, 2, 1, 4096, 4200)],
    (0, 16, 8, 2): [(8, 2, 1, 4200, 40), (8, 2, 1, 8192, 30)],
    (0, 16, 0, 2): [(8, 2, 1, 8300, 40), (40, 30, 3, 9000, 20)],
    (0, 16, 2, 0): [(8, 2, 1, 40, 16500)],
    (0, 64, 0, 0): [(40, 2, 1, 300, 200), (300, 8, 1, 130, 140)],
    (0, 128, 0, 0): [(130, 2, 1, 300, 200), (700, 4, 2, 200, 130)],
}
