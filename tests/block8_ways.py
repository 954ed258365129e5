"""Sizes (rows, outputs, features) that take each way to a product of 8-bit rows, as
tcx_hip_linear8_plan tells them: a way is a tile's rows and outputs, the sets of waves, the
units of few rows, and whether the sums are split over blocks."""

# Of few rows, tiles of 16 x 16: up to 8 rows go through LDS where a wave has one unit.
# Blocks take one tile, two and three (more than 4096 and 8192 outputs).
FEW = {
    (16, 16, 8, 1, False): [(1, 300, 1000), (3, 8200, 4000), (1, 9001, 4096), (8, 4500, 3900), (16, 8195, 4096), (13, 5003, 3600)],
    (16, 16, 8, 2, False): [(5, 300, 7000), (1, 8201, 8000), (16, 8300, 8000), (9, 5999, 5000)],
    (16, 16, 8, 3, False): [(1, 200, 8300), (2, 11040, 9111), (16, 5900, 12288)],
}
LINEAR = FEW | {
    (32, 64, 4, 0, False): [(40, 90, 500), (300, 300, 500), (8, 12301, 3900)],
    (32, 64, 4, 0, True): [(100, 300, 8192), (2189, 20, 4691)],
    (64, 64, 4, 0, False): [(250, 4001, 500)],
    (64, 64, 4, 0, True): [(64, 4096, 11264)],
    (64, 64, 1, 0, False): [(64, 20000, 200), (2, 30000, 300)],
    (64, 64, 1, 0, True): [(35, 16925, 2764)],
    (128, 64, 2, 0, False): [(1500, 900, 260)],
    (128, 64, 2, 0, True): [(227, 656, 5634)],
    (128, 128, 1, 0, False): [(600, 12000, 300)],
    (128, 128, 1, 0, True): [(614, 1878, 7432)],
    (256, 128, 1, 0, False): [(700, 9000, 300)],
    (256, 128, 1, 0, True): [(1524, 646, 5762)],
    (256, 256, 1, 0, False): [(2040, 8190, 300), (3900, 5100, 1300)],
    (256, 256, 1, 0, True): [(5972, 674, 6026)],
}
# Of gated products, whose outputs are as many of gate and of up: in one launch with 128 of each in
# a tile, or in two.
GATED_ONE_LAUNCH = {
    (64, 128, 1, 0, False): [(7, 129, 300), (100, 3000, 1000)],
    (256, 128, 1, 0, False): [(2300, 2570, 200), (4000, 2600, 200)],
}
GATED = {
    (16, 16, 8, 1, False): [(3, 260, 1000), (3, 4200, 3000), (16, 4500, 4000)],
    (16, 16, 8, 2, False): [(2, 5001, 8000), (16, 4300, 8000)],
    (16, 16, 8, 3, False): [(1, 5500, 9000), (12, 5300, 10000)],
    (32, 64, 4, 0, False): [(33, 513, 640)],
    (32, 64, 4, 0, True): [(40, 300, 9000)],
    (64, 64, 4, 0, False): [(600, 700, 6000)],
    (64, 64, 4, 0, True): [(64, 2000, 6000)],
    (64, 64, 1, 0, True): [(35, 8400, 2764)],
    (128, 64, 2, 0, False): [(724, 900, 3721)],
    (128, 64, 2, 0, True): [(1188, 194, 1064)],
    (128, 128, 1, 0, True): [(359, 1391, 6565)],
    (256, 128, 1, 0, False): [(2732, 1458, 3481)],
    (256, 128, 1, 0, True): [(429, 1155, 4374)],
    (256, 256, 1, 0, True): [(972, 2055, 6498)],
}


def flat(ways):
    return [(way, shape) for way, shapes in ways.items() for shape in shapes]
