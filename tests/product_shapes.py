"""Shapes of block products that between them take every kernel, and the tile (rows, columns, parts of k) that each is made in: power-of-two scales
to 16 bits; float32 scales to 16 bits, b's in squares or in rows; power-of-two and float32 scales to float32.  Ragged in m, n and k; n odd (rows
at any address) and a multiple of 8; several tiles a workgroup in most large ones; more blocks of k than scales are held at a time."""
T16, T16W, T32, T32W, MID = (16, 16, 1), (16, 32, 1), (32, 32, 1), (32, 64, 1), (128, 128, 1)
B4, B6, B8 = (128, 256, 1), (192, 256, 1), (256, 256, 1)
MODES = (("e8m0", "tile", 16), ("fp32", "tile", 16), ("fp32", "rows", 16), ("e8m0", "tile", 32), ("fp32", "tile", 32))
KERNELS = [
    ((3, 41, 200), (T16,) * 5), ((100, 300, 2300), (T16,) * 5), ((300, 301, 2300), (T16W,) * 5), ((200, 1000, 2300), (T32,) * 5),
    ((700, 701, 2300), (T32W, T32W, T32W, T32W, T32)),
    ((2100, 2056, 300), (MID,) * 5), ((1035, 3672, 8500), (MID,) * 5), ((1035, 3665, 2300), (MID, B4, MID, MID, MID)),
    ((6492, 2309, 2300), (B4,) * 5), ((6492, 2312, 700), (B4,) * 5), ((928, 8749, 2300), (B6, B6, B6, B4, B4)),
    ((7241, 2083, 2300), (B6, B6, B6, B4, B4)), ((7241, 2080, 700), (B6, B6, B6, B4, B4)),
    ((8097, 2873, 2300), (B8, B8, B4, B4, B4)), ((8097, 2880, 700), (B8, B8, B4, B4, B4)),
    ((1024, 1280, 5120), ((128, 256, 5),) * 5), ((900, 261, 8192), ((128, 256, 16),) * 5),
]
