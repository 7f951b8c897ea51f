"""Sizes of the 4-bit product's tests by the kernel that each is meant for."""
# kernel: (rows, n_out, n_in) with rows of x in whole chunks of 16 bytes
PLAIN = {
    "wave 4x16": [(1, 70, 256), (4, 33, 1024), (3, 4096, 2048)],
    "wave 16x16": [(15, 2571, 208), (23, 1995, 1040), (361, 66, 912)],
    "wave 16x32": [(14, 6046, 176), (91, 1152, 480), (418, 264, 272)],
    "wave 32x32": [(59, 2653, 1120), (1690, 155, 224)],
    "wave 48x32": [(169, 2696, 2080), (1661, 199, 400)],
    "stages 32x128": [(1092, 1656, 448), (949, 1115, 368)],
    "stages 64x128": [(507, 4798, 368), (2237, 1151, 1152)],
    "stages 256x256": [(3470, 4788, 224), (2049, 7535, 672)],
}
# (rows, n_out, n_in, experts), one slot a token
GROUPED = {
    "wave 4x16": [(1, 16, 64, 4), (18, 154, 80, 16), (104, 18, 304, 4)],
    "wave 4x32": [(51, 90, 64, 64), (5, 1326, 1408, 64)],
    "wave 16x32": [(66, 1517, 288, 8), (25, 3953, 800, 4), (3308, 18, 2352, 64)],
    "stages 32x128": [(276, 507, 192, 8), (8, 3491, 240, 16)],
    "stages 64x128": [(1875, 1322, 224, 4), (3334, 603, 80, 32)],
}


def listed(by_kernel):
    return [(k, *s) for k, sizes in by_kernel.items() for s in sizes]
