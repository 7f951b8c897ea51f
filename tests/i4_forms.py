"""Sizes of the 4-bit product's tests by the form of kernel that each is meant for: the
tile, whether x's rows are in whole chunks of 16 bytes, and the groups.  Odd rows lie one
byte on, at a stride of one byte more than their length.  Every size has several
tiles, a last one that is not full, several steps of 128 and a last one that is not whole."""
# (tile, odd): (rows, n_out, n_in), for each of GROUPS
GROUPS = (32, 64, 128, 384)
PLAIN = {
    ("wave 4x16", 0): (1, 45, 464), ("wave 4x16", 1): (3, 45, 450),
    ("wave 16x16", 0): (5, 2870, 464), ("wave 16x16", 1): (5, 3679, 453),
    ("wave 16x32", 0): (5, 5327, 464), ("wave 16x32", 1): (5, 4956, 464),
    ("wave 32x32", 0): (17, 5945, 480), ("wave 32x32", 1): (18, 8062, 644),
    ("wave 48x32", 0): (33, 5697, 464), ("wave 48x32", 1): (3966, 65, 780),
    ("stages 32x128", 0): (5514, 98, 480), ("stages 32x128", 1): (3976, 167, 473),
    ("stages 64x128", 0): (5110, 262, 464), ("stages 64x128", 1): (4877, 263, 454),
}
# the largest tile, which groups of 32 reach with short rows alone
LARGE = {32: (5121, 2788, 208), 64: (4788, 2330, 464), 128: (2956, 3722, 464), 384: (2956, 3722, 464)}
# (tile, odd): (rows, n_out, n_in, experts), one slot a token
GROUPED = {
    ("wave 4x16", 0): (7, 45, 464, 16), ("wave 4x16", 1): (3, 45, 453, 3),
    ("wave 4x32", 0): (64, 67, 480, 64), ("wave 4x32", 1): (32, 145, 455, 64),
    ("wave 16x32", 0): (555, 65, 464, 64), ("wave 16x32", 1): (5, 7089, 467, 2),
    ("stages 32x128", 0): (15, 3315, 464, 40), ("stages 32x128", 1): (57, 891, 455, 64),
    ("stages 64x128", 0): (4104, 259, 496, 64), ("stages 64x128", 1): (3986, 267, 532, 64),
}

# (tile, odd, group, rows, n_out, n_in, experts), experts 0: not grouped
FORMS = [(t, o, g, *s, 0) for (t, o), s in PLAIN.items() for g in GROUPS]
FORMS += [("stages 256x256", 0, g, *s, 0) for g, s in LARGE.items()]
FORMS += [(t, o, g, *s) for (t, o), s in GROUPED.items() for g in GROUPS]
