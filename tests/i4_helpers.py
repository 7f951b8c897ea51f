"""4-bit weights of the tests: the packed layout in numpy, the products' 64-bit
form and how far a result may be from it."""
import numpy as np

import zkml_amd as z
from i8_helpers import ROUND, TINY, TYPES, Result, matrix, values, words


def packed(q, rng=None):
    """int8 weights (rows, cols) as the library lays them out; `rng` fills what lies
    behind a row's last weight with anything (else zeros)."""
    rows, cols = q.shape
    runs = -(-cols // 128)
    full = np.zeros((rows, runs * 128), dtype=np.int64) if rng is None else rng.integers(-8, 8, (rows, runs * 128))
    full[:, :cols] = q
    part = full.reshape(rows, runs, 2, 64) & 15
    return (part[:, :, 0] | part[:, :, 1] << 4).astype(np.uint8).reshape(rows, runs * 64)


def unpacked(b, cols):
    rows = b.shape[0]
    v = b.reshape(rows, -1, 64).astype(np.int64)
    q = np.stack([v & 15, v >> 4], axis=2).reshape(rows, -1)[:, :cols]
    return q - 16 * (q > 7)


def product(x, q, scale, group, sx, bias, relu):
    """(y, size): the 64-bit result of int8 rows, and what its terms' magnitudes come
    to.  scale: (groups, n_out) float64.  Sums of 32 products are exact in any split,
    so that the size is that of such sums times their scales."""
    n_in = x.shape[1]
    y = np.zeros((x.shape[0], q.shape[0]))
    size = np.zeros_like(y)
    for k in range(0, n_in, 32):
        part = x[:, k:k + 32].astype(np.float64) @ q[:, k:k + 32].astype(np.float64).T
        y += part * scale[k // group]
        size += np.abs(part * scale[k // group])
    s = 1.0 if sx is None else sx.astype(np.float64)[:, None]
    y, size = y * s, size * np.abs(s)
    if bias is not None:
        y, size = y + bias, size + np.abs(bias)
    return (np.maximum(y, 0) if relu else y), size


def wide_product(x, q, scale, group, sx, bias, relu):
    """product() for many results: a group of up to 128 at a time, whose sums are exact
    in 32-bit floats (below 128 * 128 * 8), a term's size from the magnitudes' sum."""
    n_in, run = x.shape[1], min(group, 128)
    y = np.zeros((x.shape[0], q.shape[0]))
    size = np.zeros_like(y)
    xf, qf = x.astype(np.float32), q.astype(np.float32)
    for k in range(0, n_in, run):
        s = scale[k // group]
        y += (xf[:, k:k + run] @ qf[:, k:k + run].T) * s
        size += (np.abs(xf[:, k:k + run]) @ np.abs(qf[:, k:k + run]).T) * np.abs(s)
    s = 1.0 if sx is None else sx.astype(np.float64)[:, None]
    y, size = y * s, size * np.abs(s)
    if bias is not None:
        y, size = y + bias, size + np.abs(bias)
    return (np.maximum(y, 0) if relu else y), size


def near(got, want, size, n_in, kind):
    """Within a rounding of 2^-24 of the terms' size for each 32 weights and three
    more (a term itself, the token's scale, the bias), and one of the result's type."""
    lim = (-(-n_in // 32) + 3) * 2.0**-24 * size
    lim = lim + (np.abs(want) + lim) * ROUND[kind] + TINY[kind]
    bad = ~(np.abs(values(got, kind) - want) <= lim)
    assert not bad.any(), f"{int(bad.sum())} of {bad.size} off, first at {np.argwhere(bad)[0]}"


def inputs(rng, rows, n_out, n_in, group, scale_kind="f32", experts=1):
    """x, sx, q, scales (words), their values."""
    x = rng.integers(-127, 128, (rows, n_in)).astype(np.int8)
    # f16 results end at 65504: scales small enough for it
    sx = np.exp(rng.normal(-6, 0.5, rows)).astype(np.float32)
    q = rng.integers(-8, 8, (experts * n_out, n_in)).astype(np.int8)
    s = words(np.exp(rng.normal(-3, 0.5, (experts, -(-n_in // group), n_out))), scale_kind)
    return x, sx, q, s, values(s, scale_kind)


__all__ = ["packed", "unpacked", "product", "wide_product", "near", "inputs", "Result", "matrix", "TYPES", "values", "words",
           "z"]
