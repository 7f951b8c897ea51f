"""GPU tests of the 8-bit integer layers (cuda-zkml_amd/csrc/i8_matmul.hip).

The sums are exact integers: numpy's int64 product gives them bit for bit.  A
scaled result is float(acc) * (sx * sw) + b in 32-bit floats, four roundings of
2^-24 relative to |acc sx sw| + |b| at the most, then one to the result's type;
the expected values are computed in 64 bits from the same inputs.
"""
import ctypes

import numpy as np
import pytest

import zkml_amd as z
from i8_helpers import ROUND, TINY, TYPES, At, Result, matrix, values, words

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return z.Context(0)


def say(*a):
    print(*a, flush=True)


def near(got, want, size, kind):
    """|got - want| within four roundings of 2^-24 of `size` and one of the type."""
    got = values(got, kind)
    lim = 4 * 2.0**-24 * size
    lim = lim + (np.abs(want) + lim) * ROUND[kind] + TINY[kind]
    bad = ~(np.abs(got - want) <= lim)
    assert not bad.any(), f"{int(bad.sum())} of {bad.size} off, first at {np.argwhere(bad)[0]}"


SIZES = [(1, 1, 1), (1, 1, 16), (3, 5, 7), (1, 64, 64), (2, 33, 65), (16, 16, 64), (17, 15, 63), (32, 32, 32),
         (64, 64, 64), (65, 63, 129), (1, 1000, 4097), (5, 300, 1001), (31, 130, 255), (33, 70, 256), (128, 128, 128),
         (130, 257, 1000), (256, 256, 512), (300, 513, 640), (1025, 31, 64), (1000, 32, 64), (40, 2050, 300),
         (257, 300, 1153), (700, 520, 96)]


@pytest.mark.parametrize("rows,n_out,n_in", SIZES)
def test_sums_are_exact(ctx, rows, n_out, n_in):
    rng = np.random.default_rng([rows, n_out, n_in])
    x = rng.integers(-128, 128, (rows, n_in)).astype(np.int8)
    w = rng.integers(-128, 128, (n_out, n_in)).astype(np.int8)
    say("[i8 sums]", rows, n_out, n_in)
    y = Result(ctx, rows, n_out, "i32")
    ctx.i8_matmul(matrix(ctx, x), matrix(ctx, w), rows, n_out, n_in, y.at)
    want = x.astype(np.int64) @ w.astype(np.int64).T
    assert np.array_equal(y.read(), want)
    # ReLU on the integers
    y = Result(ctx, rows, n_out, "i32")
    ctx.i8_matmul(matrix(ctx, x), matrix(ctx, w), rows, n_out, n_in, y.at, relu=True)
    assert np.array_equal(y.read(), np.maximum(want, 0))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scales,bias,relu", [("both", True, False), ("both", False, True), ("token", True, True),
                                              ("channel", False, False), ("none", True, False)])
@pytest.mark.parametrize("rows,n_out,n_in", [(1, 700, 1000), (6, 33, 70), (100, 65, 333), (270, 260, 1024)])
def test_scaled(ctx, kind, scales, bias, relu, rows, n_out, n_in):
    rng = np.random.default_rng([rows, n_out, n_in])
    x = rng.integers(-127, 128, (rows, n_in)).astype(np.int8)
    w = rng.integers(-127, 128, (n_out, n_in)).astype(np.int8)
    # f16 ends at 65504: scales small enough for it
    sx = np.exp(rng.normal(-6, 0.5, rows)).astype(np.float32) if scales in ("both", "token") else None
    sw = np.exp(rng.normal(-6, 0.5, n_out)).astype(np.float32) if scales in ("both", "channel") else None
    b = rng.normal(0, 1, n_out).astype(np.float32) if bias else None
    if scales == "none":
        x //= 16
        w //= 16
    say("[i8 scaled]", kind, scales, rows, n_out, n_in)
    y = Result(ctx, rows, n_out, kind)
    up = lambda a: None if a is None else ctx.upload(a)  # noqa: E731
    ctx.i8_matmul(matrix(ctx, x), matrix(ctx, w), rows, n_out, n_in, y.at, TYPES[kind], x_scale=up(sx),
                  w_scale=up(sw), bias=up(b), relu=relu)
    want = (x.astype(np.int64) @ w.astype(np.int64).T).astype(np.float64)
    want = want * (1 if sx is None else sx.astype(np.float64)[:, None]) * (1 if sw is None else sw.astype(np.float64))
    size = np.abs(want) + (0 if b is None else np.abs(b))
    want = want + (0 if b is None else b)
    if relu:
        want = np.maximum(want, 0)
    near(y.read(), want, size, kind)


@pytest.mark.parametrize("kind", ["i32", "f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n_out,n_in", [(1, 70, 100), (5, 65, 1000), (40, 130, 77), (260, 300, 515),
                                             (300, 256, 1024)])
@pytest.mark.parametrize("lead,pad", [(1, 3), (4, 12), (8, 5), (16, 16)])
def test_strides_and_offsets(ctx, kind, rows, n_out, n_in, lead, pad):
    """Rows of x, w and y at other strides and at odd addresses; nothing beside
    y is written, nothing beside x and w is used."""
    rng = np.random.default_rng([rows, lead, pad])
    x = rng.integers(-8, 9, (rows, n_in)).astype(np.int8)
    w = rng.integers(-8, 9, (n_out, n_in)).astype(np.int8)
    say("[i8 strides]", kind, rows, n_out, n_in, lead, pad)
    y = Result(ctx, rows, n_out, kind, ld=n_out + pad, lead=lead)
    ctx.i8_matmul(matrix(ctx, x, n_in + pad, lead), matrix(ctx, w, n_in + 2 * pad, lead + 1), rows, n_out, n_in,
                  y.at, TYPES[kind], ld_x=n_in + pad, ld_w=n_in + 2 * pad, ld_y=n_out + pad)
    want = x.astype(np.int64) @ w.astype(np.int64).T
    if kind == "i32":
        assert np.array_equal(y.read(), want)
    else:
        near(y.read(), want.astype(np.float64), np.abs(want), kind)


def wide_sums(x, w):
    """The exact sums by way of float64, whose 53 bits hold them."""
    return (x.astype(np.float64) @ w.astype(np.float64).T).astype(np.int64)


# sizes whose work fills the chip: the large tiles, whole and ragged, rows that
# are multiples of 16 bytes, of 4, and of one
@pytest.mark.parametrize("rows,n_out,n_in", [(1100, 1200, 2080), (1500, 1030, 656), (2050, 2200, 4112),
                                             (4100, 4090, 1040), (4100, 4200, 2064), (1500, 1030, 660),
                                             (1100, 1300, 1001), (4000, 4100, 1189), (100, 3000, 1003),
                                             (9, 7000, 1030), (20, 20, 5569), (3000, 40, 2002)])
def test_large_tiles(ctx, rows, n_out, n_in):
    rng = np.random.default_rng([rows, n_out, n_in])
    x = rng.integers(-128, 128, (rows, n_in), dtype=np.int8)
    w = rng.integers(-128, 128, (n_out, n_in), dtype=np.int8)
    say("[i8 large]", rows, n_out, n_in)
    y = Result(ctx, rows, n_out, "i32", ld=n_out + 3)
    ctx.i8_matmul(ctx.upload(x), ctx.upload(w), rows, n_out, n_in, y.at, ld_y=n_out + 3)
    want = wide_sums(x, w)
    assert np.array_equal(y.read(), want)
    sx, sw = (np.exp(rng.normal(-6, 0.5, n)).astype(np.float32) for n in (rows, n_out))
    y = Result(ctx, rows, n_out, "bf16")
    ctx.i8_matmul(ctx.upload(x), ctx.upload(w), rows, n_out, n_in, y.at, z.BF16, x_scale=ctx.upload(sx),
                  w_scale=ctx.upload(sw))
    v = want * (sx.astype(np.float64)[:, None] * sw.astype(np.float64))
    near(y.read(), v, np.abs(v), "bf16")


# many short rows: one and two halves of 64 bytes, at whole words and not, up to
# three times 16 channels
@pytest.mark.parametrize("rows,n_out,n_in,pad,kind", [(4096, 32, 64, 0, "i32"), (5001, 10, 64, 0, "f32"),
                                                      (5001, 48, 128, 0, "bf16"), (4103, 47, 100, 0, "f32"),
                                                      (4111, 33, 17, 0, "f16"), (4096, 16, 16, 5, "i32"),
                                                      (4100, 3, 127, 0, "bf16"), (4099, 31, 65, 2, "i32"),
                                                      (300001, 1, 33, 0, "i32"), (270000, 21, 63, 1, "f32"),
                                                      (4095, 48, 128, 0, "i32"), (4096, 49, 64, 0, "i32")])
def test_many_short_rows(ctx, rows, n_out, n_in, pad, kind):
    rng = np.random.default_rng([rows, n_out, n_in])
    x = rng.integers(-128, 128, (rows, n_in), dtype=np.int8)
    w = rng.integers(-128, 128, (n_out, n_in), dtype=np.int8)
    say("[i8 short rows]", kind, rows, n_out, n_in, pad)
    y = Result(ctx, rows, n_out, kind, ld=n_out + pad)
    padded = lambda a: ctx.upload(np.pad(a, ((0, 0), (0, pad)), constant_values=99))  # noqa: E731
    want = wide_sums(x, w)
    if kind == "i32":
        ctx.i8_matmul(padded(x), padded(w), rows, n_out, n_in, y.at, ld_x=n_in + pad, ld_w=n_in + pad, ld_y=n_out + pad,
                      relu=True)
        assert np.array_equal(y.read(), np.maximum(want, 0))
        return
    sx, sw = (np.exp(rng.normal(-6, 0.5, n)).astype(np.float32) for n in (rows, n_out))
    b = rng.normal(0, 1, n_out).astype(np.float32)
    ctx.i8_matmul(padded(x), padded(w), rows, n_out, n_in, y.at, TYPES[kind], x_scale=ctx.upload(sx), w_scale=ctx.upload(sw),
                  bias=ctx.upload(b), ld_x=n_in + pad, ld_w=n_in + pad, ld_y=n_out + pad)
    v = want * (sx.astype(np.float64)[:, None] * sw.astype(np.float64))
    near(y.read(), v + b, np.abs(v) + np.abs(b), kind)


def test_longest_sum(ctx):
    """The largest sum of the longest row: 2^14 * 131071 < 2^31."""
    n_in = 131071
    x = np.full((2, n_in), -128, dtype=np.int8)
    x[1] = 127
    w = np.full((3, n_in), -128, dtype=np.int8)
    y = Result(ctx, 2, 3, "i32")
    say("[i8 longest]")
    ctx.i8_matmul(matrix(ctx, x), matrix(ctx, w), 2, 3, n_in, y.at)
    assert np.array_equal(y.read(), x.astype(np.int64) @ w.astype(np.int64).T)
    with pytest.raises(z.ZkError, match="131071"):
        ctx.i8_matmul(matrix(ctx, x[:, :1]), matrix(ctx, w[:, :1]), 1, 1, n_in + 1, y.at)


@pytest.mark.parametrize("rows", [0, 1, 70])
def test_empty_sizes(ctx, rows):
    """No rows, no channels: nothing is written.  No inputs: the sum is zero."""
    b = np.array([1.5, -2.0, 0.25], dtype=np.float32)
    one = ctx.upload(np.ones(256, dtype=np.int8))
    say("[i8 empty]", rows)
    y = Result(ctx, rows, 3, "f32")
    ctx.i8_matmul(one, one, rows, 3, 0, y.at, z.F32, bias=ctx.upload(b), relu=True)
    assert np.array_equal(y.read(), np.tile(np.maximum(b, 0), (rows, 1)))
    y = Result(ctx, rows, 3, "f32")
    ctx.i8_matmul(one, one, rows, 0, 3, y.at, z.F32, ld_y=3)
    ctx.i8_matmul(one, one, 0, 3, 3, y.at, z.F32)
    assert (y.ctx.d2h(y.buf, (y.size,), np.uint32) == 0xAAAAAAAA).all()
    y = Result(ctx, rows, 3, "f32")
    ctx.i8_linear(one, z.F32, one, None, rows, 3, 0, y.at, z.F32,
                  ctx.alloc(max(1, ctx.i8_linear_work(rows, 0))), bias=ctx.upload(b))
    assert np.array_equal(y.read(), np.tile(b, (rows, 1)))


@pytest.mark.parametrize("rows", [1, 100])
def test_scales_that_are_not_numbers(ctx, rows):
    """A NaN scale shows in its row or channel only, ReLU or not."""
    x, w = np.ones((rows, 20), dtype=np.int8), np.ones((5, 20), dtype=np.int8)
    sx, sw = np.ones(rows, dtype=np.float32), np.ones(5, dtype=np.float32)
    sx[0], sw[3] = np.nan, np.inf
    y = Result(ctx, rows, 5, "bf16")
    ctx.i8_matmul(matrix(ctx, x), matrix(ctx, w), rows, 5, 20, y.at, z.BF16, x_scale=ctx.upload(sx),
                  w_scale=ctx.upload(sw), relu=True)
    got = values(y.read(), "bf16")
    assert np.isnan(got[0]).all()
    assert (got[1:, [0, 1, 2, 4]] == 20).all() and np.isposinf(got[1:, 3]).all()


def test_offsets_past_32_bits(ctx):
    """Rows of x, w and y that start above 4 GiB from the first."""
    rows, n_out, n_in, ld = 3, 3, 100, (1 << 31) + 48
    rng = np.random.default_rng(1)
    x = rng.integers(-128, 128, (rows, n_in)).astype(np.int8)
    w = rng.integers(-128, 128, (n_out, n_in)).astype(np.int8)
    big, big2 = ctx.alloc(2 * ld + n_in), ctx.alloc(2 * ld + n_in)
    say("[i8 64-bit offsets]")
    for r in range(3):
        ctx.h2d(At(big, r * ld), x[r])
        ctx.h2d(At(big2, r * ld), w[r])
    y = ctx.alloc(2 * ld * 4 + 16)
    ctx.i8_matmul(big, big2, rows, n_out, n_in, y, ld_x=ld, ld_w=ld, ld_y=ld)
    want = x.astype(np.int64) @ w.astype(np.int64).T
    for r in range(3):
        assert np.array_equal(ctx.d2h(At(y, r * ld * 4), (3,), np.int32), want[r])


# ------------------------------------------------------------ rows to 8 bits
def quantized(x, kind):
    """(q, s) in 64 bits from the type's own values."""
    v = values(x, kind)
    a = np.abs(v).max(axis=1, initial=0.0)
    with np.errstate(all="ignore"):
        q = np.where(a[:, None] > 0, np.rint(127 * v / a[:, None]), 0.0)
    s = a / 127
    bad = ~np.isfinite(v).all(axis=1)
    q[bad], s[bad] = 0, np.nan
    return q, s


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,lead,pad", [(1, 1, 0, 0), (3, 7, 1, 2), (5, 64, 0, 0), (4, 1000, 3, 5),
                                                (2, 4096, 0, 0), (7, 8200, 8, 8), (1, 40000, 1, 0), (33, 129, 0, 1)])
def test_quantize(ctx, kind, rows, cols, lead, pad):
    rng = np.random.default_rng([rows, cols])
    v = rng.normal(0, 1, (rows, cols)) * np.exp(rng.normal(0, 2, (rows, 1)))
    x = words(v, kind)
    say("[i8 quantize]", kind, rows, cols, lead, pad)
    q = Result(ctx, rows, cols, "i8", ld=cols + pad, lead=lead)
    s = Result(ctx, 1, rows, "f32")
    ctx.i8_quantize(matrix(ctx, x, cols + pad, lead), TYPES[kind], rows, cols, q.at, s.at, ld_x=cols + pad,
                    ld_q=cols + pad)
    want, scale = quantized(x, kind)
    got = q.read().astype(np.int64)
    # 16-bit values: 127 x is exact in 32 bits and the division has one
    # rounding, so the nearest integer is that of the exact quotient; 32-bit
    # values: two roundings, so a quotient within 2^-16 of a half may go either way
    if kind == "f32":
        v = values(x, kind)
        exact = 127 * v / np.abs(v).max(axis=1)[:, None]
        edge = np.abs(np.abs(exact - np.floor(exact)) - 0.5) < 2.0**-16
        assert np.array_equal(got[~edge], want[~edge]) and (np.abs(got - exact) <= 0.5 + 2.0**-16).all()
    else:
        assert np.array_equal(got, want)
    assert (np.abs(s.read()[0] - scale) <= scale * 2.0**-24).all()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cols", [5, 300, 4096])
def test_quantize_edges(ctx, kind, cols):
    """Rows of zeros, one value alone, half-way quotients, values near the ends
    of the type, infinities and NaN."""
    top = {"f32": 3.0e38, "f16": 65504.0, "bf16": 3.0e38}[kind]
    low = {"f32": 2.0**-130, "f16": 2.0**-24, "bf16": 2.0**-120}[kind]
    rows = np.zeros((9, cols))
    rows[1, cols - 1] = -3.0
    rows[2, :3] = [127.0, 0.5, 1.5]
    rows[3, :3] = [2.0, 1.0, -1.0]  # 63.5: to 64
    rows[4, :3] = [top, -top / 2, top / 4]
    rows[5, :3] = [low, low, 0]
    rows[6, 0], rows[6, 1] = np.inf, 1
    rows[7, 0], rows[7, cols - 1] = 1, np.nan
    rows[8, 0] = -np.inf
    x = words(rows, kind)
    q, s = Result(ctx, 9, cols, "i8"), Result(ctx, 1, 9, "f32")
    say("[i8 quantize edges]", kind, cols)
    ctx.i8_quantize(matrix(ctx, x), TYPES[kind], 9, cols, q.at, s.at)
    want, scale = quantized(x, kind)
    got, gs = q.read(), s.read()[0].astype(np.float64)
    assert np.array_equal(got, want)
    assert np.isnan(gs[6:]).all() and gs[0] == 0 and got[3, 1] == 64
    # 2^-130 / 127 is below the smallest normal number: half a unit of 2^-149
    assert (np.abs(gs[:6] - scale[:6]) <= scale[:6] * 2.0**-24 + 2.0**-150).all()


@pytest.mark.parametrize("kind,out", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("rows,n_out,n_in,pad", [(1, 100, 4096, 0), (1, 1, 1, 0), (1, 513, 1001, 3), (2, 64, 64, 0),
                                                 (4, 33, 300, 1), (9, 200, 1000, 8), (70, 130, 515, 0),
                                                 (300, 256, 1024, 0), (5, 8200, 9000, 0), (16, 8195, 2900, 1),
                                                 (3, 70, 15000, 0), (16, 40, 3000, 2), (17, 50, 2000, 0),
                                                 (3, 8200, 16200, 0), (16, 8193, 2900, 0),
                                                 (2, 30, 16, 0), (2, 30, 15, 0)])
def test_linear(ctx, kind, out, rows, n_out, n_in, pad):
    """The linear layer is the product over its rows' quantized values: compared
    with the 64-bit product of the library's own q and s, which test_quantize
    checks, so that no half-way case matters here."""
    rng = np.random.default_rng([rows, n_out, n_in])
    x = words(rng.normal(0, 1, (rows, n_in)) * np.exp(rng.normal(0, 1, (rows, 1))), kind)
    if rows > 2:
        x[2] = 0
    w = rng.integers(-127, 128, (n_out, n_in)).astype(np.int8)
    sw = np.exp(rng.normal(-5, 0.5, n_out)).astype(np.float32)
    b = rng.normal(0, 1, n_out).astype(np.float32)
    say("[i8 linear]", kind, out, rows, n_out, n_in)
    xd, wd = matrix(ctx, x, n_in + pad), matrix(ctx, w, n_in + pad)
    q, s = Result(ctx, rows, n_in, "i8"), Result(ctx, 1, rows, "f32")
    ctx.i8_quantize(xd, TYPES[kind], rows, n_in, q.at, s.at, ld_x=n_in + pad)
    work = ctx.alloc(ctx.i8_linear_work(rows, n_in))
    y = Result(ctx, rows, n_out, out, ld=n_out + pad)
    ctx.i8_linear(xd, TYPES[kind], wd, ctx.upload(sw), rows, n_out, n_in, y.at, TYPES[out], work, bias=ctx.upload(b),
                  ld_x=n_in + pad, ld_w=n_in + pad, ld_y=n_out + pad)
    acc = (q.read().astype(np.int64) @ w.astype(np.int64).T).astype(np.float64)
    v = acc * s.read()[0].astype(np.float64)[:, None] * sw.astype(np.float64)
    near(y.read(), v + b, np.abs(v) + np.abs(b), out)


def test_linear_row_with_nan(ctx):
    for rows in (1, 3, 100):
        x = np.ones((rows, 50), dtype=np.float32)
        x[0, 7] = np.nan
        w = np.ones((4, 50), dtype=np.int8)
        y = Result(ctx, rows, 4, "f32")
        ctx.i8_linear(matrix(ctx, x), z.F32, matrix(ctx, w), None, rows, 4, 50, y.at, z.F32,
                      ctx.alloc(ctx.i8_linear_work(rows, 50)), relu=True)
        got = y.read()
        assert np.isnan(got[0]).all() and np.isfinite(got[1:]).all()


# ------------------------------------------------------------ experts' products
def routed(rng, tokens, slots, experts, dropped=0.0, skew=0.0):
    """(offsets, order) of a random route, in numpy."""
    p = np.exp(-skew * np.arange(experts))
    e = rng.choice(experts, size=tokens * slots, p=p / p.sum())
    e[rng.random(tokens * slots) < dropped] = experts
    order = np.argsort(e, kind="stable")
    offsets = np.searchsorted(e[order], np.arange(experts + 1)).astype(np.int32)
    order[offsets[-1]:] = -1
    return offsets, order.astype(np.int32)


@pytest.mark.parametrize("kind", ["i32", "f32", "bf16"])
@pytest.mark.parametrize("tokens,slots,experts,n_out,n_in,dropped,skew", [
    (1, 1, 1, 5, 16, 0, 0), (1, 2, 8, 130, 1000, 0, 0), (5, 2, 16, 64, 256, 0.3, 0), (40, 2, 3, 65, 129, 0, 1),
    (33, 4, 64, 100, 64, 0.1, 0.1), (300, 2, 5, 70, 333, 0.2, 1), (700, 1, 2, 257, 128, 0, 3),
    (128, 8, 128, 31, 40, 0, 0), (600, 4, 4, 256, 512, 0.05, 0.5), (3, 1, 1024, 20, 30, 0, 0)])
def test_experts_product(ctx, kind, tokens, slots, experts, n_out, n_in, dropped, skew):
    rng = np.random.default_rng([tokens, slots, experts])
    offsets, order = routed(rng, tokens, slots, experts, dropped, skew)
    x = rng.integers(-127, 128, (tokens, n_in)).astype(np.int8)
    w = rng.integers(-127, 128, (experts * n_out, n_in)).astype(np.int8)
    scaled = kind != "i32"
    sx = np.exp(rng.normal(-5, 0.5, tokens)).astype(np.float32)
    sw = np.exp(rng.normal(-5, 0.5, (experts, n_out))).astype(np.float32)
    b = rng.normal(0, 1, (experts, n_out)).astype(np.float32)
    rows = tokens * slots
    say("[i8 experts]", kind, tokens, slots, experts, n_out, n_in)
    y = Result(ctx, rows, n_out, kind, ld=n_out + 3)
    more = dict(x_scale=ctx.upload(sx), w_scale=ctx.upload(sw), bias=ctx.upload(b)) if scaled else {}
    ctx.i8_matmul_experts(matrix(ctx, x, n_in + 5), matrix(ctx, w), ctx.upload(offsets), rows, experts, n_out, n_in,
                          y.at, TYPES[kind], order=ctx.upload(order), slots=slots, tokens=tokens, ld_x=n_in + 5,
                          ld_y=n_out + 3, **more)
    got = y.read()
    used = offsets[-1]
    token = order[:used] // slots
    e = np.searchsorted(offsets[1:], np.arange(used), side="right")
    acc = np.zeros((rows, n_out), dtype=np.int64)
    for i in range(experts):
        at = slice(offsets[i], offsets[i + 1])
        acc[at] = x[token[at]].astype(np.int64) @ w[i * n_out:(i + 1) * n_out].astype(np.int64).T
    assert not got[used:].any()
    if not scaled:
        assert np.array_equal(got, acc)
        return
    v = acc[:used] * sx.astype(np.float64)[token][:, None] * sw.astype(np.float64)[e]
    near(got[:used], v + b[e], np.abs(v) + np.abs(b[e]), kind)


@pytest.mark.parametrize("tokens,slots,experts,n_out,n_in,skew", [(2000, 4, 8, 700, 1040, 0.3),
                                                                  (2000, 4, 8, 700, 1041, 0.3),
                                                                  (3000, 3, 3, 2100, 1056, 0.5),
                                                                  (3000, 3, 3, 2100, 1057, 0.5),
                                                                  (2600, 4, 2, 2100, 2064, 0.2),
                                                                  (900, 8, 200, 300, 272, 0.02)])
def test_experts_product_large(ctx, tokens, slots, experts, n_out, n_in, skew):
    """The large tiles with rows by expert, some of them dropped."""
    rng = np.random.default_rng([tokens, experts, n_in])
    offsets, order = routed(rng, tokens, slots, experts, 0.05, skew)
    x = rng.integers(-127, 128, (tokens, n_in), dtype=np.int8)
    w = rng.integers(-127, 128, (experts * n_out, n_in), dtype=np.int8)
    rows = tokens * slots
    say("[i8 experts large]", tokens, slots, experts, n_out, n_in)
    y = Result(ctx, rows, n_out, "i32")
    ctx.i8_matmul_experts(ctx.upload(x), ctx.upload(w), ctx.upload(offsets), rows, experts, n_out, n_in, y.at,
                          order=ctx.upload(order), slots=slots, tokens=tokens)
    got = y.read()
    for e in range(experts):
        at = slice(offsets[e], offsets[e + 1])
        assert np.array_equal(got[at], wide_sums(x[order[at] // slots], w[e * n_out:(e + 1) * n_out])), e
    assert not got[offsets[-1]:].any()


def test_experts_product_without_an_order(ctx):
    """Rows that are sorted already: row p of x, its own scale."""
    rng = np.random.default_rng(3)
    offsets = np.array([0, 0, 3, 70, 70, 71], dtype=np.int32)
    x = rng.integers(-127, 128, (71, 90)).astype(np.int8)
    w = rng.integers(-127, 128, (5 * 40, 90)).astype(np.int8)
    y = Result(ctx, 71, 40, "i32")
    ctx.i8_matmul_experts(matrix(ctx, x), matrix(ctx, w), ctx.upload(offsets), 71, 5, 40, 90, y.at)
    got = y.read()
    for e in range(5):
        at = slice(offsets[e], offsets[e + 1])
        assert np.array_equal(got[at], x[at].astype(np.int64) @ w[40 * e:40 * e + 40].astype(np.int64).T)


def test_experts_product_takes_bad_indexes_as_none(ctx):
    """Order values that name no token give zeros; offsets above the rows are
    taken as the rows."""
    x, w = np.ones((2, 20), dtype=np.int8), np.ones((2 * 3, 20), dtype=np.int8)
    order = np.array([0, 7, -1, 1 << 30], dtype=np.int32)
    offsets = np.array([0, 2, 1000], dtype=np.int32)
    y = Result(ctx, 4, 3, "i32")
    ctx.i8_matmul_experts(matrix(ctx, x), matrix(ctx, w), ctx.upload(offsets), 4, 2, 3, 20, y.at,
                          order=ctx.upload(order), slots=1, tokens=2)
    got = y.read()
    assert (got[0] == 20).all() and not got[1:].any()


@pytest.mark.parametrize("n_in", [8, 300])
def test_experts_product_without_tokens(ctx, n_in):
    """No token: every row is zero, and nothing of x is read."""
    order = np.zeros(70, dtype=np.int32)
    y = Result(ctx, 70, 5, "f32")
    ctx.i8_matmul_experts(ctx.alloc(1), matrix(ctx, np.ones((2 * 5, n_in), dtype=np.int8)),
                          ctx.upload(np.array([0, 30, 70], dtype=np.int32)), 70, 2, 5, n_in, y.at, z.F32,
                          order=ctx.upload(order), slots=1, tokens=0)
    assert not y.read().any()


# ------------------------------------------------------------ refusals, streams
def test_refusals(ctx):
    d = ctx.alloc(4096)

    def mm(**k):
        a = dict(x=d, w=d, rows=2, n_out=3, n_in=16, y=d, y_type=z.F32)
        a.update(k)
        x, w, rows, n_out, n_in, y = (a.pop(n) for n in ("x", "w", "rows", "n_out", "n_in", "y"))
        ctx.i8_matmul(x, w, rows, n_out, n_in, y, **a)

    for bad, why in [(dict(x=None), "null"), (dict(w=None), "null"), (dict(y=None), "null"),
                     (dict(ld_x=15), "stride"), (dict(ld_w=15), "stride"), (dict(ld_y=2), "stride"),
                     (dict(y_type=4), "type"), (dict(y_type=-1), "type"), (dict(y=At(d, 2)), "aligned"),
                     (dict(x_scale=At(d, 1)), "aligned"), (dict(w_scale=At(d, 2)), "aligned"),
                     (dict(bias=At(d, 3)), "aligned"), (dict(y_type=z.I32, bias=d), "no bias"),
                     (dict(y_type=z.I32, x_scale=d), "no scales"), (dict(n_in=131072, ld_x=131072, ld_w=131072), "131071"),
                     (dict(rows=1 << 31), "2\\^31"), (dict(n_out=1 << 31, ld_y=1 << 31), "2\\^31"),
                     (dict(n_out=(1 << 26) + 1, ld_y=1 << 27), "2\\^26")]:
        with pytest.raises(z.ZkError, match=why):
            mm(**bad)
    for args, why in [((None, z.F32, 1, 4, d, d), "null"), ((d, z.I32, 1, 4, d, d), "f32, f16 or bf16"),
                      ((d, z.F32, 1, 4, None, d), "null"), ((d, z.F32, 1, 4, d, None), "null"),
                      ((At(d, 2), z.F32, 1, 4, d, d), "aligned"), ((d, z.F32, 1 << 31, 4, d, d), "2\\^31")]:
        with pytest.raises(z.ZkError, match=why):
            ctx.i8_quantize(*args)
    with pytest.raises(z.ZkError, match="stride"):
        ctx.i8_quantize(d, z.F32, 2, 4, d, d, ld_x=3)
    with pytest.raises(z.ZkError, match="stride"):
        ctx.i8_quantize(d, z.F32, 2, 4, d, d, ld_q=3)
    small = ctx.alloc(ctx.i8_linear_work(2, 16) - 1)
    for work in (None, small, At(d, 8)):
        with pytest.raises(z.ZkError, match="workspace"):
            ctx.i8_linear(d, z.F32, d, d, 2, 3, 16, d, z.F32, work)
    with pytest.raises(z.ZkError, match="f32, f16 or bf16"):
        ctx.i8_linear(d, z.F32, d, d, 2, 3, 16, d, z.I32, d)
    for bad, why in [(dict(experts=0), "1024"), (dict(experts=1025), "1024"), (dict(slots=0), "slots"),
                     (dict(offsets=None), "null"), (dict(rows=(1 << 22) + 1), "too many"),
                     (dict(order=At(d, 2)), "aligned"), (dict(offsets=At(d, 1)), "aligned")]:
        a = dict(x=d, w=d, offsets=d, rows=2, experts=2, n_out=3, n_in=16, y=d)
        a.update(bad)
        with pytest.raises(z.ZkError, match=why):
            ctx.i8_matmul_experts(**a)
    assert z.lib().zk_i8_matmul(None, None, 0, None, None, 0, None, None, 0, 0, 0, 0, None, 0, 0, None) == 1
    assert ctx.i8_linear_work(1 << 31, 4) == 0 and ctx.i8_linear_work(4, 131072) == 0


def test_other_streams_and_graphs(ctx):
    """Calls on a stream of the caller's, on the default stream, and recorded
    into a graph that is replayed on new inputs between eager calls."""
    hip, vp = ctypes.CDLL("libamdhip64.so"), ctypes.c_void_p
    rng = np.random.default_rng(1)
    rows, n_out, n_in = 20, 70, 300
    w = ctx.upload(rng.integers(-127, 128, (n_out, n_in)).astype(np.int8))
    sw = ctx.upload(rng.random(n_out).astype(np.float32))
    x, work = ctx.alloc(rows * n_in * 4), ctx.alloc(ctx.i8_linear_work(rows, n_in))
    y, ref = ctx.alloc(rows * n_out * 4), ctx.alloc(rows * n_out * 4)

    def call(out, on):
        ctx.i8_linear(x, z.F32, w, sw, rows, n_out, n_in, out, z.F32, work, stream=on)

    def fresh():
        ctx.h2d(x, rng.normal(0, 1, (rows, n_in)).astype(np.float32))
        ctx.h2d(y, np.zeros((rows, n_out), dtype=np.float32))

    def same():
        call(ref, None)  # the context's own stream: the tests above check it
        ctx.sync()
        got = ctx.d2h(y, (rows, n_out), np.float32)
        assert got.any() and np.array_equal(got, ctx.d2h(ref, (rows, n_out), np.float32))

    say("[i8 streams]")
    fresh()
    call(y, z.LEGACY_STREAM)
    assert hip.hipDeviceSynchronize() == 0
    same()
    st, graph, exe = vp(), vp(), vp()
    assert hip.hipStreamCreate(ctypes.byref(st)) == 0
    try:
        fresh()
        call(y, st)
        assert hip.hipStreamSynchronize(st) == 0
        same()
        assert hip.hipStreamBeginCapture(st, 0) == 0
        call(y, st)
        assert hip.hipStreamEndCapture(st, ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0)) == 0
        for _ in range(4):
            fresh()
            assert hip.hipGraphLaunch(exe, st) == 0
            assert hip.hipStreamSynchronize(st) == 0
            same()
    finally:
        if exe:
            hip.hipGraphExecDestroy(exe)
        if graph:
            hip.hipGraphDestroy(graph)
        hip.hipStreamDestroy(st)


def test_a_statement_s_scores(ctx):
    """The integers of the product are those a statement proves: one linear
    layer over a batch, against the statement builder's scores."""
    rng = np.random.default_rng(5)
    w, b = rng.integers(-127, 128, (10, 64)), rng.integers(-1000, 1000, 10)
    x = rng.integers(0, 17, (6, 64))
    st = z.statement_v2([z.layer_linear(64, 10, w, b)], x)
    y = Result(ctx, 6, 10, "i32")
    ctx.i8_matmul(matrix(ctx, x.astype(np.int8)), matrix(ctx, w.astype(np.int8)), 6, 10, 64, y.at)
    assert np.array_equal(y.read() + b, st.scores)
