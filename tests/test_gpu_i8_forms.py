"""GPU tests of what an 8-bit layer makes of its sums (cuda-zkml_amd/csrc/i8_matmul.hip):
(float(acc) * x_scale) * w_scale + bias with each operation rounded to 32 bits, then
once to the result's type.  numpy's float32 operations in the same order give the
same bits, so nothing here has a tolerance.
"""
import numpy as np
import pytest

import zkml_amd as z
from i8_helpers import TYPES, At, Result, matrix, values, words
from i8_sizes import GROUPED, PLAIN, listed

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return z.Context(0)


def say(*a):
    print(*a, flush=True)


def elementary(acc, sx, sw, b, relu, kind):
    """The definition in numpy's float32.  Token scales from 2^96 on: a power of two
    moved to the channels' scales, which changes no rounding and keeps float(acc) sx
    inside the 32-bit floats."""
    up = np.where(np.abs(sx) >= 2.0**96, np.float32(2.0**32), np.float32(1))
    with np.errstate(over="ignore", under="ignore"):
        y = (acc.astype(np.float32) * (sx / up)[:, None]) * (sw[None, :] * up[:, None]) + b
        if relu:
            y = np.where(y < 0, np.float32(0), y)
        assert y.dtype == np.float32
        return words(y, kind)


# rows, n_out, n_in: rows under 16 bytes, many short rows, few rows, rows at whole
# 16 bytes and not
FORMS = [(5, 7, 8), (5000, 32, 64), (9, 40, 200), (1000, 600, 512), (1000, 600, 513)]
# the scales' logarithms: ordinary ones; a product below the 32-bit floats, whose
# results are inside; one above them, where only sums of zero are finite; a token's
# scale near either end that the channel's brings back
SCALES = {"ordinary": (-6, -6), "below": (-69, -28), "above": (69, 27), "token high": (80, -70), "token low": (-86, 70)}


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scales", list(SCALES))
@pytest.mark.parametrize("rows,n_out,n_in", FORMS)
def test_results_are_those_of_the_elementary_operations(ctx, kind, scales, rows, n_out, n_in):
    rng = np.random.default_rng([rows, n_out, n_in, len(scales)])
    x = rng.integers(-127, 128, (rows, n_in)).astype(np.int8)
    w = rng.integers(-127, 128, (n_out, n_in)).astype(np.int8)
    x[1] = 0  # sums of zero are zero whatever the scales are
    acc = x.astype(np.int64) @ w.astype(np.int64).T
    lx, lw = SCALES[scales]
    sx, sw = (np.exp(rng.normal(m, 0.5, n)).astype(np.float32) for m, n in ((lx, rows), (lw, n_out)))
    b = rng.normal(0, 1, n_out).astype(np.float32) if scales == "ordinary" else np.zeros(n_out, dtype=np.float32)
    say("[i8 forms]", kind, scales, rows, n_out, n_in)
    for bias, relu in ((None, False), (b, True)):
        y = Result(ctx, rows, n_out, kind)
        ctx.i8_matmul(matrix(ctx, x), matrix(ctx, w), rows, n_out, n_in, y.at, TYPES[kind], x_scale=ctx.upload(sx),
                      w_scale=ctx.upload(sw), bias=None if bias is None else ctx.upload(bias), relu=relu)
        want = elementary(acc, sx, sw, np.float32(0) if bias is None else bias, relu, kind)
        assert np.array_equal(y.read(), want)


@pytest.mark.parametrize("rows", [3, 40])
def test_linear_at_the_ends_of_the_range(ctx, rows):
    """Rows near the largest 32-bit float and near the smallest, and channels that
    bring them back: the results are those of the quantized rows."""
    rng = np.random.default_rng(rows)
    n_out, n_in = 50, 300
    for size, back in ((2e38, -76), (1e-34, 66)):
        x = (rng.uniform(-1, 1, (rows, n_in)) * size).astype(np.float32)
        w = rng.integers(-127, 128, (n_out, n_in)).astype(np.int8)
        sw = np.exp(rng.normal(back, 0.5, n_out)).astype(np.float32)
        xd, q, s = matrix(ctx, x), Result(ctx, rows, n_in, "i8"), Result(ctx, 1, rows, "f32")
        ctx.i8_quantize(xd, z.F32, rows, n_in, q.at, s.at)
        y = Result(ctx, rows, n_out, "f32")
        say("[i8 linear ends]", rows, size)
        ctx.i8_linear(xd, z.F32, matrix(ctx, w), ctx.upload(sw), rows, n_out, n_in, y.at, z.F32,
                      ctx.alloc(ctx.i8_linear_work(rows, n_in)))
        got = y.read()
        want = elementary(q.read().astype(np.int64) @ w.astype(np.int64).T, s.read()[0], sw, np.float32(0), False, "f32")
        assert np.array_equal(got, want) and np.isfinite(got).all() and got.any()


@pytest.mark.parametrize("exponent", [-100, -65, 0, 63, 100])
def test_f32_quotients_beside_a_half(ctx, exponent):
    """An f32 row's integers are those of 127 x and its quotient rounded to 32 bits
    each, also where these roundings end on the other side of a half than the exact
    quotient (71.49999974 and 60.50000069 in the first two rows)."""
    rng = np.random.default_rng(exponent + 200)
    rows, cols = 64, 129
    x = np.zeros((rows, cols), dtype=np.float32)
    x[:, 0] = np.concatenate([[11694970, 16616451], rng.integers(1 << 23, 1 << 24, rows - 2)]) * 2.0**-23
    half = (rng.integers(0, 127, (rows, cols - 1)) + 0.5) * x[:, :1] / 127
    x[:, 1:] = half.astype(np.float32) + rng.integers(-2, 3, half.shape) * np.spacing(half.astype(np.float32))
    x[:, 1:] *= rng.choice([-1, 1], half.shape)
    x[0, 1], x[1, 1] = 6584176 * 2.0**-23, 7915711 * 2.0**-23
    x = np.clip(x, -x[:, :1], x[:, :1])
    x = np.ldexp(x, exponent)
    q, s = Result(ctx, rows, cols, "i8"), Result(ctx, 1, rows, "f32")
    say("[i8 halves]", exponent)
    ctx.i8_quantize(matrix(ctx, x), z.F32, rows, cols, q.at, s.at)
    got, want = q.read(), np.rint((np.float32(127) * x) / x[:, :1])
    assert want.dtype == np.float32 and np.array_equal(got, want) and got[0, 1] == 72 and got[1, 1] == 60
    assert np.array_equal(s.read()[0], x[:, 0] / np.float32(127))
    # and so does the linear layer of few rows, which quantizes on the way
    w = np.eye(cols, dtype=np.int8)
    y = Result(ctx, 8, cols, "f32")
    ctx.i8_linear(matrix(ctx, x[:8]), z.F32, matrix(ctx, w), None, 8, cols, cols, y.at, z.F32,
                  ctx.alloc(ctx.i8_linear_work(8, cols)))
    assert np.array_equal(y.read(), want[:8] * s.read()[0][:8, None])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,slots,experts,n_out,n_in", [(5, 2, 4, 7, 8), (5, 2, 4, 40, 200), (900, 2, 3, 300, 272)])
def test_experts_results_are_those_of_the_elementary_operations(ctx, kind, tokens, slots, experts, n_out, n_in):
    rng = np.random.default_rng([tokens, n_out, n_in])
    rows = tokens * slots
    e = np.sort(rng.integers(0, experts, rows))
    offsets = np.searchsorted(e, np.arange(experts + 1)).astype(np.int32)
    order = rng.permutation(rows).astype(np.int32)
    x = rng.integers(-127, 128, (tokens, n_in)).astype(np.int8)
    w = rng.integers(-127, 128, (experts, n_out, n_in)).astype(np.int8)
    for lx, lw in SCALES.values():
        sx = np.exp(rng.normal(lx, 0.5, tokens)).astype(np.float32)
        sw = np.exp(rng.normal(lw, 0.5, (experts, n_out))).astype(np.float32)
        y = Result(ctx, rows, n_out, kind)
        say("[i8 experts forms]", kind, tokens, n_out, n_in, lx, lw)
        ctx.i8_matmul_experts(matrix(ctx, x), matrix(ctx, w.reshape(-1, n_in)), ctx.upload(offsets), rows, experts,
                              n_out, n_in, y.at, TYPES[kind], x_scale=ctx.upload(sx), w_scale=ctx.upload(sw),
                              order=ctx.upload(order), slots=slots, tokens=tokens)
        got = y.read()
        for i in range(experts):
            at = slice(offsets[i], offsets[i + 1])
            t = order[at] // slots
            acc = x[t].astype(np.int64) @ w[i].astype(np.int64).T
            assert np.array_equal(got[at], elementary(acc, sx[t], sw[i], np.float32(0), False, kind)), i


# ------------------------------------------------------------ every kernel, every type
def sums(x, w):
    """The exact sums by way of float64, whose 53 bits hold them."""
    return (x.astype(np.float64) @ w.astype(np.float64).T).astype(np.int64)


# by type: bias, ReLU
EPILOGUES = {"i32": (False, True), "f32": (True, True), "f16": (True, False), "bf16": (False, True)}


@pytest.mark.parametrize("kernel,rows,n_out,n_in", listed(PLAIN))
def test_every_kernel_in_every_type(ctx, kernel, rows, n_out, n_in):
    rng = np.random.default_rng([rows, n_out, n_in])
    x = rng.integers(-128, 128, (rows, n_in), dtype=np.int8)
    w = rng.integers(-128, 128, (n_out, n_in), dtype=np.int8)
    sx, sw = (np.exp(rng.normal(-6, 0.5, n)).astype(np.float32) for n in (rows, n_out))
    b = rng.normal(0, 1, n_out).astype(np.float32)
    xd, wd, sxd, swd, bd = (ctx.upload(a) for a in (x, w, sx, sw, b))
    acc = sums(x, w)
    for kind, (bias, relu) in EPILOGUES.items():
        say("[i8 kernels]", kernel, kind, rows, n_out, n_in)
        y = Result(ctx, rows, n_out, kind, ld=n_out + 3)
        scaled = {} if kind == "i32" else dict(x_scale=sxd, w_scale=swd, bias=bd if bias else None)
        ctx.i8_matmul(xd, wd, rows, n_out, n_in, y.at, TYPES[kind], relu=relu, ld_y=n_out + 3, **scaled)
        if kind == "i32":
            want = np.maximum(acc, 0) if relu else acc
        else:
            want = elementary(acc, sx, sw, b if bias else np.float32(0), relu, kind)
        assert np.array_equal(y.read(), want), kind


@pytest.mark.parametrize("kernel,rows,n_out,n_in,experts", listed(GROUPED))
def test_every_kernel_by_expert_in_every_type(ctx, kernel, rows, n_out, n_in, experts):
    """Unevenly filled experts, one of them empty where there are several, and rows
    of none behind them."""
    rng = np.random.default_rng([rows, n_out, n_in, experts])
    slots = 2 if rows % 2 == 0 else 1
    tokens = rows // slots
    e = rng.choice(experts, size=rows, p=(p := np.exp(-0.3 * np.arange(experts))) / p.sum())
    if experts > 2:
        e[e == 1] = 0
    e[rng.random(rows) < 0.05] = experts
    order = np.argsort(e, kind="stable").astype(np.int32)
    offsets = np.searchsorted(e[order], np.arange(experts + 1)).astype(np.int32)
    used = offsets[-1]
    order[used:] = -1
    x = rng.integers(-127, 128, (tokens, n_in), dtype=np.int8)
    w = rng.integers(-127, 128, (experts, n_out, n_in), dtype=np.int8)
    sx = np.exp(rng.normal(-6, 0.5, tokens)).astype(np.float32)
    sw = np.exp(rng.normal(-6, 0.5, (experts, n_out))).astype(np.float32)
    b = rng.normal(0, 1, (experts, n_out)).astype(np.float32)
    xd, wd, sxd, swd, bd, fd, od = (ctx.upload(a) for a in (x, w, sx, sw, b, offsets, order))
    at = [slice(offsets[i], offsets[i + 1]) for i in range(experts)]
    acc = [sums(x[order[a] // slots], w[i]) for i, a in enumerate(at)]
    for kind, (bias, relu) in EPILOGUES.items():
        say("[i8 kernels by expert]", kernel, kind, rows, n_out, n_in, experts)
        y = Result(ctx, rows, n_out, kind, ld=n_out + 3)
        scaled = {} if kind == "i32" else dict(x_scale=sxd, w_scale=swd, bias=bd if bias else None)
        ctx.i8_matmul_experts(xd, wd, fd, rows, experts, n_out, n_in, y.at, TYPES[kind], relu=relu, order=od,
                              slots=slots, tokens=tokens, ld_y=n_out + 3, **scaled)
        got = y.read()
        assert not got[used:].any(), kind
        for i, a in enumerate(at):
            if kind == "i32":
                want = np.maximum(acc[i], 0) if relu else acc[i]
            else:
                want = elementary(acc[i], sx[order[a] // slots], sw[i], b[i] if bias else np.float32(0), relu, kind)
            assert np.array_equal(got[a], want), (kind, i)


@pytest.mark.parametrize("n_in", [8, 300])
def test_no_tokens_need_no_x(ctx, n_in):
    """An empty x has no address (a torch tensor's is 0): every row is zero."""
    y = Result(ctx, 70, 5, "f32")
    w = ctx.upload(np.ones((2 * 5, n_in), dtype=np.int8))
    offsets, order = ctx.upload(np.array([0, 30, 70], dtype=np.int32)), ctx.upload(np.zeros(70, dtype=np.int32))
    ctx.i8_matmul_experts(None, w, offsets, 70, 2, 5, n_in, y.at, z.F32, order=order, slots=1, tokens=0)
    assert not y.read().any()
    with pytest.raises(z.ZkError, match="null"):
        ctx.i8_matmul_experts(None, w, offsets, 70, 2, 5, n_in, y.at, z.F32, order=order, slots=1, tokens=1)


def test_rows_in_two_launches(ctx):
    """More than 2^22 tiles of 16 x 16: the rows from the 256th on are a launch of
    their own, with their own part of x, of the scales and of y."""
    rows, n_out, n_in, at = 259, 1 << 22, 16, 253
    rng = np.random.default_rng(2)
    x = rng.integers(-128, 128, (rows, n_in), dtype=np.int8)
    w = rng.integers(-128, 128, (n_out, n_in), dtype=np.int8)
    sx, sw = (np.exp(rng.normal(-6, 0.5, n)).astype(np.float32) for n in (rows, n_out))
    y = ctx.alloc(rows * n_out * 2)
    say("[i8 two launches]")
    ctx.i8_matmul(ctx.upload(x), ctx.upload(w), rows, n_out, n_in, y, z.BF16, x_scale=ctx.upload(sx),
                  w_scale=ctx.upload(sw))
    got = ctx.d2h(At(y, at * n_out * 2), (rows - at, n_out), np.uint16)
    # (sums below 2^24 are exact in 32-bit floats)
    acc = x[at:].astype(np.float32) @ w.astype(np.float32).T
    assert np.array_equal(got, elementary(acc, sx[at:], sw, np.float32(0), False, "bf16"))


# ------------------------------------------------------------ many rows to 8 bits
# pieces of 16 bytes a row: up to 64, to 256 and to 1024 at 2048 rows, at 512 and at
# fewer, and more
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(2100, 201), (2100, 1001), (600, 1001), (600, 4001), (600, 9001), (2100, 2501)])
def test_quantize_many_rows(ctx, kind, rows, cols):
    rng = np.random.default_rng([rows, cols])
    x = words(rng.normal(0, 1, (rows, cols)) * np.exp(rng.normal(0, 2, (rows, 1))), kind)
    q, s = Result(ctx, rows, cols, "i8", ld=cols + 1), Result(ctx, 1, rows, "f32")
    say("[i8 quantize]", kind, rows, cols)
    ctx.i8_quantize(ctx.upload(x), TYPES[kind], rows, cols, q.at, s.at, ld_q=cols + 1)
    v = values(x, kind).astype(np.float32)
    a = np.abs(v).max(axis=1)
    assert np.array_equal(q.read(), np.rint(np.float32(127) * v / a[:, None]))
    assert np.array_equal(s.read()[0], a / np.float32(127))


# at most 16 rows of at most 36 KB in 8 bits are quantized on the way, 16 channels a
# block or 32 (from 8192 on); more go through the quantizer
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n_out,n_in", [(1, 33, 17), (16, 70, 2047), (8, 100, 4062), (2, 100, 18000),
                                             (16, 8195, 2001), (8, 8200, 4062), (1, 8193, 36000), (3, 8193, 129),
                                             (9, 100, 4095), (1, 50, 37000), (17, 50, 300)])
def test_linear_of_few_rows(ctx, kind, rows, n_out, n_in):
    test_linear_of_many_rows(ctx, kind, rows, n_out, n_in)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n_out,n_in", [(700, 130, 4001), (2100, 300, 1008)])
def test_linear_of_many_rows(ctx, kind, rows, n_out, n_in):
    rng = np.random.default_rng([rows, n_in])
    x = words(rng.normal(0, 1, (rows, n_in)), kind)
    w = rng.integers(-127, 128, (n_out, n_in), dtype=np.int8)
    sw, b = np.exp(rng.normal(-5, 0.5, n_out)).astype(np.float32), rng.normal(0, 1, n_out).astype(np.float32)
    y = Result(ctx, rows, n_out, kind)
    say("[i8 linear]", kind, rows, n_out, n_in)
    ctx.i8_linear(ctx.upload(x), TYPES[kind], ctx.upload(w), ctx.upload(sw), rows, n_out, n_in, y.at, TYPES[kind],
                  ctx.alloc(ctx.i8_linear_work(rows, n_in)), bias=ctx.upload(b))
    v = values(x, kind).astype(np.float32)
    a = np.abs(v).max(axis=1)
    q = np.rint(np.float32(127) * v / a[:, None]).astype(np.int8)
    assert np.array_equal(y.read(), elementary(sums(q, w), a / np.float32(127), sw, b, False, kind))
