"""GPU tests of the layers with 4-bit weights (cuda-zkml_amd/csrc/i4_matmul.hip)
against their 64-bit form; the tolerances are those of i4_helpers.near."""
import numpy as np
import pytest

import zkml_amd as z
from i4_helpers import inputs, near, packed, product, unpacked, wide_product
from i4_sizes import GROUPED as GROUPED_SIZES, PLAIN, listed
from i8_helpers import TYPES, At, Result, matrix, values, words

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return z.Context(0)


def say(*a):
    print(*a, flush=True)


def up(ctx, a):
    return None if a is None else ctx.upload(a)


SIZES = [(1, 1, 1), (1, 1, 32), (1, 5, 31), (2, 16, 64), (1, 33, 65), (3, 20, 127), (4, 17, 128), (5, 64, 129),
         (1, 1000, 4096), (2, 300, 1001), (7, 130, 2050), (15, 31, 300), (16, 16, 128), (17, 65, 640), (31, 48, 1024),
         (33, 257, 259), (48, 100, 2048), (64, 64, 512), (65, 129, 384), (100, 200, 1000), (130, 300, 768),
         (260, 270, 1024), (513, 129, 897)]


@pytest.mark.parametrize("group", [32, 64, 128, 384])
@pytest.mark.parametrize("rows,n_out,n_in", SIZES)
def test_product(ctx, rows, n_out, n_in, group):
    rng = np.random.default_rng([rows, n_out, n_in, group])
    x, sx, q, s, sv = inputs(rng, rows, n_out, n_in, group)
    say("[i4 product]", rows, n_out, n_in, group)
    y = Result(ctx, rows, n_out, "f32")
    ctx.i4_matmul(ctx.upload(x), ctx.upload(packed(q, rng)), ctx.upload(s), rows, n_out, n_in, group, y.at,
                  x_scale=ctx.upload(sx))
    near(y.read(), *product(x, q, sv[0], group, sx, None, False), n_in, "f32")


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale_kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scales,bias,relu", [(True, True, False), (True, False, True), (False, True, True)])
@pytest.mark.parametrize("rows,n_out,n_in,group", [(1, 700, 1000, 128), (6, 33, 70, 32), (40, 65, 333, 64),
                                                   (270, 260, 1024, 256)])
def test_types(ctx, kind, scale_kind, scales, bias, relu, rows, n_out, n_in, group):
    rng = np.random.default_rng([rows, n_out, n_in])
    x, sx, q, s, sv = inputs(rng, rows, n_out, n_in, group, scale_kind)
    if not scales:
        sx = None
        x //= 16  # f16 results end at 65504
    b = rng.normal(0, 1, n_out).astype(np.float32) if bias else None
    say("[i4 types]", kind, scale_kind, scales, rows, n_out, n_in)
    y = Result(ctx, rows, n_out, kind)
    ctx.i4_matmul(ctx.upload(x), ctx.upload(packed(q)), ctx.upload(s), rows, n_out, n_in, group, y.at, TYPES[kind],
                  scale_type=TYPES[scale_kind], x_scale=up(ctx, sx), bias=up(ctx, b), relu=relu)
    near(y.read(), *product(x, q, sv[0], group, sx, b, relu), n_in, kind)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,n_out,n_in,group", [(1, 70, 100, 32), (5, 65, 1000, 128), (40, 130, 77, 64),
                                                   (140, 270, 515, 128), (260, 300, 1024, 64), (300, 256, 512, 128)])
@pytest.mark.parametrize("lead,pad", [(1, 3), (4, 12), (8, 5), (16, 16)])
def test_strides_and_offsets(ctx, kind, rows, n_out, n_in, group, lead, pad):
    """Rows of x and y at other strides and at odd addresses, rows of w apart;
    nothing beside y is written, nothing beside x is used."""
    rng = np.random.default_rng([rows, lead, pad])
    x, sx, q, s, sv = inputs(rng, rows, n_out, n_in, group)
    say("[i4 strides]", kind, rows, n_out, n_in, lead, pad)
    y = Result(ctx, rows, n_out, kind, ld=n_out + pad, lead=lead)
    w = packed(q, rng)
    ctx.i4_matmul(matrix(ctx, x, n_in + pad, lead), matrix(ctx, w, w.shape[1] + 48, 32), ctx.upload(s), rows, n_out,
                  n_in, group, y.at, TYPES[kind], x_scale=ctx.upload(sx), ld_x=n_in + pad, ld_w=w.shape[1] + 48,
                  ld_y=n_out + pad)
    near(y.read(), *product(x, q, sv[0], group, sx, None, False), n_in, kind)


# many rows: whole and ragged tiles, rows of whole 16-byte pieces and not
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("rows,n_out,n_in", [(700, 1200, 2048), (1500, 1030, 656), (2050, 2200, 1040),
                                             (1100, 1300, 1001), (129, 4100, 3001)])
def test_many_rows(ctx, rows, n_out, n_in, group):
    rng = np.random.default_rng([rows, n_out, n_in, group])
    x, sx, q, s, sv = inputs(rng, rows, n_out, n_in, group, "f16")
    b = rng.normal(0, 1, n_out).astype(np.float32)
    say("[i4 many rows]", rows, n_out, n_in, group)
    y = Result(ctx, rows, n_out, "bf16", ld=n_out + 3)
    ctx.i4_matmul(ctx.upload(x), ctx.upload(packed(q, rng)), ctx.upload(s), rows, n_out, n_in, group, y.at, z.BF16,
                  scale_type=z.F16, x_scale=ctx.upload(sx), bias=ctx.upload(b), relu=True, ld_y=n_out + 3)
    near(y.read(), *product(x, q, sv[0], group, sx, b, True), n_in, "bf16")


# the sizes of each kernel for whole chunks and groups of 128, with odd rows and other groups
# too, which may take another one (each form at its own sizes: test_gpu_i4_forms.py)
@pytest.mark.parametrize("group", [32, 64, 128, 384])
@pytest.mark.parametrize("odd", [0, 1])
@pytest.mark.parametrize("name,rows,n_out,n_in", listed(PLAIN))
def test_every_kernel(ctx, name, rows, n_out, n_in, odd, group):
    if rows * n_out > 4e6 and group not in ((64, 128) if odd else (32, 64, 128)):
        pytest.skip("the largest sizes with fewer groups")
    rng = np.random.default_rng([rows, n_out, n_in, group])
    x, sx, q, s, sv = inputs(rng, rows, n_out, n_in, group, "bf16")
    b = rng.normal(0, 1, n_out).astype(np.float32)
    say("[i4 kernel]", name, rows, n_out, n_in, odd, group)
    y = Result(ctx, rows, n_out, "f16", ld=n_out + 1 + odd)
    ctx.i4_matmul(matrix(ctx, x, n_in + odd, odd), ctx.upload(packed(q, rng)), ctx.upload(s), rows, n_out, n_in, group,
                  y.at, z.F16, scale_type=z.BF16, x_scale=ctx.upload(sx), bias=ctx.upload(b), ld_x=n_in + odd,
                  ld_y=n_out + 1 + odd)
    near(y.read(), *wide_product(x, q, sv[0], group, sx, b, False), n_in, "f16")


@pytest.mark.parametrize("group", [32, 64, 256])
@pytest.mark.parametrize("odd", [0, 1])
@pytest.mark.parametrize("name,rows,n_out,n_in,experts", listed(GROUPED_SIZES))
def test_every_grouped_kernel(ctx, name, rows, n_out, n_in, experts, odd, group):
    rng = np.random.default_rng([rows, n_out, n_in, group])
    x, sx, q, s, sv = inputs(rng, rows, n_out, n_in, group, "f16", experts)
    offsets, order = routes(rng, rows, 1, experts, 0.05)
    b = rng.normal(0, 1, (experts, n_out)).astype(np.float32)
    say("[i4 grouped kernel]", name, rows, n_out, n_in, experts, odd, group)
    y = Result(ctx, rows, n_out, "f32")
    ctx.i4_matmul_experts(matrix(ctx, x, n_in + odd, odd), ctx.upload(packed(q, rng)), ctx.upload(s),
                          ctx.upload(offsets), rows, experts, n_out, n_in, group, y.at, scale_type=z.F16,
                          x_scale=ctx.upload(sx), bias=ctx.upload(b), order=ctx.upload(order), tokens=rows,
                          ld_x=n_in + odd)
    want, size = np.zeros((rows, n_out)), np.zeros((rows, n_out))
    for e in range(experts):
        at = np.arange(offsets[e], offsets[e + 1])
        if len(at):
            want[at], size[at] = wide_product(x[order[at]], q[e * n_out:(e + 1) * n_out], sv[e], group, sx[order[at]],
                                              b[e], False)
    near(y.read(), want, size, n_in, "f32")


@pytest.mark.parametrize("rows,n_out,n_in,group", [(1, 9, 200000, 128), (3, 5, 70001, 1280), (1, 70000, 96, 32),
                                                   (70000, 3, 64, 64)])
def test_long_and_wide(ctx, rows, n_out, n_in, group):
    rng = np.random.default_rng([rows, n_out, n_in])
    x, sx, q, s, sv = inputs(rng, rows, n_out, n_in, group)
    say("[i4 long]", rows, n_out, n_in, group)
    y = Result(ctx, rows, n_out, "f32")
    ctx.i4_matmul(ctx.upload(x), ctx.upload(packed(q, rng)), ctx.upload(s), rows, n_out, n_in, group, y.at,
                  x_scale=ctx.upload(sx))
    near(y.read(), *product(x, q, sv[0], group, sx, None, False), n_in, "f32")


@pytest.mark.parametrize("rows,n_out,n_in,group", [(1, 64, 256, 128), (20, 40, 256, 64), (300, 300, 256, 32)])
def test_extremes_stay_in_their_row_and_channel(ctx, rows, n_out, n_in, group):
    """The largest sums are exact; a scale of infinity or NaN reaches its channel or
    its row and nothing else."""
    x = np.full((rows, n_in), -128, dtype=np.int8)
    q = np.full((n_out, n_in), -8, dtype=np.int8)
    s, sx = np.ones((n_in // group, n_out), dtype=np.float32), np.ones(rows, dtype=np.float32)
    s[1, 3], s[0, 5], sx[rows - 1] = np.inf, np.nan, np.nan
    y = Result(ctx, rows, n_out, "f32")
    ctx.i4_matmul(ctx.upload(x), ctx.upload(packed(q)), ctx.upload(s), rows, n_out, n_in, group, y.at,
                  x_scale=ctx.upload(sx), relu=True)
    want = np.full((rows, n_out), 1024.0 * n_in, dtype=np.float32)
    want[:, 3], want[:, 5], want[rows - 1] = np.inf, np.nan, np.nan
    assert np.array_equal(y.read(), want, equal_nan=True)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale_kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,group,lead,pad", [(1, 1, 32, 0, 0), (3, 31, 32, 1, 2), (5, 129, 64, 0, 0),
                                                      (70, 1000, 128, 3, 1), (33, 520, 256, 0, 8), (9, 384, 32, 0, 0)])
def test_quantize(ctx, kind, scale_kind, rows, cols, group, lead, pad):
    rng = np.random.default_rng([rows, cols, group])
    w = words(rng.normal(0, 1, (rows, cols)) * np.exp(rng.normal(0, 1, (rows, 1))), kind)
    wv = values(w, kind).astype(np.float32)
    wv[0, :group] = 0  # a group of zeros
    w = words(wv, kind)
    groups = -(-cols // group)
    ld = -(-cols // 128) * 64 + 16
    say("[i4 quantize]", kind, scale_kind, rows, cols, group)
    q, s = Result(ctx, rows, ld - 16, "i8", ld=ld), Result(ctx, groups, rows, scale_kind)
    ctx.i4_quantize(matrix(ctx, w, cols + pad, lead), TYPES[kind], rows, cols, group, q.at, s.at, TYPES[scale_kind],
                    ld_w=cols + pad, ld_q=ld)
    a = np.stack([np.abs(wv[:, g * group:(g + 1) * group]).max(axis=1) for g in range(groups)])
    want_s = words(a / np.float32(7), scale_kind)
    got_s, got_q = s.read(), q.read().view(np.uint8)
    assert np.array_equal(got_s.view(np.uint8), want_s.view(np.uint8))
    sv = values(want_s, scale_kind).astype(np.float32).T.repeat(group, axis=1)[:, :cols]
    want = np.clip(np.rint(np.divide(wv, sv, out=np.zeros_like(wv), where=sv > 0)), -8, 7)
    got = unpacked(got_q, cols)
    assert np.array_equal(got, want)
    assert np.array_equal(got_q, packed(got)), "padding is not zero"


def test_quantize_of_what_has_no_scale(ctx):
    w = np.ones((4, 256), dtype=np.float32)
    w[0, 5], w[1, 200], w[2, :128], w[3, 0] = np.inf, np.nan, 0.0, 1e-45
    w[3, 1:128] = 0
    q, s = Result(ctx, 4, 128, "i8"), Result(ctx, 2, 4, "f32")
    ctx.i4_quantize(ctx.upload(w), z.F32, 4, 256, 128, q.at, s.at)
    got, sc = unpacked(q.read().view(np.uint8), 256), s.read()
    seventh = np.float32(1) / np.float32(7)
    assert np.array_equal(sc, np.array([[np.nan, seventh, 0, 0], [seventh, np.nan, seventh, seventh]], np.float32),
                          equal_nan=True)
    want = np.full((4, 256), 7)
    want[0, :128] = want[1, 128:] = want[2, :128] = want[3, :128] = 0
    assert np.array_equal(got, want)


@pytest.mark.parametrize("rows,n_in,group", [(1, 256, 128), (40, 200, 32), (300, 300, 64)])
def test_quantize_beyond_the_scales_type(ctx, rows, n_in, group):
    """A scale that rounds to infinity has zeros, and what is made of it shows it."""
    rng = np.random.default_rng(group)
    w = rng.normal(0, 1, (5, n_in)).astype(np.float32)
    w[2, :group] *= 1e8
    groups = -(-n_in // group)
    q, s = Result(ctx, 5, -(-n_in // 128) * 64, "i8"), Result(ctx, groups, 5, "f16")
    ctx.i4_quantize(ctx.upload(w), z.F32, 5, n_in, group, q.at, s.at, z.F16)
    sc, got = s.read(), unpacked(q.read().view(np.uint8), n_in)
    assert sc[0, 2] == np.inf and np.isinf(sc).sum() == 1 and not got[2, :group].any()
    y = Result(ctx, rows, 5, "f32")
    ctx.i4_matmul(ctx.upload(np.ones((rows, n_in), np.int8)), q.at, s.at, rows, 5, n_in, group, y.at, scale_type=z.F16)
    assert np.isnan(y.read()[:, 2]).all() and np.isfinite(np.delete(y.read(), 2, axis=1)).all()


LINEAR = [(1, 100, 64, 32), (1, 1024, 8192, 128), (3, 70, 1001, 64), (16, 33, 500, 128), (17, 200, 1024, 128),
          (40, 129, 2100, 64), (300, 257, 640, 128), (8, 100, 20000, 128), (2, 20, 7, 32), (5, 40, 16, 64), (4, 50, 33, 128),
          (16, 300, 2200, 256), (1, 8200, 256, 128), (2, 8192, 130, 32), (13, 31, 1500, 64), (1, 70, 36000, 128)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n_out,n_in,group", LINEAR)
def test_linear(ctx, kind, rows, n_out, n_in, group):
    """The quantizer's integers, read back, through the product."""
    rng = np.random.default_rng([rows, n_out, n_in])
    x = words(rng.normal(0, 1, (rows, n_in)) * np.exp(rng.normal(0, 1, (rows, 1))), kind)
    _, _, q, s, sv = inputs(rng, rows, n_out, n_in, group, "f16")
    s, sv = words(sv / 64, "f16"), values(words(sv / 64, "f16"), "f16")
    b = rng.normal(0, 1, n_out).astype(np.float32)
    say("[i4 linear]", kind, rows, n_out, n_in)
    pad = 5
    xd = matrix(ctx, x, n_in + pad, 1)
    y = Result(ctx, rows, n_out, kind, ld=n_out + 1)
    ctx.i4_linear(xd, TYPES[kind], ctx.upload(packed(q, rng)), ctx.upload(s), rows, n_out, n_in, group, y.at,
                  TYPES[kind], ctx.alloc(ctx.i4_linear_work(rows, n_in)), scale_type=z.F16, bias=ctx.upload(b),
                  ld_x=n_in + pad, ld_y=n_out + 1)
    q8, s8 = Result(ctx, rows, n_in, "i8"), Result(ctx, 1, rows, "f32")
    ctx.i8_quantize(xd, TYPES[kind], rows, n_in, q8.at, s8.at, ld_x=n_in + pad)
    near(y.read(), *product(q8.read(), q, sv[0], group, s8.read()[0], b, False), n_in, kind)


@pytest.mark.parametrize("kind,rows,n_out,n_in", [
    ("bf16", 16, 60, 2048), ("bf16", 16, 60, 2049), ("f32", 1, 50, 16384), ("f32", 1, 50, 16385),
    ("f16", 1, 40, 32768), ("f16", 1, 40, 32769), ("f32", 8, 4096, 2048), ("f32", 8, 4112, 2048),
    ("bf16", 12, 4112, 2048), ("bf16", 13, 4112, 2048), ("f16", 4, 30, 8189), ("f32", 17, 30, 64)])
@pytest.mark.parametrize("group", [64, 128])
def test_linear_beside_its_limits(ctx, kind, rows, n_out, n_in, group):
    """Sizes on both sides of where the rows are quantized on the way."""
    rng = np.random.default_rng([rows, n_out, n_in, group])
    x = words(rng.normal(0, 1, (rows, n_in)), kind)
    _, _, q, s, _ = inputs(rng, rows, n_out, n_in, group, "f32")
    s = s / np.float32(64)
    sv = values(s, "f32")
    say("[i4 linear limits]", kind, rows, n_out, n_in, group)
    xd, y = ctx.upload(x), Result(ctx, rows, n_out, "f32")
    ctx.i4_linear(xd, TYPES[kind], ctx.upload(packed(q, rng)), ctx.upload(s), rows, n_out, n_in, group, y.at, z.F32,
                  ctx.alloc(ctx.i4_linear_work(rows, n_in)))
    q8, s8 = Result(ctx, rows, n_in, "i8"), Result(ctx, 1, rows, "f32")
    ctx.i8_quantize(xd, TYPES[kind], rows, n_in, q8.at, s8.at)
    near(y.read(), *wide_product(q8.read(), q, sv[0], group, s8.read()[0], None, False), n_in, "f32")


def test_linear_rows_without_a_scale(ctx):
    x = np.ones((4, 200), dtype=np.float32)
    x[1, 7], x[2] = np.inf, 0.0
    x[3, 199] = np.nan
    y = Result(ctx, 4, 20, "f32")
    ctx.i4_linear(ctx.upload(x), z.F32, ctx.upload(packed(np.ones((20, 200), np.int8))),
                  ctx.upload(np.ones((2, 20), np.float32)), 4, 20, 200, 128, y.at, z.F32,
                  ctx.alloc(ctx.i4_linear_work(4, 200)), bias=ctx.upload(np.full(20, 3, np.float32)))
    got = y.read()
    assert np.isnan(got[1]).all() and np.isnan(got[3]).all() and (got[2] == 3).all()
    assert np.abs(got[0] - 203).max() <= 203 * 4 * 2.0**-24


# tokens, slots, experts, n_out, n_in, group, part of the pairs dropped
GROUPED = [(1, 1, 1, 16, 64, 32, 0), (5, 2, 16, 70, 300, 128, 0), (33, 2, 8, 130, 260, 64, 0.2),
           (40, 4, 8, 64, 1000, 128, 0.1), (3, 8, 64, 33, 129, 32, 0), (200, 2, 4, 257, 512, 128, 0),
           (600, 2, 3, 300, 640, 64, 0.1), (100, 1, 100, 31, 100, 256, 0), (50, 2, 4, 40, 77, 32, 1.0),
           (700, 3, 5, 140, 1001, 128, 0.05)]


def routes(rng, tokens, slots, experts, dropped):
    e = rng.integers(0, experts, tokens * slots)
    e[rng.random(tokens * slots) < dropped] = -1
    key = np.where(e >= 0, e, experts)
    order = np.argsort(key, kind="stable")
    offsets = np.searchsorted(key[order], np.arange(experts + 1)).astype(np.int32)
    order[offsets[-1]:] = -1
    return offsets, order.astype(np.int32)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("ordered", [True, False])
@pytest.mark.parametrize("tokens,slots,experts,n_out,n_in,group,dropped", GROUPED)
def test_experts(ctx, kind, ordered, tokens, slots, experts, n_out, n_in, group, dropped):
    rng = np.random.default_rng([tokens, slots, experts, n_in])
    rows = tokens * slots
    offsets, order = routes(rng, tokens, slots, experts, dropped)
    n_x = tokens if ordered else rows
    x, sx, q, s, sv = inputs(rng, n_x, n_out, n_in, group, "bf16", experts)
    b = rng.normal(0, 1, (experts, n_out)).astype(np.float32)
    say("[i4 experts]", kind, ordered, tokens, slots, experts, n_out, n_in)
    y = Result(ctx, rows, n_out, kind, ld=n_out + 2)
    more = dict(order=ctx.upload(order), slots=slots, tokens=tokens) if ordered else {}
    ctx.i4_matmul_experts(matrix(ctx, x, n_in + 3, 1), ctx.upload(packed(q, rng)), ctx.upload(s), ctx.upload(offsets),
                          rows, experts, n_out, n_in, group, y.at, TYPES[kind], scale_type=z.BF16,
                          x_scale=ctx.upload(sx), bias=ctx.upload(b), relu=True, ld_x=n_in + 3, ld_y=n_out + 2, **more)
    want, size = np.zeros((rows, n_out)), np.zeros((rows, n_out))
    for e in range(experts):
        at = np.arange(offsets[e], offsets[e + 1])
        if len(at):
            t = order[at] // slots if ordered else at
            want[at], size[at] = product(x[t], q[e * n_out:(e + 1) * n_out], sv[e], group, sx[t], b[e], True)
    near(y.read(), want, size, n_in, kind)


@pytest.mark.parametrize("rows,n_out", [(6, 20), (200, 300)])
def test_experts_bad_orders_and_offsets(ctx, rows, n_out):
    """Indexes that name no token give zeros; offsets outside the rows are held inside."""
    rng = np.random.default_rng(rows)
    tokens, n_in = 4, 192
    x, sx, q, s, sv = inputs(rng, tokens, n_out, n_in, 64, experts=2)
    order = rng.integers(-3, 2 * tokens + 3, rows).astype(np.int32)
    order[0], order[1] = 2**31 - 1, -2**31
    offsets = np.array([0, rows // 2, rows + 1000], dtype=np.int32)
    y = Result(ctx, rows, n_out, "f32")
    ctx.i4_matmul_experts(ctx.upload(x), ctx.upload(packed(q)), ctx.upload(s), ctx.upload(offsets), rows, 2, n_out,
                          n_in, 64, y.at, x_scale=ctx.upload(sx), order=ctx.upload(order), slots=2, tokens=tokens)
    want, size = np.zeros((rows, n_out)), np.zeros((rows, n_out))
    for p in range(rows):
        t, e = order[p] // 2, int(p >= rows // 2)
        if 0 <= t < tokens:
            want[p], size[p] = (a[0] for a in product(x[t:t + 1], q[e * n_out:(e + 1) * n_out], sv[e], 64,
                                                      sx[t:t + 1], None, False))
    near(y.read(), want, size, n_in, "f32")


def test_empty(ctx):
    d = ctx.upload(np.zeros(4096, dtype=np.int8))
    ctx.i4_matmul(None, None, None, 0, 8, 64, 32, None)
    ctx.i4_matmul(d, d, d, 4, 0, 64, 32, None, ld_y=0)
    ctx.i4_quantize(None, z.F32, 0, 64, 32, None, None)
    ctx.i4_quantize(None, z.F32, 4, 0, 32, None, None)
    ctx.i4_linear(None, z.F32, None, None, 0, 8, 64, 32, None, z.F32, None)
    ctx.i4_matmul_experts(None, d, d, d, 0, 2, 8, 64, 32, None)
    b = np.arange(5, dtype=np.float32)
    y = Result(ctx, 3, 5, "f32")
    ctx.i4_matmul(None, None, None, 3, 5, 0, 32, y.at, bias=ctx.upload(b))
    assert np.array_equal(y.read(), np.tile(b, (3, 1)))
    y = Result(ctx, 3, 5, "f32")
    ctx.i4_matmul_experts(None, d, d, ctx.upload(np.array([0, 3], dtype=np.int32)), 3, 1, 5, 64, 32, y.at, tokens=0,
                          bias=ctx.upload(b))
    assert not y.read().any()


def test_refusals(ctx):
    d = ctx.alloc(1 << 16)
    mat = dict(x=d, w=d, w_scale=d, rows=2, n_out=4, n_in=256, group=128, y=d)
    lin = dict(x=d, x_type=z.F32, w=d, w_scale=d, rows=2, n_out=4, n_in=256, group=128, y=d, y_type=z.F32, work=d)
    exp = dict(x=d, w=d, w_scale=d, offsets=d, rows=2, experts=2, n_out=4, n_in=256, group=128, y=d)
    qua = dict(w=d, w_type=z.F32, rows=2, cols=256, group=128, q=d, scale=d)
    groups = [(dict(group=g), "group") for g in (0, -128, 16, 96, 127, 129, 192)]
    shared = groups + [(dict(y=None), "null"), (dict(w=None), "null"), (dict(w_scale=None), "null"),
                       (dict(y_type=z.I32), "f32, f16 or bf16"), (dict(scale_type=z.I32), "f32, f16 or bf16"),
                       (dict(n_in=(1 << 24) + 1), "2\\^24"), (dict(n_out=(1 << 26) + 1), "2\\^26"),
                       (dict(rows=1 << 31), "2\\^31"), (dict(ld_x=255), "stride"), (dict(ld_w=112), "stride"),
                       (dict(ld_y=3), "stride"), (dict(w=At(d, 8)), "16 bytes"), (dict(ld_w=136), "16 bytes"),
                       (dict(y=At(d, 2)), "aligned"), (dict(w_scale=At(d, 2)), "aligned"),
                       (dict(bias=At(d, 1)), "aligned")]
    for f, a, more in [
            (ctx.i4_matmul, mat, [(dict(x=None), "null"), (dict(x_scale=At(d, 2)), "aligned")]),
            (ctx.i4_linear, lin, [(dict(x=None), "null"), (dict(x_type=z.I32), "f32, f16 or bf16"),
                                  (dict(work=None), "workspace"), (dict(work=At(d, 8)), "workspace"),
                                  (dict(work=ctx.alloc(ctx.i4_linear_work(2, 256) - 1)), "workspace")]),
            (ctx.i4_matmul_experts, exp, [(dict(x=None), "null"), (dict(offsets=None), "null"),
                                          (dict(experts=0), "1024"),
                                          (dict(experts=1025), "1024"), (dict(slots=0), "slots"),
                                          (dict(offsets=At(d, 1)), "aligned"), (dict(order=At(d, 2)), "aligned"),
                                          (dict(rows=(1 << 22) + 1), "too many"),
                                          (dict(order=d, slots=2), "tokens")])]:
        f(**a)
        for bad, why in shared + more:
            with pytest.raises(z.ZkError, match=why):
                f(**dict(a, **bad))
    ctx.i4_quantize(**qua)
    for bad, why in groups + [(dict(w=None), "null"), (dict(q=None), "null"), (dict(scale=None), "null"),
                              (dict(w_type=z.I32), "f32, f16 or bf16"), (dict(scale_type=z.I32), "f32, f16 or bf16"),
                              (dict(rows=1 << 31), "2\\^31"), (dict(cols=(1 << 24) + 1), "2\\^24"),
                              (dict(ld_w=255), "stride"), (dict(ld_q=112), "stride"), (dict(ld_q=136), "16 bytes"),
                              (dict(q=At(d, 8)), "16 bytes"), (dict(w=At(d, 2)), "aligned"),
                              (dict(scale=At(d, 2)), "aligned")]:
        with pytest.raises(z.ZkError, match=why):
            ctx.i4_quantize(**dict(qua, **bad))
    ctx.sync()


def test_sizes_without_a_device():
    assert [z.Context.i4_row_bytes(k) for k in (0, 1, 64, 128, 129, 1 << 24, (1 << 24) + 1)] == \
        [0, 64, 64, 64, 128, 1 << 23, 0]
    assert z.Context.i4_linear_work(1 << 31, 4) == 0 and z.Context.i4_linear_work(4, (1 << 24) + 1) == 0
    assert z.Context.i4_linear_work(3, 100) >= 3 * 104
