"""GPU tests of every form of the 4-bit product's kernels (i4_forms) against the 64-bit
form, within the bounds of i4_helpers.near: ordinary values, and both ends of a
32-bit float's range."""
import numpy as np
import pytest

import zkml_amd as z
from i4_forms import FORMS
from i4_helpers import inputs, near, packed, product, wide_product
from i8_helpers import Result, matrix, values
from test_gpu_i4 import routes

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return z.Context(0)


def say(*a):
    print(*a, flush=True)


def run(ctx, form, x, sx, q, s, b, rng):
    """(got, want, size) of a form's product; s in f32."""
    name, odd, group, rows, n_out, n_in, experts = form
    y = Result(ctx, rows, n_out, "f32", ld=n_out + 1)
    xd, wd, sd = matrix(ctx, x, n_in + odd, odd), ctx.upload(packed(q, rng)), ctx.upload(s)
    more = dict(x_scale=None if sx is None else ctx.upload(sx), bias=None if b is None else ctx.upload(b),
                ld_x=n_in + odd, ld_y=n_out + 1)
    sv = values(s, "f32")
    if not experts:
        ctx.i4_matmul(xd, wd, sd, rows, n_out, n_in, group, y.at, **more)
        return y.read(), *wide_product(x, q, sv[0], group, sx, None if b is None else b[0], False)
    offsets, order = routes(rng, rows, 1, experts, 0.05)
    ctx.i4_matmul_experts(xd, wd, sd, ctx.upload(offsets), rows, experts, n_out, n_in, group, y.at,
                          order=ctx.upload(order), tokens=rows, **more)
    want, size = np.zeros((rows, n_out)), np.zeros((rows, n_out))
    for e in range(experts):
        at = np.arange(offsets[e], offsets[e + 1])
        if len(at):
            want[at], size[at] = wide_product(x[order[at]], q[e * n_out:(e + 1) * n_out], sv[e], group,
                                              None if sx is None else sx[order[at]], None if b is None else b[e], False)
    return y.read(), want, size


@pytest.mark.parametrize("form", FORMS, ids=lambda f: "-".join(map(str, f)))
def test_every_form(ctx, form):
    _, _, group, rows, n_out, n_in, experts = form
    rng = np.random.default_rng([rows, n_out, n_in, group])
    x, sx, q, s, _ = inputs(rng, rows, n_out, n_in, group, experts=max(1, experts))
    b = rng.normal(0, 1, (max(1, experts), n_out)).astype(np.float32)
    say("[i4 form]", *form)
    near(*run(ctx, form, x, sx, q, s, b, rng), n_in, "f32")


def positive(form):
    """Inputs of a form whose terms are all positive and within a factor of 2, 2 and 4 of the
    largest; what a result can be at the most."""
    _, _, group, rows, n_out, n_in, experts = form
    rng = np.random.default_rng([rows, n_out, n_in, group, 1])
    x = rng.integers(64, 128, (rows, n_in)).astype(np.int8)
    q = rng.integers(4, 8, (max(1, experts) * n_out, n_in)).astype(np.int8)
    s = rng.uniform(1, 2, (max(1, experts), -(-n_in // group), n_out)).astype(np.float32)
    return rng, x, q, s, 127.0 * 7 * 2 * n_in


@pytest.mark.parametrize("form", FORMS, ids=lambda f: "-".join(map(str, f)))
def test_results_up_to_the_end_of_the_range(ctx, form):
    """Sums of scaled groups that a 32-bit float holds are not lost on the way."""
    rng, x, q, s, most = positive(form)
    s = s * np.float32(2.0 ** (128 - np.ceil(np.log2(most))))
    say("[i4 large]", *form)
    got, want, size = run(ctx, form, x, None, q, s, None, rng)
    assert 2.0**124 < want.max() < 2.0**128
    near(got, want, size, form[5], "f32")


@pytest.mark.parametrize("form", FORMS, ids=lambda f: "-".join(map(str, f)))
def test_scales_at_the_low_end_of_the_range(ctx, form):
    """Scales down to 2^-122 count in full."""
    rng, x, q, s, _ = positive(form)
    s = s * np.float32(2.0 ** (-122 - np.floor(np.log2(s.min()))))
    assert 2.0**-122 <= s.min() < 2.0**-121
    say("[i4 small]", *form)
    near(*run(ctx, form, x, np.full(form[3], 2.0**100, np.float32), q, s, None, rng), form[5], "f32")


def test_scales_below_the_normal_numbers(ctx):
    """They count to a multiple of 2^-145."""
    s = np.array([[2.0**-145 * k for k in range(40)]], np.float32)
    for rows in (1, 300):
        y = Result(ctx, rows, 40, "f32")
        ctx.i4_matmul(ctx.upload(np.full((rows, 64), 3, np.int8)), ctx.upload(packed(np.full((40, 64), 5, np.int8))),
                      ctx.upload(s), rows, 40, 64, 64, y.at, x_scale=ctx.upload(np.full(rows, 2.0**127, np.float32)))
        assert np.array_equal(y.read(), np.tile(np.arange(40) * np.float32(960 * 2.0**-18), (rows, 1)))


@pytest.mark.parametrize("rows,n_out,n_in,group", [(1, 64, 256, 32), (4, 50, 333, 64), (9, 100, 640, 128)])
def test_linear_up_to_the_end_of_the_range(ctx, rows, n_out, n_in, group):
    """The few rows that are quantized on the way."""
    rng, x, q, s, most = positive((None, 0, group, rows, n_out, n_in, 0))
    x[:, 0] = 127  # a row's scale is 1, its values are the quantized ones
    s = s * np.float32(2.0 ** (128 - np.ceil(np.log2(most))))
    y = Result(ctx, rows, n_out, "f32")
    ctx.i4_linear(ctx.upload(x.astype(np.float32)), z.F32, ctx.upload(packed(q, rng)), ctx.upload(s), rows, n_out, n_in,
                  group, y.at, z.F32, ctx.alloc(ctx.i4_linear_work(rows, n_in)))
    want, size = product(x, q, values(s, "f32")[0], group, None, None, False)
    assert 2.0**124 < want.max() < 2.0**128
    near(y.read(), want, size, n_in, "f32")


# the last group ends inside the last step
@pytest.mark.parametrize("odd", [0, 1])
@pytest.mark.parametrize("rows,n_out,n_in,group", [(1, 64, 160, 32), (4, 40, 200, 64), (20, 40, 208, 32),
                                                   (60, 100, 336, 64), (300, 300, 160, 32), (700, 260, 304, 64)])
def test_infinite_scale_of_a_last_group(ctx, rows, n_out, n_in, group, odd):
    """What lies behind a row's end has no part in an infinite scale of its last group."""
    x, q = np.full((rows, n_in), 5, dtype=np.int8), np.full((n_out, n_in), -3, dtype=np.int8)
    groups = -(-n_in // group)
    s = np.ones((groups, n_out), dtype=np.float32)
    s[-1, 3], s[-1, 7], s[-1, 11] = np.inf, -np.inf, np.nan
    want = np.full((rows, n_out), -15.0 * n_in, dtype=np.float32)
    want[:, 3], want[:, 7], want[:, 11] = -np.inf, np.inf, np.nan
    w, sd = ctx.upload(packed(q)), ctx.upload(s)
    say("[i4 last group]", rows, n_out, n_in, group, odd)
    y = Result(ctx, rows, n_out, "f32")
    ctx.i4_matmul(matrix(ctx, x, n_in + odd, odd), w, sd, rows, n_out, n_in, group, y.at, ld_x=n_in + odd)
    assert np.array_equal(y.read(), want, equal_nan=True)
    # rows of 127: a scale of 1
    y = Result(ctx, rows, n_out, "f32")
    ctx.i4_linear(ctx.upload(np.full((rows, n_in), 127, dtype=np.float32)), z.F32, w, sd, rows, n_out, n_in, group, y.at,
                  z.F32, ctx.alloc(ctx.i4_linear_work(rows, n_in)))
    want[np.isfinite(want)] = -381.0 * n_in
    assert np.array_equal(y.read(), want, equal_nan=True)
    y = Result(ctx, rows, n_out, "f32")
    ctx.i4_matmul_experts(matrix(ctx, x, n_in + odd, odd), w, sd, ctx.upload(np.array([0, rows], np.int32)), rows, 1,
                          n_out, n_in, group, y.at, ld_x=n_in + odd)
    want[np.isfinite(want)] = -15.0 * n_in
    assert np.array_equal(y.read(), want, equal_nan=True)
