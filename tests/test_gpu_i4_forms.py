"""GPU tests of every form of the 4-bit product's kernels (i4_forms) against the 64-bit
form, within the bounds of i4_helpers.near."""
import numpy as np
import pytest

import zkml_amd as z
from i4_forms import FORMS
from i4_helpers import inputs, near, packed, wide_product
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
