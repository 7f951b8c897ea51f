"""GPU tests of the 4-bit products at the largest sizes that they take: 2^26 channels, rows
of 2^24 weights, groups as long, 2^22 rows of experts.  Few weights and scales differ from
their neighbours, so that results are exact and known."""
import ctypes

import numpy as np
import pytest

import zkml_amd as z
from i8_helpers import At

pytestmark = pytest.mark.gpu

hip, vp = ctypes.CDLL("libamdhip64.so"), ctypes.c_void_p


@pytest.fixture(scope="module")
def ctx():
    return z.Context(0)


def filled(ctx, n, byte):
    d = ctx.alloc(n)
    assert hip.hipMemset(vp(d.ptr), byte, ctypes.c_size_t(n)) == 0 and hip.hipDeviceSynchronize() == 0
    return d


def test_the_widest_layer(ctx):
    """More rows than one launch has tiles for; channels told apart by their scales."""
    n, k, rows = 1 << 26, 32, 17
    rng = np.random.default_rng(1)
    s = rng.integers(1, 64, n).astype(np.float16)
    print("[widest layer]", flush=True)
    w, y = filled(ctx, n * 64, 0x11), ctx.alloc(rows * n * 2)  # weights of 1
    x = np.tile(np.arange(1, rows + 1, dtype=np.int8)[:, None], (1, k))
    ctx.i4_matmul(ctx.upload(x), w, ctx.upload(s), rows, n, k, k, y, z.F16, scale_type=z.F16)
    for t in (0, 7, 15, 16):
        # up to 32 * 17 * 63 < 2^16, steps of 32 (11 bits hold them)
        got = ctx.d2h(At(y, t * n * 2), (n,), np.float16)
        assert np.array_equal(got, (s.astype(np.float32) * (32 * (t + 1))).astype(np.float16))


@pytest.mark.parametrize("group", [32, 128, 1 << 24, 0x7fffff80])
@pytest.mark.parametrize("rows,n_out", [(1, 3), (40, 20)])
@pytest.mark.parametrize("short", [0, 5])
def test_the_longest_rows(ctx, rows, n_out, group, short):
    n_in = (1 << 24) - short
    rng = np.random.default_rng([rows, group])
    ends = [0, 1, 127, 128, (1 << 23) + 77, n_in - 129, n_in - 2, n_in - 1]
    at = np.unique(np.concatenate([ends, rng.integers(0, n_in, 40)]))
    values = rng.integers(-8, 8, (n_out, len(at)))
    row_bytes = (n_in + 127) // 128 * 64
    w, x = np.zeros((n_out, row_bytes), np.uint8), np.ones((rows, n_in), np.int8)
    run, i = at // 128, at % 128
    for j in range(len(at)):
        w[:, run[j] * 64 + i[j] % 64] |= ((values[:, j] & 15) << (4 if i[j] >= 64 else 0)).astype(np.uint8)
    x[:, at] = rng.integers(-127, 128, (rows, len(at)))
    x[:, 0] = 127
    groups = -(-n_in // group)
    s = np.ones((groups, n_out), np.float32)
    s[-1] = 2
    want = (x[:, at].astype(np.int64) @ (values * np.where(at // group == groups - 1, 2, 1)).T).astype(np.float32)
    print("[longest rows]", rows, n_out, group, short, flush=True)
    wd, sd, y = ctx.upload(w), ctx.upload(s), ctx.alloc(rows * n_out * 4)
    ctx.i4_matmul(ctx.upload(x), wd, sd, rows, n_out, n_in, group, y)
    assert np.array_equal(ctx.d2h(y, (rows, n_out), np.float32), want)
    if rows == 1:  # a row whose largest value is 127 is its own 8-bit row
        ctx.i4_linear(ctx.upload(x.astype(np.float32)), z.F32, wd, sd, rows, n_out, n_in, group, y, z.F32,
                      ctx.alloc(ctx.i4_linear_work(rows, n_in)))
        assert np.array_equal(ctx.d2h(y, (rows, n_out), np.float32), want)


def test_the_most_rows_of_experts(ctx):
    rows, experts, n, k = 1 << 22, 1024, 5, 32
    rng = np.random.default_rng(3)
    cuts = np.sort(rng.integers(0, rows, experts - 1))
    offsets = np.concatenate([[0], cuts, [rows - 100]]).clip(0, rows - 100).astype(np.int32)
    s = rng.integers(1, 1000, (experts, 1, n)).astype(np.float32)
    order = rng.permutation(rows).astype(np.int32)
    x = rng.integers(-9, 10, (rows // 4, k)).astype(np.int8)
    print("[most rows of experts]", flush=True)
    y = ctx.alloc(rows * n * 4)
    ctx.i4_matmul_experts(ctx.upload(x), filled(ctx, experts * n * 64, 0x33), ctx.upload(s), ctx.upload(offsets), rows,
                          experts, n, k, k, y, order=ctx.upload(order), slots=4, tokens=rows // 4)
    sums = 3 * x.astype(np.int64).sum(1)
    expert = np.searchsorted(offsets, np.arange(rows), side="right") - 1
    want = (sums[order // 4, None] * s[np.minimum(expert, experts - 1), 0]).astype(np.float32)
    want[rows - 100:] = 0
    assert np.array_equal(ctx.d2h(y, (rows, n), np.float32), want)


@pytest.mark.parametrize("rows,n_out,group,experts", [(2000, 2000, 1 << 23, 0), (2500, 2000, 64, 0), (511, 4000, 128, 1),
                                                      (511, 4000, 64, 1), (520, 4000, 128, 1)])
def test_long_rows_in_stages(ctx, rows, n_out, group, experts):
    """Rows as long as lie within 32 bits of one another in a block, or, grouped, in x; and a
    few more."""
    n_in = (1 << 23) - 16
    assert z.lib().zk_debug_i4_kernel(rows, n_out, n_in, n_in, 0, group, experts).startswith(b"stages")
    rng = np.random.default_rng(rows)
    row_bytes = (n_in + 127) // 128 * 64
    s, sx = rng.integers(1, 8, n_out).astype(np.float32), rng.integers(1, 5, rows).astype(np.float32)
    print("[long rows in stages]", rows, n_out, group, experts, flush=True)
    x, w, y = filled(ctx, rows * n_in, 1), filled(ctx, n_out * row_bytes, 0x11), ctx.alloc(rows * n_out * 4)
    sd, sxd = ctx.upload(np.tile(s, (-(-n_in // group), 1))), ctx.upload(sx)
    if experts:
        order = rng.permutation(rows).astype(np.int32)
        ctx.i4_matmul_experts(x, w, sd, ctx.upload(np.array([0, rows], np.int32)), rows, 1, n_out, n_in, group, y,
                              x_scale=sxd, order=ctx.upload(order), tokens=rows)
        sx = sx[order]
    else:
        ctx.i4_matmul(x, w, sd, rows, n_out, n_in, group, y, x_scale=sxd)
    # multiples of 16 s, of which 32-bit floats hold all sums on the way
    assert np.array_equal(ctx.d2h(y, (rows, n_out), np.float32), np.float32(n_in) * s * sx[:, None])
