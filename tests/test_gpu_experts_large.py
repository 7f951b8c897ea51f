"""GPU tests of the routed experts (cuda-zkml_amd/csrc/experts.hip) at sizes where
other kernels, or more blocks, take part than at small ones: sorts up to the most
pairs there may be, rows that pass the caches."""
import numpy as np
import pytest

import zkml_amd as z
from i8_helpers import TYPES, Result, matrix, values, words
from test_gpu_experts import expected, rounded, route, say, sort

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return z.Context(0)


@pytest.mark.parametrize("pairs,experts", [(1 << 20, 1024), ((1 << 22) - 1, 8), (1 << 22, 1), (1 << 22, 1024)])
def test_sort_of_many_pairs(ctx, pairs, experts):
    rng = np.random.default_rng([pairs, experts])
    e = rng.integers(0, experts, pairs)
    e[rng.random(pairs) < 0.1] = -1
    say("[experts sort]", pairs, experts)
    for got, want in zip(sort(ctx, e, experts), expected(e, experts)):
        assert np.array_equal(got, want)


@pytest.mark.parametrize("pairs", [640, 8192, 30000])
@pytest.mark.parametrize("each", [1, 2, 31, 63, 64, 65, 200])
def test_sort_of_neighbours_with_the_same_expert(ctx, pairs, each):
    """The running counts of a wave: 64 pairs at a time share a count, take one each,
    or anything between, and the next 64 go on from there."""
    e = np.arange(pairs) // each % 7
    e[::11] = 3
    say("[experts sort]", pairs, each)
    for got, want in zip(sort(ctx, e, 7), expected(e, 7)):
        assert np.array_equal(got, want)


# over 32 MB of rows, at widths that end inside a piece of 16 bytes
@pytest.mark.parametrize("kind,cols", [("f32", 1501), ("f16", 2801), ("bf16", 2804)])
@pytest.mark.parametrize("lead,pad", [(0, 0), (1, 3)])
def test_rows_that_pass_the_caches(ctx, kind, cols, lead, pad):
    tokens, slots, experts = 3000, 4, 16
    rows, ld = tokens * slots, cols + pad
    rng = np.random.default_rng([cols, lead])
    _, order, place = route(rng, tokens, slots, experts, 0.1)
    x, g = (words(rng.standard_normal((tokens, cols), dtype=np.float32), kind) for _ in range(2))
    y = words(rng.standard_normal((rows, cols), dtype=np.float32), kind)
    w = rng.random((tokens, slots)).astype(np.float32)
    od, pd, wd = ctx.upload(order.astype(np.int32)), ctx.upload(place.astype(np.int32)), ctx.upload(w)
    pair, pick = np.maximum(order, 0), np.maximum(place, 0).reshape(tokens, slots)
    held, named = (order >= 0)[:, None], (place >= 0).reshape(tokens, slots)
    say("[experts large gather]", kind, cols, lead)
    out = Result(ctx, rows, cols, kind, ld=ld, lead=lead)
    ctx.experts_gather(matrix(ctx, x, ld, lead), TYPES[kind], cols, od, rows, tokens, slots, out.at, ld_x=ld, ld_out=ld)
    assert np.array_equal(out.read(), np.where(held, x[pair // slots], x.dtype.type(0)))
    say("[experts large combine]", kind, cols, lead)
    yd, yv = matrix(ctx, y, ld, lead, fill=0xFF), values(y, kind)
    for weight in (w, None):
        out = Result(ctx, tokens, cols, kind, ld=ld, lead=lead)
        ctx.experts_combine(yd, TYPES[kind], cols, pd, rows, tokens, slots, out.at,
                            weight=None if weight is None else wd, ld_y=ld, ld_out=ld)
        want, size = np.zeros((tokens, cols)), np.zeros((tokens, cols))
        for j in range(slots):
            f = named[:, j] * (1.0 if weight is None else weight[:, j].astype(np.float64))
            term = f[:, None] * yv[pick[:, j]]
            want, size = want + term, size + np.abs(term)
        rounded(out.read(), want, size, slots, kind)
    say("[experts large combine grad]", kind, cols, lead)
    gy, gw = Result(ctx, rows, cols, kind, ld=ld, lead=lead), Result(ctx, tokens, slots, "f32")
    ctx.experts_combine_grad(matrix(ctx, g, ld, lead, fill=0xFF), yd, TYPES[kind], cols, od, pd, wd, rows, tokens, slots,
                             gy.at, gw.at, ld_grad=ld, ld_y=ld, ld_grad_y=ld)
    gv = values(g, kind)
    dy = np.where(held, w.astype(np.float64).reshape(-1)[pair][:, None] * gv[pair // slots], 0.0)
    rounded(gy.read(), dy, np.abs(dy), 0, kind)
    terms = [yv[pick[:, j]] * gv * named[:, j:j + 1] for j in range(slots)]
    rounded(gw.read(), np.stack([t.sum(1) for t in terms], 1), np.stack([np.abs(t).sum(1) for t in terms], 1), cols, "f32")
