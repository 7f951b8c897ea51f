"""GPU tests of the routed experts (cuda-zkml_amd/csrc/experts.hip): the stable
sort against numpy's, rows gathered bit for bit, sums and gradients against
their formulas in 64 bits and against differences.

A weighted sum of s terms in 32 bits is within (s + 1) 2^-24 of the sum of the
terms' magnitudes, then rounded once to the rows' type; a dot product of c
terms is within (c + 1) 2^-24 of its terms' magnitudes.
"""
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


def expected(e, experts):
    """(offsets, order, place) by numpy's stable sort."""
    key = np.where((e >= 0) & (e < experts), e, experts)
    order = np.argsort(key, kind="stable")
    offsets = np.searchsorted(key[order], np.arange(experts + 1)).astype(np.int32)
    place = np.empty(len(e), dtype=np.int64)
    place[order] = np.arange(len(e))
    place[key == experts] = -1
    order[offsets[-1]:] = -1
    return offsets, order, place


def sort(ctx, e, experts):
    n = len(e)
    off, order, place = (Result(ctx, 1, m, "i32") for m in (experts + 1, n, n))
    need = ctx.experts_sort_work(n, experts)
    work = ctx.alloc(need) if need else None
    ctx.experts_sort(ctx.upload(e.astype(np.int32)), n, experts, off.at, order.at, place.at, work)
    return off.read()[0], order.read()[0], place.read()[0]


@pytest.mark.parametrize("pairs", [0, 1, 2, 63, 64, 65, 1000, 1024, 1025, 8192, 8193, 16384, 16385, 40001, 300000])
@pytest.mark.parametrize("experts", [1, 2, 8, 63, 64, 1000, 1024])
def test_sort(ctx, pairs, experts):
    rng = np.random.default_rng([pairs, experts])
    e = rng.integers(0, experts, pairs)
    e[rng.random(pairs) < 0.1] = -1
    e[rng.random(pairs) < 0.05] = experts
    say("[experts sort]", pairs, experts)
    for got, want in zip(sort(ctx, e, experts), expected(e, experts)):
        assert np.array_equal(got, want)


@pytest.mark.parametrize("pairs", [5, 1000, 20000])
@pytest.mark.parametrize("route", ["one", "last", "none", "runs", "far"])
def test_sort_routes(ctx, pairs, route):
    """Everything to one expert, to the last, nowhere, long runs, indexes far
    outside the range."""
    experts = 16
    e = {"one": np.full(pairs, 3), "last": np.full(pairs, experts - 1), "none": np.full(pairs, -1),
         "runs": np.arange(pairs) * experts // pairs, "far": np.where(np.arange(pairs) % 3, 2**31 - 1, -2**31)}[route]
    for got, want in zip(sort(ctx, e, experts), expected(e, experts)):
        assert np.array_equal(got, want)


def test_sort_refusals(ctx):
    d = ctx.alloc(1 << 20)
    for args, why in [((d, 4, 0, d, d, d), "1024"), ((d, 4, 1025, d, d, d), "1024"),
                      ((d, (1 << 22) + 1, 4, d, d, d), "2\\^22"), ((None, 4, 4, d, d, d), "null"),
                      ((d, 4, 4, None, d, d), "null"), ((d, 4, 4, d, None, d), "null"),
                      ((d, 4, 4, d, d, None), "null"), ((At(d, 1), 4, 4, d, d, d), "aligned"),
                      ((d, 20000, 4, d, d, d), "workspace")]:
        with pytest.raises(z.ZkError, match=why):
            ctx.experts_sort(*args)
    assert ctx.experts_sort_work(20000, 0) == 0 and ctx.experts_sort_work((1 << 22) + 1, 4) == 0
    with pytest.raises(z.ZkError, match="workspace"):
        ctx.experts_sort(d, 20000, 4, d, d, d, ctx.alloc(ctx.experts_sort_work(20000, 4) - 1))


# tokens, slots, experts, cols, part of the pairs dropped, leading elements, stride beyond the row
ROWS = [(1, 1, 1, 1, 0, 0, 0), (3, 2, 4, 7, 0, 1, 2), (5, 1, 8, 8, 0.3, 0, 0), (33, 2, 8, 1000, 0, 0, 0),
        (40, 3, 5, 129, 0.2, 3, 5), (17, 8, 16, 260, 0, 0, 4), (7, 11, 16, 75, 0.1, 2, 1),
        (200, 4, 32, 2048, 0.1, 0, 0), (2, 2, 2, 5000, 0.5, 8, 8), (64, 2, 3, 3, 0, 0, 0)]


def route(rng, tokens, slots, experts, dropped):
    e = rng.integers(0, experts, tokens * slots)
    e[rng.random(tokens * slots) < dropped] = -1
    return expected(e, experts)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,slots,experts,cols,dropped,lead,pad", ROWS)
def test_gather(ctx, kind, tokens, slots, experts, cols, dropped, lead, pad):
    rng = np.random.default_rng([tokens, slots, cols])
    _, order, _ = route(rng, tokens, slots, experts, dropped)
    x = words(rng.normal(0, 1, (tokens, cols)), kind)
    rows = tokens * slots
    say("[experts gather]", kind, tokens, slots, cols)
    out = Result(ctx, rows, cols, kind, ld=cols + pad, lead=lead)
    ctx.experts_gather(matrix(ctx, x, cols + pad, lead), TYPES[kind], cols, ctx.upload(order.astype(np.int32)), rows,
                       tokens, slots, out.at, ld_x=cols + pad, ld_out=cols + pad)
    want = np.where((order >= 0)[:, None], x[np.maximum(order, 0) // slots], 0)
    assert np.array_equal(out.read().view(np.uint8), want.astype(x.dtype).view(np.uint8))


def rounded(got, want, size, terms, kind):
    lim = (terms + 1) * 2.0**-24 * size
    lim = lim + (np.abs(want) + lim) * ROUND[kind] + TINY[kind]
    bad = ~(np.abs(values(got, kind) - want) <= lim)
    assert not bad.any(), f"{int(bad.sum())} of {bad.size} off, first at {np.argwhere(bad)[0]}"


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("tokens,slots,experts,cols,dropped,lead,pad", ROWS)
def test_combine(ctx, kind, weighted, tokens, slots, experts, cols, dropped, lead, pad):
    rng = np.random.default_rng([tokens, slots, cols])
    _, _, place = route(rng, tokens, slots, experts, dropped)
    rows = tokens * slots
    y = words(rng.normal(0, 1, (rows, cols)), kind)
    w = rng.random((tokens, slots)).astype(np.float32)
    say("[experts combine]", kind, tokens, slots, cols)
    out = Result(ctx, tokens, cols, kind, ld=cols + pad, lead=lead)
    ctx.experts_combine(matrix(ctx, y, cols + pad, lead, fill=0xFF), TYPES[kind], cols,
                        ctx.upload(place.astype(np.int32)), rows, tokens, slots, out.at,
                        weight=ctx.upload(w) if weighted else None, ld_y=cols + pad, ld_out=cols + pad)
    p = place.reshape(tokens, slots)
    terms = np.where((p >= 0)[..., None], values(y, kind)[np.maximum(p, 0)], 0.0)
    if weighted:
        terms = terms * w.astype(np.float64)[..., None]
    rounded(out.read(), terms.sum(1), np.abs(terms).sum(1), slots, kind)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,slots,experts,cols,dropped,lead,pad", ROWS)
def test_combine_grad(ctx, kind, tokens, slots, experts, cols, dropped, lead, pad):
    rng = np.random.default_rng([tokens, slots, cols])
    _, order, place = route(rng, tokens, slots, experts, dropped)
    rows = tokens * slots
    y, g = words(rng.normal(0, 1, (rows, cols)), kind), words(rng.normal(0, 1, (tokens, cols)), kind)
    w = rng.random((tokens, slots)).astype(np.float32)
    say("[experts combine grad]", kind, tokens, slots, cols)
    gy, gw = Result(ctx, rows, cols, kind, ld=cols + pad, lead=lead), Result(ctx, tokens, slots, "f32")
    gd, yd = matrix(ctx, g, cols + pad, lead, fill=0xFF), matrix(ctx, y, cols + pad, lead, fill=0xFF)
    od, pd, wd = ctx.upload(order.astype(np.int32)), ctx.upload(place.astype(np.int32)), ctx.upload(w)
    lds = dict(ld_grad=cols + pad, ld_y=cols + pad, ld_grad_y=cols + pad)
    ctx.experts_combine_grad(gd, yd, TYPES[kind], cols, od, pd, wd, rows, tokens, slots, gy.at, gw.at, **lds)
    gv, yv = values(g, kind), values(y, kind)
    pair = np.maximum(order, 0)
    want = np.where((order >= 0)[:, None], w.astype(np.float64).reshape(-1)[pair][:, None] * gv[pair // slots], 0.0)
    got = gy.read()
    rounded(got, want, np.abs(want), 0, kind)
    p = place.reshape(tokens, slots)
    terms = np.where((p >= 0)[..., None], yv[np.maximum(p, 0)], 0.0) * gv[:, None, :]
    rounded(gw.read(), terms.sum(2), np.abs(terms).sum(2), cols, "f32")
    # without the weights' gradient, and without weights
    gy2 = Result(ctx, rows, cols, kind, ld=cols + pad, lead=lead)
    ctx.experts_combine_grad(gd, None, TYPES[kind], cols, od, pd, wd, rows, tokens, slots, gy2.at, **lds)
    assert np.array_equal(gy2.read().view(np.uint8), got.view(np.uint8))
    gy3 = Result(ctx, rows, cols, kind, ld=cols + pad, lead=lead)
    ctx.experts_combine_grad(gd, None, TYPES[kind], cols, od, pd, None, rows, tokens, slots, gy3.at, **lds)
    want = np.where((order >= 0)[:, None], g[pair // slots], 0).astype(g.dtype)
    assert np.array_equal(gy3.read().view(np.uint8), want.view(np.uint8))


def test_gradients_against_differences(ctx):
    """combine is linear in y and in the weights, and gather in x: the change of
    <g, out> for a step d is <gradient, d>, up to the roundings of both sides."""
    rng = np.random.default_rng(9)
    tokens, slots, experts, cols = 50, 4, 8, 300
    rows = tokens * slots
    _, order, place = route(rng, tokens, slots, experts, 0.1)
    y, dy = rng.normal(0, 1, (2, rows, cols)).astype(np.float32)
    x, dx = rng.normal(0, 1, (2, tokens, cols)).astype(np.float32)
    w, dw = rng.random((2, tokens, slots)).astype(np.float32)
    g, gr = rng.normal(0, 1, (tokens, cols)).astype(np.float32), rng.normal(0, 1, (rows, cols)).astype(np.float32)
    od, pd = ctx.upload(order.astype(np.int32)), ctx.upload(place.astype(np.int32))

    def combine(y, w):
        out = Result(ctx, tokens, cols, "f32")
        ctx.experts_combine(ctx.upload(y), z.F32, cols, pd, rows, tokens, slots, out.at, weight=ctx.upload(w))
        return out.read().astype(np.float64)

    def gather(x):
        out = Result(ctx, rows, cols, "f32")
        ctx.experts_gather(ctx.upload(x), z.F32, cols, od, rows, tokens, slots, out.at)
        return out.read().astype(np.float64)

    gy, gw, gx = Result(ctx, rows, cols, "f32"), Result(ctx, tokens, slots, "f32"), Result(ctx, tokens, cols, "f32")
    ctx.experts_combine_grad(ctx.upload(g), ctx.upload(y), z.F32, cols, od, pd, ctx.upload(w), rows, tokens, slots,
                             gy.at, gw.at)
    ctx.experts_combine(ctx.upload(gr), z.F32, cols, pd, rows, tokens, slots, gx.at)
    y1, w1, x1 = y + dy, w + dw, x + dx
    base = combine(y, w)
    for step, grad, out, at, weight in [(y1.astype(np.float64) - y, gy, combine(y1, w) - base, g, None),
                                        (w1.astype(np.float64) - w, gw, combine(y, w1) - base, g, None),
                                        (x1.astype(np.float64) - x, gx, gather(x1) - gather(x), gr, None)]:
        left, terms = (out * at).sum(), grad.read().astype(np.float64) * step
        # each output and each gradient carries a few roundings of values of a few units
        lim = 16 * 2.0**-24 * (np.abs(out * at).sum() + np.abs(base).sum() * np.abs(at).max() + np.abs(terms).sum())
        assert abs(left - terms.sum()) <= lim


def test_infinite_rows_stay_where_they_are(ctx):
    """A row that no place names, and the rows of dropped pairs, reach no sum."""
    y = np.full((4, 20), np.inf, dtype=np.float32)
    y[1] = 2.0
    place = np.array([1, -1, -1, -1, 9, 1], dtype=np.int32)  # 9: outside the rows
    out = Result(ctx, 3, 20, "f32")
    ctx.experts_combine(ctx.upload(y), z.F32, 20, ctx.upload(place), 4, 3, 2, out.at)
    got = out.read()
    assert (got[0] == 2).all() and not got[1].any() and (got[2] == 2).all()


@pytest.mark.parametrize("cols", [20, 700])
@pytest.mark.parametrize("slots", [1, 2, 6])
def test_positions_of_no_pair_get_no_gradient(ctx, cols, slots):
    """A position whose order is -1, or any other value that names no pair, becomes
    a row of zeros: as with a position that holds none."""
    rng = np.random.default_rng([cols, slots])
    tokens = 6
    rows = tokens * slots
    _, order, place = route(rng, tokens, slots, 4, 0.0)
    dropped = rng.permutation(rows)[:5]
    place[order[dropped]] = -1
    order[dropped] = [-1, rows, rows + 1, 1 << 30, -2**31]
    g, y = rng.normal(0, 1, (tokens, cols)).astype(np.float32), rng.normal(0, 1, (rows, cols)).astype(np.float32)
    w = rng.random((tokens, slots)).astype(np.float32)
    gy, gw = Result(ctx, rows, cols, "f32"), Result(ctx, tokens, slots, "f32")
    ctx.experts_combine_grad(ctx.upload(g), ctx.upload(y), z.F32, cols, ctx.upload(order.astype(np.int32)),
                             ctx.upload(place.astype(np.int32)), ctx.upload(w), rows, tokens, slots, gy.at, gw.at)
    at = (order >= 0) & (order < rows)
    pair = np.where(at, order, 0)
    want = np.where(at[:, None], w.reshape(-1)[pair][:, None] * g[pair // slots], np.float32(0))
    assert np.array_equal(gy.read(), want)
    assert not gw.read()[place.reshape(tokens, slots) < 0].any()


@pytest.mark.parametrize("tokens", [0, 3])
def test_empty(ctx, tokens):
    d = ctx.upload(np.zeros(4096, dtype=np.int32))
    ctx.experts_gather(d, z.F32, 0, d, 6, tokens, 2, d, ld_x=1, ld_out=1)
    ctx.experts_gather(d, z.F32, 8, d, 0, tokens, 2, d)
    ctx.experts_combine(d, z.F32, 0, d, 6, tokens, 2, d, ld_y=1, ld_out=1)
    gw = Result(ctx, tokens, 2, "f32")
    ctx.experts_combine_grad(d, d, z.F32, 0, d, d, None, 2 * tokens, tokens, 2, d, gw.at)
    assert not gw.read().any()
    out = Result(ctx, 6, 5, "f32")
    ctx.experts_gather(None, z.F32, 5, d, 6, 0, 2, out.at)
    assert not out.read().any()
    out = Result(ctx, tokens, 5, "f32")
    ctx.experts_combine(None, z.F32, 5, d, 0, tokens, 2, out.at)
    assert not out.read().any()


def test_row_refusals(ctx):
    d = ctx.alloc(1 << 16)
    gather = dict(x=d, rows_type=z.F32, cols=8, order=d, rows=4, tokens=2, slots=2, out=d)
    combine = dict(y=d, rows_type=z.F32, cols=8, place=d, rows=4, tokens=2, slots=2, out=d)
    grad = dict(grad=d, y=d, rows_type=z.F32, cols=8, order=d, place=d, weight=d, rows=4, tokens=2, slots=2,
                grad_y=d, grad_weight=d)
    shared = [(dict(rows_type=z.I32), "f32, f16 or bf16"), (dict(slots=0), "slots"),
              (dict(tokens=1 << 22), "2\\^22"), (dict(rows=(1 << 22) + 1), "2\\^22"), (dict(cols=1 << 31), "2\\^31")]
    for f, a, more in [
            (ctx.experts_gather, gather, [(dict(x=None), "null"), (dict(order=None), "null"), (dict(out=None), "null"),
                                          (dict(ld_x=7), "stride"), (dict(ld_out=7), "stride"),
                                          (dict(x=At(d, 2)), "aligned"), (dict(order=At(d, 2)), "aligned")]),
            (ctx.experts_combine, combine, [(dict(y=None), "null"), (dict(place=None), "null"),
                                            (dict(out=None), "null"), (dict(ld_y=7), "stride"),
                                            (dict(ld_out=7), "stride"), (dict(out=At(d, 1)), "aligned"),
                                            (dict(weight=At(d, 2)), "aligned")]),
            (ctx.experts_combine_grad, grad, [(dict(grad=None), "null"), (dict(y=None), "null"),
                                              (dict(order=None), "null"), (dict(place=None), "null"),
                                              (dict(grad_y=None), "null"), (dict(ld_grad=7), "stride"),
                                              (dict(ld_y=7), "stride"), (dict(ld_grad_y=7), "stride"),
                                              (dict(rows=5), "more rows"), (dict(grad_weight=At(d, 2)), "aligned")])]:
        f(**a)
        for bad, why in shared + more:
            with pytest.raises(z.ZkError, match=why):
                f(**dict(a, **bad))
