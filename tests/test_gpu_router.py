"""GPU tests of the experts' router (cuda-zkml_amd/csrc/router.hip) against its
64-bit forms (router_forms), whose bounds are the tolerances."""
import numpy as np
import pytest

import router_forms as forms
import zkml_amd as z
from i8_helpers import ROUND, TINY, TYPES, At, Result, matrix, values, words

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return z.Context(0)


def say(*a):
    print(*a, flush=True)


def scores(rng, tokens, experts, kind, masked=0.0, ties=False):
    """(words, values with masked scores as -inf)."""
    s = rng.normal(0, 1.5, (tokens, experts)) + rng.normal(0, 0.5, experts)
    if ties:
        s = np.round(s)
    if kind == "i32":
        s = np.round(s * 4096).astype(np.int32)
        hidden = rng.random(s.shape) < masked
        s[hidden] = -2**31
        v = np.where(hidden, -np.inf, s.astype(np.float64))
        return s, v
    s[rng.random(s.shape) < masked] = -np.inf
    w = words(s, kind)
    return w, values(w, kind)


def within(got, want, lim, kind="f32"):
    lim = lim + (np.abs(want) + lim) * ROUND[kind] + TINY[kind]
    bad = ~(np.abs(values(got, kind) - want) <= lim)
    assert not bad.any(), f"{int(bad.sum())} of {bad.size} off, first at {np.argwhere(bad)[0]}"


def outputs(ctx, tokens, experts, slots, balance):
    o = {"expert": Result(ctx, tokens, slots, "i32"), "weight": Result(ctx, tokens, slots, "f32")}
    if balance:
        o.update(count=Result(ctx, 1, experts + 1, "i32"), prob=Result(ctx, 1, experts, "f32"),
                 loss=Result(ctx, 1, 1, "f32"))
    return o


def work_of(ctx, tokens, experts):
    n = ctx.experts_route_work(tokens, experts)
    return ctx.alloc(n) if n else None


# tokens, experts, slots
SIZES = [(1, 1, 1), (1, 8, 2), (3, 2, 2), (5, 3, 8), (33, 8, 2), (17, 16, 4), (64, 17, 3), (100, 32, 6), (70, 60, 4), (257, 60, 2),
         (300, 1024, 3), (700, 400, 2),
         (65, 64, 8), (129, 65, 5), (300, 128, 8), (40, 129, 4), (31, 256, 32), (50, 300, 17), (9, 512, 8),
         (20, 1000, 10), (7, 1024, 32), (3000, 24, 2)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16", "i32"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("masked,ties,pad", [(0.0, False, 0), (0.4, True, 3)])
@pytest.mark.parametrize("tokens,experts,slots", SIZES)
def test_route(ctx, kind, renormalize, masked, ties, pad, tokens, experts, slots):
    rng = np.random.default_rng([tokens, experts, slots])
    s, v = scores(rng, tokens, experts, kind, masked, ties)
    scale = 2.0**-12 if kind == "i32" else 0.75
    say("[route]", kind, renormalize, masked, tokens, experts, slots)
    d = matrix(ctx, s, experts + pad, pad, fill=0xFF)
    want = forms.chosen(v, slots)
    w, lim = forms.weights(v, scale, want, renormalize)
    count, prob, loss, prob_lim, loss_lim = forms.balance(v, scale, want)
    for balance in (False, True):
        o = outputs(ctx, tokens, experts, slots, balance)
        more = dict({k: r.at for k, r in o.items()}, work=work_of(ctx, tokens, experts) if balance else None)
        ctx.experts_route(d, TYPES[kind], tokens, experts, slots, scale=scale, renormalize=renormalize,
                          ld=experts + pad, **more)
        assert np.array_equal(o["expert"].read(), want)
        within(o["weight"].read(), w, lim)
        if balance:
            assert np.array_equal(o["count"].read()[0], count)
            within(o["prob"].read()[0], prob, prob_lim)
            within(o["loss"].read(), np.array([[loss]]), loss_lim)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16", "i32"])
@pytest.mark.parametrize("tokens,experts,slots", SIZES + [(40000, 128, 2), (20000, 200, 1)])
def test_balance_of_given_routes(ctx, kind, tokens, experts, slots):
    rng = np.random.default_rng([tokens, experts, slots, 1])
    s, v = scores(rng, tokens, experts, kind)
    none = rng.random(tokens) < 0.1  # tokens without a score: padding
    s[none] = -2**31 if kind == "i32" else words(np.array([-np.inf]), kind)[0]
    v[none] = -np.inf
    expert = rng.integers(-1, experts + 1, (tokens, slots)).astype(np.int32)
    expert[none] = -1
    expert[rng.random((tokens, slots)) < 0.01] = -2**31
    scale = 2.0**-12 if kind == "i32" else 1.25
    say("[balance]", kind, tokens, experts, slots)
    o = outputs(ctx, tokens, experts, slots, True)
    ctx.experts_balance(ctx.upload(s), TYPES[kind], tokens, experts, slots, ctx.upload(expert), o["count"].at,
                        o["prob"].at, o["loss"].at, work_of(ctx, tokens, experts), scale=scale)
    count, prob, loss, prob_lim, loss_lim = forms.balance(v, scale, expert)
    assert np.array_equal(o["count"].read()[0], count)
    within(o["prob"].read()[0], prob, prob_lim)
    within(o["loss"].read(), np.array([[loss]]), loss_lim)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("masked,pad", [(0.0, 0), (0.3, 5)])
@pytest.mark.parametrize("tokens,experts,slots", SIZES)
def test_gradient(ctx, kind, renormalize, masked, pad, tokens, experts, slots):
    rng = np.random.default_rng([tokens, experts, slots, 2])
    s, v = scores(rng, tokens, experts, kind, masked)
    expert = forms.chosen(v, slots).astype(np.int32)
    expert[rng.random(expert.shape) < 0.1] = -1  # over capacity
    gw, gl = rng.normal(0, 1, (tokens, slots)).astype(np.float32), np.float32(0.3)
    # a slot that names no expert has no weight, whatever its gradient
    gw[expert < 0] = np.nan
    count = forms.balance(v, 0.75, expert)[0]
    d, ed = matrix(ctx, s, experts + pad, pad, fill=0xFF), ctx.upload(expert)
    say("[route grad]", kind, renormalize, masked, tokens, experts, slots)
    for weights, loss in ((True, True), (True, False), (False, True)):
        out = Result(ctx, tokens, experts, kind, ld=experts + pad, lead=pad)
        ctx.experts_route_grad(d, TYPES[kind], tokens, experts, slots, ed, out.at, scale=0.75, renormalize=renormalize,
                               grad_weight=ctx.upload(gw) if weights else None,
                               count=ctx.upload(count.astype(np.int32)) if loss else None,
                               grad_loss=ctx.upload(gl.reshape(1)) if loss else None, ld=experts + pad,
                               ld_grad=experts + pad)
        want, lim = forms.gradient(v, 0.75, expert, renormalize, gw if weights else None, count if loss else None, gl)
        within(out.read(), want, lim, kind)


@pytest.mark.parametrize("renormalize", [True, False])
def test_gradient_of_the_same_expert_twice(ctx, renormalize):
    rng = np.random.default_rng(4)
    s, v = scores(rng, 50, 12, "f32")
    expert = rng.integers(-1, 4, (50, 6)).astype(np.int32)
    gw = rng.normal(0, 1, (50, 6)).astype(np.float32)
    out = Result(ctx, 50, 12, "f32")
    ctx.experts_route_grad(ctx.upload(s), z.F32, 50, 12, 6, ctx.upload(expert), out.at, renormalize=renormalize,
                           grad_weight=ctx.upload(gw))
    within(out.read(), *forms.gradient(v, 1.0, expert, renormalize, gw))


@pytest.mark.parametrize("renormalize", [True, False])
def test_gradient_against_differences(ctx, renormalize):
    """The change of sum gw w + gl loss, routes and counts held, for steps of 2^-12 up
    and down in 64 bits: off by the third derivative, at most step^2 of the terms' size."""
    rng = np.random.default_rng(5)
    tokens, experts, slots, scale, gl = 30, 20, 3, 0.75, 0.4
    s, v = scores(rng, tokens, experts, "f32", 0.2)
    expert = forms.chosen(v, slots).astype(np.int32)
    gw = rng.normal(0, 1, (tokens, slots)).astype(np.float32)
    count = forms.balance(v, scale, expert)[0]
    f = count[:-1] / (count[-1] * slots)

    def value(v):
        w, _ = forms.weights(v, scale, expert, renormalize)
        p, _ = forms.softmax(v, scale)
        return (gw * w).sum(1) + gl * experts / count[-1] * (p * f).sum(1)

    out = Result(ctx, tokens, experts, "f32")
    ctx.experts_route_grad(ctx.upload(s), z.F32, tokens, experts, slots, ctx.upload(expert), out.at, scale=scale,
                           renormalize=renormalize, grad_weight=ctx.upload(gw),
                           count=ctx.upload(count.astype(np.int32)), grad_loss=ctx.upload(np.array([gl], np.float32)))
    got, h = out.read().astype(np.float64), 2.0**-12
    _, lim = forms.gradient(v, scale, expert, renormalize, gw, count, gl)
    for e in range(experts):
        step = np.zeros(experts)
        step[e] = h
        want = (value(v + step) - value(v - step)) / (2 * h)
        size = np.abs(gw).sum(1) + gl
        assert (np.abs(got[:, e] - want) <= lim[:, e] + (np.abs(want) + lim[:, e]) * 2.0**-24 + h * h * size).all()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("experts", [5, 100, 700])
def test_rows_without_a_softmax(ctx, kind, experts):
    """Masked rows, rows of the type's lowest value, NaN and infinities, beside others."""
    rng = np.random.default_rng(experts)
    tokens, slots = 40, 3
    s, _ = scores(rng, tokens, experts, kind)
    v = values(s, kind)
    low = {"f32": -np.finfo(np.float32).max, "f16": -65504.0, "bf16": -(2.0**128 - 2.0**120)}[kind]
    v[3] = -np.inf
    v[7, 1:] = -np.inf
    v[9] = low
    v[11, 2:] = low
    v[13, 4] = np.nan
    v[15, 0] = np.inf
    v[17], v[17, 1] = -np.inf, np.nan
    v[39] = -np.inf
    s = words(v, kind)
    v = values(s, kind)
    bad, fine = [13, 15, 17], [t for t in range(tokens) if t not in (13, 15, 17)]
    d = ctx.upload(s)
    for renormalize in (True, False):
        o = outputs(ctx, tokens, experts, slots, True)
        ctx.experts_route(d, TYPES[kind], tokens, experts, slots, renormalize=renormalize,
                          work=work_of(ctx, tokens, experts), **{k: r.at for k, r in o.items()})
        expert, w = o["expert"].read(), o["weight"].read()
        want = forms.chosen(v[fine], slots)
        assert np.array_equal(expert[fine], want)
        within(w[fine], *forms.weights(v[fine], 1.0, want, renormalize))
        assert (expert[bad] == -1).all() and np.isnan(w[bad]).all()
        assert (expert[3] == -1).all() and not w[3].any()
        assert expert[7].tolist() == [0, -1, -1] and w[7].tolist() == [1, 0, 0]
        assert expert[9].tolist() == [0, 1, 2]
        count = o["count"].read()[0]
        assert count[-1] == tokens - 2 and count[:-1].sum() == (expert >= 0).sum()
        assert np.isnan(o["prob"].read()).all() and np.isnan(o["loss"].read()).all()
        gw = rng.normal(0, 1, (tokens, slots)).astype(np.float32)
        out = Result(ctx, tokens, experts, kind)
        ctx.experts_route_grad(d, TYPES[kind], tokens, experts, slots, o["expert"].at, out.at, renormalize=renormalize,
                               grad_weight=ctx.upload(gw), count=o["count"].at,
                               grad_loss=ctx.upload(np.ones(1, np.float32)))
        got = out.read()
        assert np.isnan(values(got[bad], kind)).all() and not values(got[[3, 39]], kind).any()
        within(got[fine], *forms.gradient(v[fine], 1.0, want, renormalize, gw[fine], count, 1.0), kind)


def test_integer_scores_keep_their_order(ctx):
    """Sums that 32-bit floats cannot tell apart, at both ends of their range."""
    s = np.array([[2**30 + 1, 2**30 + 2, 2**30], [-2**31 + 1, -2**31 + 2, -2**31], [2**31 - 1, -2**31 + 1, 0],
                  [-2**31] * 3], dtype=np.int32)
    o = outputs(ctx, 4, 3, 2, False)
    ctx.experts_route(ctx.upload(s), z.I32, 4, 3, 2, o["expert"].at, o["weight"].at, scale=2.0**-30)
    assert o["expert"].read().tolist() == [[1, 0], [1, 0], [0, 2], [-1, -1]]
    v = np.where(s == -2**31, -np.inf, s.astype(np.float64))
    within(o["weight"].read(), *forms.weights(v, 2.0**-30, o["expert"].read(), True))


def test_a_million_tokens(ctx):
    """More tokens than a launch has groups of lanes; sums over all of them."""
    rng = np.random.default_rng(8)
    tokens, experts = 1 << 20, 7
    s, v = scores(rng, tokens, experts, "bf16")
    o = outputs(ctx, tokens, experts, 4, True)
    say("[route] a million tokens")
    ctx.experts_route(ctx.upload(s), z.BF16, tokens, experts, 4, work=work_of(ctx, tokens, experts), renormalize=False,
                      **{k: r.at for k, r in o.items()})
    want = forms.chosen(v, 4)
    assert np.array_equal(o["expert"].read(), want)
    within(o["weight"].read(), *forms.weights(v, 1.0, want, False))
    count, prob, loss, prob_lim, loss_lim = forms.balance(v, 1.0, want)
    assert np.array_equal(o["count"].read()[0], count)
    within(o["prob"].read()[0], prob, prob_lim)
    within(o["loss"].read(), np.array([[loss]]), loss_lim)
    again = outputs(ctx, tokens, experts, 4, True)
    ctx.experts_route(ctx.upload(s), z.BF16, tokens, experts, 4, work=work_of(ctx, tokens, experts), renormalize=False,
                      **{k: r.at for k, r in again.items()})
    for k in o:
        assert o[k].read().tobytes() == again[k].read().tobytes(), "two runs differ"


def test_no_tokens(ctx):
    o = outputs(ctx, 0, 5, 2, True)
    ctx.experts_route(None, z.F32, 0, 5, 2, None, None, count=o["count"].at, prob=o["prob"].at, loss=o["loss"].at)
    assert not o["count"].read().any() and not o["prob"].read().any() and not o["loss"].read().any()
    ctx.experts_route(None, z.F32, 0, 5, 2, None, None)
    o = outputs(ctx, 0, 5, 2, True)
    ctx.experts_balance(None, z.I32, 0, 5, 2, None, o["count"].at, o["prob"].at, o["loss"].at)
    assert not o["count"].read().any() and not o["loss"].read().any()
    ctx.experts_route_grad(None, z.F32, 0, 5, 2, None, None, grad_weight=o["loss"].at)


def test_refusals(ctx):
    d = ctx.upload(np.zeros(1 << 14, dtype=np.int32))
    work = ctx.alloc(ctx.experts_route_work(1200, 8))
    short = ctx.alloc(ctx.experts_route_work(1200, 8) - 4)
    route = dict(scores=d, scores_type=z.F32, tokens=1200, experts=8, slots=2, expert=ctx.alloc(9600),
                 weight=ctx.alloc(9600), count=ctx.alloc(64), prob=ctx.alloc(64), loss=ctx.alloc(64), work=work)
    balance = {k: x for k, x in route.items() if k != "weight"}
    grad = dict(scores=d, scores_type=z.F32, tokens=1200, experts=8, slots=2, expert=d, grad_scores=ctx.alloc(38400),
                grad_weight=d, count=d, grad_loss=d)
    shared = [(dict(experts=0), "1024"), (dict(experts=1025), "1024"), (dict(slots=0), "32 slots"),
              (dict(slots=33), "32 slots"), (dict(tokens=1 << 22), "2\\^22"), (dict(tokens=(1 << 22) + 1), "2\\^22"),
              (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("inf")), "scale"),
              (dict(scale=float("nan")), "scale"), (dict(ld=7), "stride"), (dict(scores=None), "null"),
              (dict(scores=At(d, 2)), "aligned"), (dict(expert=None), "null"), (dict(expert=At(d, 2)), "aligned"),
              (dict(scores_type=9), "type")]
    both = [(dict(count=None), "null"), (dict(prob=None), "null"), (dict(loss=None), "null"),
            (dict(loss=At(d, 2)), "aligned"), (dict(work=None), "workspace"), (dict(work=short), "workspace"),
            (dict(work=At(d, 4)), "workspace")]
    for f, a, more in [(ctx.experts_route, route, both + [(dict(weight=None), "null")]),
                       (ctx.experts_balance, balance, both),
                       (ctx.experts_route_grad, grad, [
                           (dict(grad_scores=None), "null"), (dict(grad_scores=At(d, 2)), "aligned"),
                           (dict(grad_loss=None), "null"), (dict(ld_grad=7), "stride"),
                           (dict(scores_type=z.I32), "gradient"),
                           (dict(grad_weight=None, count=None), "neither")])]:
        f(**a)
        for bad, why in shared + more:
            with pytest.raises(z.ZkError, match=why):
                f(**dict(a, **bad))
    ctx.sync()
    assert ctx.experts_route_work(4, 0) == 0 and ctx.experts_route_work((1 << 22) + 1, 8) == 0
