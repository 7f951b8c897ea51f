"""GPU tests of the experts' router (cuda-zkml_amd/csrc/router.hip) where its inputs end:
padding that carries routes, scores and scales at the ends of the range, gradients that
are no numbers, and the sums over many tokens."""
import numpy as np
import pytest

import router_forms as forms
import zkml_amd as z
from i8_helpers import TYPES, Result, values, words
from test_gpu_router import outputs, say, scores, within, work_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return z.Context(0)


def balance(s, scale, expert):
    """forms.balance over the tokens that have a score, within the sums as they are made:
    a lane adds its tokens one after the other, 16 or those of one group of lanes in 256
    blocks (of 64, 16 or 8 groups); then at most 2 sums over lanes, 15 over waves, and a
    product and two roundings on the way; the blocks' are added in 64 bits."""
    on = (s > -np.inf).any(axis=1)
    tokens, experts, n = len(s), s.shape[1], int(on.sum())
    groups = 64 if experts <= 256 else 16 if experts <= 512 else 8
    depth = max(16, -(-tokens // (256 * groups))) + 20
    p, R = forms.softmax(s, scale)
    count = np.array([(expert[on] == e).sum() for e in range(experts)] + [n])
    prob = p.sum(axis=0) / max(n, 1)
    lim = (p * R).sum(axis=0) / max(n, 1) + depth * 2.0**-24 * prob + 2.0**-126
    f = count[:-1] / max(1, n * expert.shape[1])
    loss = experts * (f * prob).sum()
    return count, prob, loss, lim, experts * (f * lim).sum() + 2.0**-23 * loss


def check_balance(o, want):
    count, prob, loss, prob_lim, loss_lim = want
    assert np.array_equal(o["count"].read()[0], count)
    within(o["prob"].read()[0], prob, prob_lim)
    within(o["loss"].read(), np.array([[loss]]), loss_lim)


@pytest.mark.parametrize("kind", ["f32", "bf16", "i32"])
@pytest.mark.parametrize("tokens,experts,slots", [(1, 4, 1), (50, 20, 2), (300, 1024, 3), (3000, 24, 20), (700, 400, 2)])
def test_padding_that_names_experts(ctx, kind, tokens, experts, slots):
    """Tokens without a score count for nothing, whatever their routes hold; one block's
    batches and larger ones."""
    rng = np.random.default_rng([tokens, experts])
    s, v = scores(rng, tokens, experts, kind)
    none = rng.random(tokens) < 0.4
    none[-1] = True
    s[none] = -2**31 if kind == "i32" else words(np.array([-np.inf]), kind)[0]
    v[none] = -np.inf
    expert = rng.integers(0, experts, (tokens, slots)).astype(np.int32)
    expert[none, 0] = 0
    scale = 2.0**-12 if kind == "i32" else 1.25
    say("[balance with padding]", kind, tokens, experts, slots)
    o = outputs(ctx, tokens, experts, slots, True)
    ctx.experts_balance(ctx.upload(s), TYPES[kind], tokens, experts, slots, ctx.upload(expert), o["count"].at,
                        o["prob"].at, o["loss"].at, work_of(ctx, tokens, experts), scale=scale)
    check_balance(o, balance(v, scale, expert))


def pass_through(ctx, s, v, kind, scale, slots, renormalize, gw, gl):
    """Routes with balance and the gradient of these scores, against the 64-bit forms."""
    tokens, experts = v.shape
    want = forms.chosen(v, slots)
    d, o = ctx.upload(s), outputs(ctx, tokens, experts, slots, True)
    ctx.experts_route(d, TYPES[kind], tokens, experts, slots, scale=scale, renormalize=renormalize,
                      work=work_of(ctx, tokens, experts), **{k: r.at for k, r in o.items()})
    assert np.array_equal(o["expert"].read(), want)
    within(o["weight"].read(), *forms.weights(v, scale, want, renormalize))
    check_balance(o, balance(v, scale, want))
    if kind == "i32":
        return
    out = Result(ctx, tokens, experts, kind)
    ctx.experts_route_grad(d, TYPES[kind], tokens, experts, slots, o["expert"].at, out.at, scale=scale,
                           renormalize=renormalize, grad_weight=ctx.upload(gw), count=o["count"].at,
                           grad_loss=ctx.upload(np.array([gl], np.float32)))
    count = o["count"].read()[0]
    within(out.read(), *forms.gradient(v, scale, want, renormalize, gw, count, np.float32(gl)), kind)


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16", "i32"])
@pytest.mark.parametrize("tokens,experts", [(200, 12), (60, 300)])
def test_the_largest_scales(ctx, kind, renormalize, tokens, experts):
    """Scales up to the end of the range: a softmax of zeros and equal parts."""
    rng = np.random.default_rng([tokens, experts, 3])
    s, v = scores(rng, tokens, experts, kind, 0.2, ties=True)
    for scale in (2.0**127, float(np.finfo(np.float32).max)):
        say("[large scale]", kind, renormalize, tokens, experts)
        # gradients that the scores' type holds
        g = 2.0**-116 if kind == "f16" else 2.0**-20
        pass_through(ctx, s, v, kind, scale, 3, renormalize, (rng.normal(0, 1, (tokens, 3)) * g).astype(np.float32), g)


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_differences_beyond_the_range(ctx, kind, renormalize):
    """Scores whose difference no 32-bit float holds, at a scale where it matters."""
    rng = np.random.default_rng(11)
    big = 2.0**127 * 1.75
    v = rng.choice([-big, -big / 2, 0.0, big / 4, big], (100, 6))
    v[0], v[1] = [big, -big, -big, -big, -big, -big], [-np.inf, -big, big, -np.inf, big, 0]
    s = words(v, kind)
    say("[far scores]", kind, renormalize)
    pass_through(ctx, s, v, kind, 2.0**-124, 3, renormalize,
                 (rng.normal(0, 1, (100, 3)) * 2.0**100).astype(np.float32), 2.0**100)


@pytest.mark.parametrize("renormalize", [True, False])
def test_the_smallest_scales(ctx, renormalize):
    """A scale below the normal numbers costs the gradient nothing of its precision."""
    rng = np.random.default_rng(12)
    v = words(rng.uniform(-1, 1, (100, 6)) * 2.0**127, "f32")
    say("[small scale]", renormalize)
    pass_through(ctx, v, v.astype(np.float64), "f32", 2.0**-140, 3, renormalize,
                 (rng.normal(0, 1, (100, 3)) * 2.0**110).astype(np.float32), 2.0**110)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("tokens,experts,slots", [(40, 13, 3), (30, 300, 20)])
def test_masked_scores_of_any_gradient(ctx, kind, renormalize, tokens, experts, slots):
    """Incoming gradients that overflowed, or are no numbers, leave masked scores' at zero;
    the weights' stay with their token."""
    rng = np.random.default_rng([tokens, experts, 5])
    s, v = scores(rng, tokens, experts, kind, 0.4)
    v[2] = -np.inf
    s[2] = words(v[2], kind)
    expert = forms.chosen(v, slots).astype(np.int32)
    gw = rng.normal(0, 1, (tokens, slots)).astype(np.float32)
    lost = [5, 9, 11]
    gw[5, 0], gw[9, 1], gw[11, 0], gw[11, 1] = np.inf, np.nan, -np.inf, np.inf
    count = forms.balance(v, 1.0, expert)[0]
    say("[masked gradients]", kind, renormalize, tokens, experts, slots)
    for gl in (0.5, np.inf, np.nan):
        out = Result(ctx, tokens, experts, kind)
        ctx.experts_route_grad(ctx.upload(s), TYPES[kind], tokens, experts, slots, ctx.upload(expert), out.at,
                               renormalize=renormalize, grad_weight=ctx.upload(gw),
                               count=ctx.upload(count.astype(np.int32)),
                               grad_loss=ctx.upload(np.array([gl], np.float32)))
        got = out.read()
        assert not values(got, kind)[v == -np.inf].any()
        if gl == 0.5:
            fine = [t for t in range(tokens) if t not in lost]
            within(got[fine], *forms.gradient(v[fine], 1.0, expert[fine], renormalize, gw[fine], count, gl), kind)


@pytest.mark.parametrize("tokens,experts,kind", [(1 << 20, 7, "bf16"), (200000, 60, "f32"), (30000, 300, "f16"),
                                                 (20000, 700, "i32")])
def test_sums_over_many_tokens(ctx, tokens, experts, kind):
    """Bounds of the sums as they are made: no wave's, block's or pass's part can be missing."""
    rng = np.random.default_rng([tokens, experts])
    s, v = scores(rng, tokens, experts, kind)
    scale = 2.0**-12 if kind == "i32" else 1.0
    expert = rng.integers(0, experts, (tokens, 2)).astype(np.int32)
    say("[many tokens]", tokens, experts, kind)
    o = outputs(ctx, tokens, experts, 2, True)
    ctx.experts_balance(ctx.upload(s), TYPES[kind], tokens, experts, 2, ctx.upload(expert), o["count"].at,
                        o["prob"].at, o["loss"].at, work_of(ctx, tokens, experts), scale=scale)
    want = balance(v, scale, expert)
    check_balance(o, want)
    prob, lim = want[1], want[3]
    assert (lim <= 1e-4 * prob).all() and abs(o["prob"].read().sum(dtype=np.float64) - 1) <= lim.sum()


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("tokens,experts,slots,kind", [(100001, 24, 2, "f32"), (33000, 70, 20, "bf16"),
                                                       (9000, 600, 3, "f16")])
def test_several_tokens_a_group_of_lanes(ctx, tokens, experts, slots, kind, renormalize):
    """Routes without the balance, and gradients, of more tokens than a launch has groups."""
    rng = np.random.default_rng(tokens)
    s, v = scores(rng, tokens, experts, kind, 0.1)
    gw = rng.normal(0, 1, (tokens, slots)).astype(np.float32)
    say("[several tokens]", tokens, experts, slots, kind, renormalize)
    d, o = ctx.upload(s), outputs(ctx, tokens, experts, slots, False)
    ctx.experts_route(d, TYPES[kind], tokens, experts, slots, renormalize=renormalize, **{k: r.at for k, r in o.items()})
    want = forms.chosen(v, slots)
    assert np.array_equal(o["expert"].read(), want)
    within(o["weight"].read(), *forms.weights(v, 1.0, want, renormalize))
    count = balance(v, 1.0, want)[0]
    out = Result(ctx, tokens, experts, kind)
    ctx.experts_route_grad(d, TYPES[kind], tokens, experts, slots, o["expert"].at, out.at, renormalize=renormalize,
                           grad_weight=ctx.upload(gw), count=ctx.upload(count.astype(np.int32)),
                           grad_loss=ctx.upload(np.array([0.3], np.float32)))
    within(out.read(), *forms.gradient(v, 1.0, want, renormalize, gw, count, np.float32(0.3)), kind)
