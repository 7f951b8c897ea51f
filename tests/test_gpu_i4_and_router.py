"""GPU tests of the 4-bit layers and the experts' router as they are used: a routed
step forward and back, calls on other streams and in graphs, rows that lie far apart."""
import ctypes

import numpy as np
import pytest

import router_forms as forms
import zkml_amd as z
from i4_helpers import inputs, near, packed, product
from i8_helpers import At, Result, values

pytestmark = pytest.mark.gpu

hip, vp = ctypes.CDLL("libamdhip64.so"), ctypes.c_void_p


@pytest.fixture(scope="module")
def ctx():
    return z.Context(0)


def say(*a):
    print(*a, flush=True)


def word(ctx, n):
    return ctx.alloc(4 * max(1, n))


@pytest.mark.parametrize("tokens,experts,slots,n_in,n_out", [(1, 8, 2, 96, 40), (37, 6, 3, 300, 70),
                                                             (900, 32, 4, 512, 130)])
def test_a_routed_step(ctx, tokens, experts, slots, n_in, n_out):
    """A 4-bit gate, the routes it names with their balance, the samples sorted, a 4-bit
    layer of each expert, the answers put back; then the gradients of the answers' weights
    and of the balance, back to the gate's scores."""
    rng = np.random.default_rng([tokens, experts])
    rows = tokens * slots
    x = rng.normal(0, 1, (tokens, n_in)).astype(np.float32)
    _, _, gate, gs, gsv = inputs(rng, tokens, experts, n_in, 64)
    _, _, q, s, sv = inputs(rng, tokens, n_out, n_in, 32, "f16", experts)
    b = rng.normal(0, 1, (experts, n_out)).astype(np.float32)
    g, gl = rng.normal(0, 1, (tokens, n_out)).astype(np.float32), np.float32(0.2)
    say("[routed step]", tokens, experts, slots)
    # forward
    xd = ctx.upload(x)
    scores = Result(ctx, tokens, experts, "f32")
    ctx.i4_linear(xd, z.F32, ctx.upload(packed(gate)), ctx.upload(gs), tokens, experts, n_in, 64, scores.at, z.F32,
                  ctx.alloc(ctx.i4_linear_work(tokens, n_in)))
    expert, weight = Result(ctx, tokens, slots, "i32"), Result(ctx, tokens, slots, "f32")
    count, prob, loss = Result(ctx, 1, experts + 1, "i32"), Result(ctx, 1, experts, "f32"), Result(ctx, 1, 1, "f32")
    scale = 1 / 64
    ctx.experts_route(scores.at, z.F32, tokens, experts, slots, expert.at, weight.at, scale=scale, count=count.at,
                      prob=prob.at, loss=loss.at, work=ctx.alloc(max(8, ctx.experts_route_work(tokens, experts))))
    offsets, order, place = word(ctx, experts + 1), word(ctx, rows), word(ctx, rows)
    work = ctx.alloc(max(4, ctx.experts_sort_work(rows, experts)))
    ctx.experts_sort(expert.at, rows, experts, offsets, order, place, work)
    q8, s8 = Result(ctx, tokens, n_in, "i8"), Result(ctx, 1, tokens, "f32")
    ctx.i8_quantize(xd, z.F32, tokens, n_in, q8.at, s8.at)
    y = Result(ctx, rows, n_out, "f32")
    ctx.i4_matmul_experts(q8.at, ctx.upload(packed(q)), ctx.upload(s), offsets, rows, experts, n_out, n_in, 32, y.at,
                          scale_type=z.F16, x_scale=s8.at, bias=ctx.upload(b), order=order, slots=slots, tokens=tokens)
    out = Result(ctx, tokens, n_out, "f32")
    ctx.experts_combine(y.at, z.F32, n_out, place, rows, tokens, slots, out.at, weight=weight.at)
    # back
    gy, gw = Result(ctx, rows, n_out, "f32"), Result(ctx, tokens, slots, "f32")
    ctx.experts_combine_grad(ctx.upload(g), y.at, z.F32, n_out, order, place, weight.at, rows, tokens, slots, gy.at,
                             gw.at)
    gscores = Result(ctx, tokens, experts, "f32")
    ctx.experts_route_grad(scores.at, z.F32, tokens, experts, slots, expert.at, gscores.at, scale=scale,
                           grad_weight=gw.at, count=count.at, grad_loss=ctx.upload(gl.reshape(1)))
    # the same in 64 bits, each step on what the one before gave
    xq, xs = q8.read(), s8.read()[0]
    near(scores.read(), *product(xq, gate, gsv[0], 64, xs, None, False), n_in, "f32")
    v = scores.read().astype(np.float64)
    want = forms.chosen(v, slots)
    assert np.array_equal(expert.read(), want)
    w, lim = forms.weights(v, scale, want, True)
    assert (np.abs(weight.read() - w) <= lim + w * 2.0**-24).all()
    n, p, value, plim, llim = forms.balance(v, scale, want)
    assert np.array_equal(count.read()[0], n)
    assert (np.abs(prob.read()[0] - p) <= plim + p * 2.0**-24).all() and abs(loss.read()[0, 0] - value) <= llim
    answers, size = np.zeros((tokens, slots, n_out)), np.zeros((tokens, slots, n_out))
    for t in range(tokens):
        for j in range(slots):
            e = want[t, j]
            answers[t, j], size[t, j] = (a[0] for a in product(xq[t:t + 1], q[e * n_out:(e + 1) * n_out], sv[e], 32,
                                                               xs[t:t + 1], b[e], False))
    # the layer's bound (near), and those of a weight and of a sum of `slots` terms
    step = (-(-n_in // 32) + 4) * 2.0**-24
    far = (size * step * w[..., None] + np.abs(answers) * (lim + 2.0**-23 * w)[..., None]).sum(1)
    far += (slots + 1) * 2.0**-24 * (np.abs(answers) * w[..., None]).sum(1)
    assert (np.abs(out.read() - (answers * w[..., None]).sum(1)) <= far).all()
    # gradient of the weights: a dot product of n_out terms; then the scores' by formula
    dw = (answers * g[:, None, :]).sum(2)
    dlim = ((size * step + np.abs(answers) * (n_out + 2) * 2.0**-24) * np.abs(g[:, None, :])).sum(2)
    assert (np.abs(gw.read() - dw) <= dlim).all()
    ds, slim = forms.gradient(v, scale, want, True, dw, n, gl)
    slim = slim + 2 * scale * dlim.max(axis=1, keepdims=True) + np.abs(ds) * 2.0**-24
    assert (np.abs(gscores.read() - ds) <= slim).all()


# ---- streams and graphs
def calls(ctx, rng):
    """name: (call(stream, ref), fresh inputs, outputs): ref takes outputs and workspace of
    its own."""
    def linear(rows, n_out, n_in):
        _, _, q, s, _ = inputs(rng, 1, n_out, n_in, 64)
        w, sc, x = ctx.upload(packed(q)), ctx.upload(s), ctx.alloc(rows * n_in * 4)
        out = [ctx.alloc(rows * n_out * 4) for _ in range(2)]
        work = [ctx.alloc(ctx.i4_linear_work(rows, n_in)) for _ in range(2)]

        def call(stream, ref):
            ctx.i4_linear(x, z.F32, w, sc, rows, n_out, n_in, 64, out[ref], z.F32, work[ref], stream=stream)
        return call, lambda: ctx.h2d(x, rng.normal(0, 1, (rows, n_in)).astype(np.float32)), [out]

    def grouped(tokens, slots, experts, n_out, n_in):
        _, _, q, s, _ = inputs(rng, 1, n_out, n_in, 128, experts=experts)
        rows = tokens * slots
        w, sc, x, e = ctx.upload(packed(q)), ctx.upload(s), ctx.alloc(tokens * n_in), ctx.alloc(rows * 4)
        offsets, order, place = ([word(ctx, n) for _ in range(2)] for n in (experts + 1, rows, rows))
        work = [ctx.alloc(max(4, ctx.experts_sort_work(rows, experts))) for _ in range(2)]
        out = [ctx.alloc(rows * n_out * 4) for _ in range(2)]

        def call(stream, ref):
            ctx.experts_sort(e, rows, experts, offsets[ref], order[ref], place[ref], work[ref], stream=stream)
            ctx.i4_matmul_experts(x, w, sc, offsets[ref], rows, experts, n_out, n_in, 128, out[ref], order=order[ref],
                                  slots=slots, tokens=tokens, stream=stream)

        def fresh():
            ctx.h2d(x, rng.integers(-127, 128, (tokens, n_in)).astype(np.int8))
            ctx.h2d(e, rng.integers(-1, experts, rows).astype(np.int32))
        return call, fresh, [out]

    def router(tokens, experts, slots):
        s = ctx.alloc(tokens * experts * 4)
        gw, gl = ctx.upload(rng.normal(0, 1, (tokens, slots)).astype(np.float32)), ctx.upload(np.ones(1, np.float32))
        sizes = (tokens * slots, tokens * slots, experts + 1, experts, 1, tokens * experts)
        outs = [[word(ctx, n) for _ in range(2)] for n in sizes]
        work = [ctx.alloc(max(8, ctx.experts_route_work(tokens, experts))) for _ in range(2)]

        def call(stream, ref):
            expert, weight, count, prob, loss, grad = (o[ref] for o in outs)
            ctx.experts_route(s, z.F32, tokens, experts, slots, expert, weight, count=count, prob=prob, loss=loss,
                              work=work[ref], stream=stream)
            ctx.experts_route_grad(s, z.F32, tokens, experts, slots, expert, grad, grad_weight=gw, count=count,
                                   grad_loss=gl, stream=stream)
        return call, lambda: ctx.h2d(s, rng.normal(0, 1, (tokens, experts)).astype(np.float32)), outs

    return {"few rows": linear(3, 70, 300), "rows": linear(40, 90, 700), "many rows": linear(700, 300, 1100),
            "experts": grouped(30, 2, 8, 100, 260), "many experts' rows": grouped(900, 3, 5, 260, 300),
            "one block": router(50, 20, 2), "blocks": router(3000, 200, 4)}


NAMES = ["few rows", "rows", "many rows", "experts", "many experts' rows", "one block", "blocks"]


def same(ctx, outs):
    ctx.sync()
    for got, ref in outs:
        a, b = ctx.d2h(got, (got.nbytes,), np.uint8), ctx.d2h(ref, (ref.nbytes,), np.uint8)
        assert a.any() and np.array_equal(a, b)


@pytest.mark.parametrize("name", NAMES)
def test_other_streams_and_graphs(ctx, name):
    """Calls on the default stream, on one of the caller's, and recorded into a graph that
    is replayed on new inputs, with eager calls of other outputs between."""
    call, fresh, outs = calls(ctx, np.random.default_rng(3))[name]
    say("[streams]", name)

    def check():
        call(None, 1)  # the context's own stream
        same(ctx, outs)

    fresh()
    call(z.LEGACY_STREAM, 0)
    assert hip.hipDeviceSynchronize() == 0
    check()
    st, graph, exe = vp(), vp(), vp()
    assert hip.hipStreamCreate(ctypes.byref(st)) == 0
    try:
        fresh()
        call(st, 0)
        assert hip.hipStreamSynchronize(st) == 0
        check()
        assert hip.hipStreamBeginCapture(st, 0) == 0
        call(st, 0)
        assert hip.hipStreamEndCapture(st, ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0)) == 0
        for _ in range(4):
            fresh()
            assert hip.hipGraphLaunch(exe, st) == 0
            assert hip.hipStreamSynchronize(st) == 0
            check()
    finally:
        if exe:
            hip.hipGraphExecDestroy(exe)
        if graph:
            hip.hipGraphDestroy(graph)
        hip.hipStreamDestroy(st)


def test_two_streams_at_once(ctx):
    """The same calls on two streams, each with outputs and a workspace of its own."""
    a, b = vp(), vp()
    for s in (a, b):
        assert hip.hipStreamCreate(ctypes.byref(s)) == 0
    try:
        for name, (call, fresh, outs) in calls(ctx, np.random.default_rng(4)).items():
            say("[two streams]", name)
            fresh()
            for _ in range(5):
                call(a, 0)
                call(b, 1)
            assert hip.hipDeviceSynchronize() == 0
            same(ctx, outs)
    finally:
        hip.hipStreamDestroy(a)
        hip.hipStreamDestroy(b)


def test_a_workspace_of_several_calls(ctx):
    """One workspace for calls of several sizes, one after the other on a stream, whatever
    it held before."""
    rng = np.random.default_rng(6)
    work = ctx.upload(np.full(1 << 20, 0xFF, dtype=np.uint8))
    for tokens, experts in [(5000, 100), (2000, 500), (9000, 33), (100, 8), (5000, 100)]:
        s = rng.normal(0, 1, (tokens, experts)).astype(np.float32)
        expert = rng.integers(0, experts, (tokens, 2)).astype(np.int32)
        assert ctx.experts_route_work(tokens, experts) <= 1 << 20
        count, prob, loss = Result(ctx, 1, experts + 1, "i32"), Result(ctx, 1, experts, "f32"), Result(ctx, 1, 1, "f32")
        ctx.experts_balance(ctx.upload(s), z.F32, tokens, experts, 2, ctx.upload(expert), count.at, prob.at, loss.at,
                            work)
        n, p, value, plim, llim = forms.balance(s.astype(np.float64), 1.0, expert)
        assert np.array_equal(count.read()[0], n)
        assert (np.abs(prob.read()[0] - p) <= plim + p * 2.0**-24).all() and abs(loss.read()[0, 0] - value) <= llim


# ---- rows that lie far apart
@pytest.mark.parametrize("rows,n_out,n_in,grouped", [(3, 40, 272, False), (600, 300, 272, False),
                                                     (600, 150, 101, False), (600, 140, 272, True),
                                                     (20, 40, 272, True)])
def test_rows_beyond_32_bits(ctx, rows, n_out, n_in, grouped):
    """x's and w's rows at strides whose last ones lie more than 4 GiB from the first."""
    rng = np.random.default_rng([rows, n_in])
    x, sx, q, s, sv = inputs(rng, rows, n_out, n_in, 64)
    w = packed(q, rng)
    ld_x, ld_w = ((1 << 32) // (rows - 1) + 16) // 16 * 16 + (n_in % 16), ((1 << 32) // (n_out - 1) + 16) // 16 * 16
    say("[far rows]", rows, n_out, n_in, grouped)
    dx, dw = ctx.alloc(rows * ld_x), ctx.alloc(n_out * ld_w)
    for buf, ld, a in ((dx, ld_x, x), (dw, ld_w, w)):
        for r in range(len(a)):
            ctx.h2d(At(buf, r * ld), a[r])
    y = Result(ctx, rows, n_out, "f32")
    more = dict(x_scale=ctx.upload(sx), ld_x=ld_x, ld_w=ld_w)
    if grouped:
        order = rng.permutation(rows).astype(np.int32)
        ctx.i4_matmul_experts(dx, dw, ctx.upload(s), ctx.upload(np.array([0, rows], dtype=np.int32)), rows, 1, n_out,
                              n_in, 64, y.at, order=ctx.upload(order), tokens=rows, **more)
        x, sx = x[order], sx[order]
    else:
        ctx.i4_matmul(dx, dw, ctx.upload(s), rows, n_out, n_in, 64, y.at, **more)
    near(y.read(), *product(x, q, sv[0], 64, sx, None, False), n_in, "f32")


def test_scores_beyond_32_bits(ctx):
    rng = np.random.default_rng(7)
    tokens, experts, slots, ld = 600, 40, 3, (1 << 21) + 3
    s = rng.normal(0, 1, (tokens, experts)).astype(np.float32)
    d, grad = ctx.alloc(tokens * ld * 4), ctx.alloc(tokens * ld * 4)
    say("[far scores]")
    for t in range(tokens):
        ctx.h2d(At(d, t * ld * 4), s[t])
    expert, weight = Result(ctx, tokens, slots, "i32"), Result(ctx, tokens, slots, "f32")
    gw = rng.normal(0, 1, (tokens, slots)).astype(np.float32)
    ctx.experts_route(d, z.F32, tokens, experts, slots, expert.at, weight.at, ld=ld)
    ctx.experts_route_grad(d, z.F32, tokens, experts, slots, expert.at, grad, grad_weight=ctx.upload(gw), ld=ld,
                           ld_grad=ld)
    v = s.astype(np.float64)
    want = forms.chosen(v, slots)
    assert np.array_equal(expert.read(), want)
    ds, lim = forms.gradient(v, 1.0, want, True, gw)
    for t in (0, 1, 255, 256, tokens - 1):
        got = values(ctx.d2h(At(grad, t * ld * 4), (experts,), np.float32), "f32")
        assert (np.abs(got - ds[t]) <= lim[t] + np.abs(ds[t]) * 2.0**-24).all()
