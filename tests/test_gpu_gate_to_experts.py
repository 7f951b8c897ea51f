"""GPU test of a statement's gate in front of 4-bit experts, without the host between: the
gate's exact sums, the routes and weights that they name, the samples sorted, a 4-bit layer
of each class, the answers put back."""
import os
import sys

import numpy as np
import pytest

import router_forms as forms
import zkml_amd as z
from i4_helpers import product, unpacked
from i8_helpers import Result

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "cuda-zkml_amd", "examples"))
from routed_scores import CLASSES, HIDDEN, PIXELS, TEMPERATURE, model, top_two  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return z.Context(0)


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("samples", [1, 37, 5000])
def test_gate_to_experts(ctx, samples, bias):
    rng = np.random.default_rng(samples)
    m, n, slots, group = model(rng), samples, 2, 32
    x = rng.integers(0, 17, (n, PIXELS)).astype(np.int8)
    x[-1] = x[0]  # (as scores are equal, so are routes)
    exact = x.astype(np.int64) @ m["gate_w"].astype(np.int64).T + (m["gate_b"] if bias else 0)
    scale = float(np.float32(1 / TEMPERATURE))
    print("[gate to experts]", samples, bias, flush=True)
    # the gate, to routes and weights
    kind = "f32" if bias else "i32"
    assert np.abs(exact).max() < 2**24
    xd, scores = ctx.upload(x), Result(ctx, n, CLASSES, kind)
    gate_b = ctx.upload(m["gate_b"].astype(np.float32)) if bias else None
    ctx.i8_matmul(xd, ctx.upload(m["gate_w"]), n, CLASSES, PIXELS, scores.at, z.F32 if bias else z.I32, bias=gate_b)
    expert, weight = Result(ctx, n, slots, "i32"), Result(ctx, n, slots, "f32")
    ctx.experts_route(scores.at, z.F32 if bias else z.I32, n, CLASSES, slots, expert.at, weight.at, scale=scale)
    # the experts: their weights quantized to 4 bits
    w, _, b = m["first"]
    wide = (w * np.float32(0.01)).reshape(CLASSES * HIDDEN, PIXELS)
    groups = PIXELS // group
    q8, s4 = [], []
    for e in range(CLASSES):
        q, s = Result(ctx, HIDDEN, 64, "i8"), Result(ctx, groups, HIDDEN, "f32")
        ctx.i4_quantize(ctx.upload(wide[e * HIDDEN:(e + 1) * HIDDEN]), z.F32, HIDDEN, PIXELS, group, q.at, s.at)
        q8.append(q.read())
        s4.append(s.read())
    q8, s4 = np.concatenate(q8), np.stack(s4)
    rows = n * slots
    offsets, order, place = (ctx.alloc(4 * k) for k in (CLASSES + 1, rows, rows))
    work = ctx.alloc(max(4, ctx.experts_sort_work(rows, CLASSES)))
    ctx.experts_sort(expert.at, rows, CLASSES, offsets, order, place, work)
    y, out = Result(ctx, rows, HIDDEN, "f32"), Result(ctx, n, HIDDEN, "f32")
    ctx.i4_matmul_experts(xd, ctx.upload(q8), ctx.upload(s4), offsets, rows, CLASSES, HIDDEN, PIXELS, group, y.at,
                          bias=ctx.upload(b), relu=True, order=order, slots=slots, tokens=n)
    ctx.experts_combine(y.at, z.F32, HIDDEN, place, rows, n, slots, out.at, weight=weight.at)
    # the same on the host
    assert np.array_equal(scores.read(), exact)
    classes, _ = top_two(exact)
    assert np.array_equal(expert.read(), classes)
    want, lim = forms.weights(exact.astype(np.float64), scale, classes, True)
    got = weight.read()
    assert (np.abs(got - want) <= lim + want * 2.0**-24).all()
    total, far = np.zeros((n, HIDDEN)), np.zeros((n, HIDDEN))
    weights = unpacked(q8.view(np.uint8), PIXELS)
    for j in range(slots):
        for e in range(CLASSES):
            at = np.nonzero(classes[:, j] == e)[0]
            v, size = product(x[at], weights[e * HIDDEN:(e + 1) * HIDDEN], s4[e].astype(np.float64), group, None, b[e],
                              True)
            total[at] += got[at, j, None] * v
            # a layer's bound (i4_helpers.near), then a product and a sum of two
            far[at] += got[at, j, None] * (size * (PIXELS // 32 + 4) + np.abs(v) * (slots + 1)) * 2.0**-24
    assert (np.abs(out.read() - total) <= far).all()
