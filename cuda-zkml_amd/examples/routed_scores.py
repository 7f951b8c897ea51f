"""Samples routed by a quantized gate to experts that answer them, on the GPU,
and a proof of one sample's route.

The gate is an integer linear layer (int8 weights, integer pixels): its scores
over the whole batch are the integers that a statement proves, so each sample's
two best classes and their margin are known before anything is proven.  The
samples are sorted by these classes; class e's expert, two linear layers with a
ReLU between them in 8-bit integers, answers its samples; the two answers of a
sample are put back weighted by the softmax of its two scores.  For the sample
with the smallest margin a statement with in-circuit routing is built, its
scores compared with the GPU's, proven and verified.

    python cuda-zkml_amd/examples/routed_scores.py [samples]
"""
import os
import sys
import tempfile

import numpy as np

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import zkml_amd as z  # noqa: E402

PIXELS, CLASSES, HIDDEN, ANSWER = 64, 10, 96, 40
TEMPERATURE = 2000.0  # of the gate's integer scores


def model(rng):
    """Gate (int8 weights, int32 bias) and experts (float weights, quantized by
    output channel)."""
    def layer(n_out, n_in):
        w = rng.normal(0, n_in ** -0.5, (CLASSES, n_out, n_in)).astype(np.float32)
        scale = np.abs(w).max(axis=2) / np.float32(127)
        return np.rint(w / scale[..., None]).astype(np.int8), scale, rng.normal(0, 0.1, (CLASSES, n_out)).astype(np.float32)

    return {"gate_w": rng.integers(-127, 128, (CLASSES, PIXELS)).astype(np.int8),
            "gate_b": rng.integers(-3000, 3000, CLASSES),
            "first": layer(HIDDEN, PIXELS), "second": layer(ANSWER, HIDDEN)}


def gate_scores(ctx, m, x):
    """The gate's exact integer scores of integer samples (n, PIXELS)."""
    n = len(x)
    d_y = ctx.alloc(n * CLASSES * 4)
    ctx.i8_matmul(ctx.upload(x.astype(np.int8)), ctx.upload(m["gate_w"]), n, CLASSES, PIXELS, d_y)
    return ctx.d2h(d_y, (n, CLASSES), np.int32).astype(np.int64) + m["gate_b"]


def top_two(scores):
    """(classes, margin): a sample's two best classes, of equal scores the first."""
    order = np.argsort(-scores, axis=1, kind="stable")[:, :2]
    best = np.take_along_axis(scores, order, axis=1)
    return order.astype(np.int32), best[:, 0] - best[:, 1]


def answers(ctx, m, x, classes, weights):
    """The experts' weighted answers (n, ANSWER)."""
    n, slots = classes.shape
    rows = n * slots
    word = lambda k: ctx.alloc(4 * max(1, k))  # noqa: E731
    # samples by class
    offsets, order, place = word(CLASSES + 1), word(rows), word(rows)
    work = ctx.alloc(max(1, ctx.experts_sort_work(rows, CLASSES)))
    ctx.experts_sort(ctx.upload(classes), rows, CLASSES, offsets, order, place, work)
    # samples to 8 bits, first layer with ReLU: each position takes its sample's row
    q, s = ctx.alloc(n * PIXELS), word(n)
    ctx.i8_quantize(ctx.upload(x.astype(np.float32)), z.F32, n, PIXELS, q, s)
    w, ws, b = (ctx.upload(a) for a in m["first"])
    hidden = word(rows * HIDDEN)
    ctx.i8_matmul_experts(q, w, offsets, rows, CLASSES, HIDDEN, PIXELS, hidden, z.F32, x_scale=s, w_scale=ws, bias=b,
                          relu=True, order=order, slots=slots, tokens=n)
    # second layer: its rows are in the experts' order already
    q2, s2 = ctx.alloc(rows * HIDDEN), word(rows)
    ctx.i8_quantize(hidden, z.F32, rows, HIDDEN, q2, s2)
    w, ws, b = (ctx.upload(a) for a in m["second"])
    y = word(rows * ANSWER)
    ctx.i8_matmul_experts(q2, w, offsets, rows, CLASSES, ANSWER, HIDDEN, y, z.F32, x_scale=s2, w_scale=ws, bias=b)
    # back to the samples' order
    out = word(n * ANSWER)
    ctx.experts_combine(y, z.F32, ANSWER, place, rows, n, slots, out, weight=ctx.upload(weights))
    return ctx.d2h(out, (n, ANSWER), np.float32)


def prove_route(ctx, m, x, threshold):
    """Statement with routing for one sample: (scores, class, flag, verified)."""
    st = z.statement_v2([z.layer_linear(PIXELS, CLASSES, m["gate_w"], m["gate_b"])], x[None], route_threshold=threshold)
    flag, best = (z.words_int(w) for w in st.publics_std()[st.layout["route_start"]:][:2])
    r1cs = ctx.r1cs(st.nc, st.nv, st.npub, st.A, st.B, st.C)
    with tempfile.TemporaryDirectory() as td:
        pk_path, vk_path = os.path.join(td, "pk.bin"), os.path.join(td, "vk.bin")
        ctx.setup(r1cs, 0xDEADBEEF42, pk_path, vk_path)
        proof, _ = ctx.prove(ctx.load_pk(pk_path), r1cs, st.w, st.npub, 0xCAFEBABE)
        with open(vk_path, "rb") as f:
            ok = z.verify(f.read(), proof, st.publics_std())
    return st.scores[0], best, flag, ok


def run(samples, seed=1):
    rng = np.random.default_rng(seed)
    ctx, m = z.Context(0), model(rng)
    x = rng.integers(0, 17, (samples, PIXELS))
    scores = gate_scores(ctx, m, x)
    classes, margin = top_two(scores)
    best = np.take_along_axis(scores, classes, axis=1) / TEMPERATURE
    weights = np.exp(best - best.max(axis=1, keepdims=True))
    weights = (weights / weights.sum(axis=1, keepdims=True)).astype(np.float32)
    out = answers(ctx, m, x, classes, weights)
    i = int(margin.argmin())
    threshold = int(np.median(margin))
    proven, best_class, flag, ok = prove_route(ctx, m, x[i], threshold)
    return {"model": m, "x": x, "scores": scores, "classes": classes, "margin": margin, "weights": weights,
            "answers": out, "sample": i, "threshold": threshold, "proven_scores": proven,
            "proven_class": best_class, "proven_flag": flag, "verified": ok}


if __name__ == "__main__":
    r = run(int(sys.argv[1]) if len(sys.argv) > 1 else 10000)
    i = r["sample"]
    print(f"{len(r['x'])} samples over {CLASSES} experts; {int((r['margin'] >= r['threshold']).sum())} with a margin "
          f"of {r['threshold']} or more")
    print(f"sample {i}: scores {r['scores'][i].tolist()}, statement's {r['proven_scores'].tolist()}")
    print(f"class {r['proven_class']}, margin {r['margin'][i]}, flag {r['proven_flag']}, proof "
          f"{'verified' if r['verified'] else 'REJECTED'}")
    sys.exit(0 if r["verified"] else 1)
