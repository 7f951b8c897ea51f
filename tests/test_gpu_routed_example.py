"""GPU test of the routed example (cuda-zkml_amd/examples/routed_scores.py): the
gate's integers against the statement's, the experts' answers against the same
layers in 64 bits."""
import importlib.util
import os

import numpy as np
import pytest

import zkml_amd

pytestmark = pytest.mark.gpu


def example():
    path = os.path.join(os.path.dirname(zkml_amd.__file__), "examples", "routed_scores.py")
    spec = importlib.util.spec_from_file_location("routed_scores", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def layer(x, w, scale, bias):
    """One expert's layer in 64 bits over rows quantized as the library does, and
    how far a row whose quotients lie near a half may move."""
    a = np.abs(x).max(axis=1, keepdims=True)
    q = np.where(a > 0, np.rint(127 * x / np.where(a > 0, a, 1)), 0.0)
    return (q @ w.astype(np.float64).T) * (a / 127) * scale + bias


def test_routed_scores():
    ex = example()
    r = ex.run(500)
    m, x = r["model"], r["x"]
    scores = x @ m["gate_w"].astype(np.int64).T + m["gate_b"]
    assert np.array_equal(r["scores"], scores)
    i = r["sample"]
    assert np.array_equal(r["proven_scores"], scores[i])
    assert r["proven_class"] == r["classes"][i, 0] == scores[i].argmax()
    assert r["proven_flag"] == int(r["margin"][i] >= r["threshold"]) and r["verified"]
    want = np.zeros((len(x), ex.ANSWER))
    for j in range(2):
        for e in range(ex.CLASSES):
            at = r["classes"][:, j] == e
            h = layer(x[at].astype(np.float64), *(a[e].astype(np.float64) for a in m["first"]))
            y = layer(np.maximum(h, 0), *(a[e].astype(np.float64) for a in m["second"]))
            want[at] += r["weights"][at, j:j + 1].astype(np.float64) * y
    # The first layer's inputs are integers up to 16: their quotients are the exact
    # ones.  Its results carry a few roundings of 2^-24, so that a hidden value
    # whose quotient lies that near to a half may be rounded the other way: one
    # step of one of the row's 127, times the largest weight of 127.
    step = np.abs(want).max() / 127
    far = np.abs(r["answers"] - want)
    assert far.max() <= step and np.median(far) <= 2.0**-20 * np.abs(want).max()
