"""The experts' router in 64 bits: routes, weights, balance, gradients, and how far
results in 32 bits may be from them.

With a = scale (s - max s), a probability exp(a) / Z carries two roundings of a
(each 2^-24 |a| relative to the result), the exponential's and the division's few,
and those of Z: a sum of `experts` terms whose own errors are weighted by p.  R is
that bound, relative to p; results made of probabilities carry it with the size of
their terms.  Below 2^-126 a value may be rounded to a step of 2^-149 or to zero.
"""
import numpy as np

FEW = 16  # roundings of exponentials, divisions and products on the way to a result


def softmax(s, scale):
    """(p, R): probabilities of the scores (masked: -inf) and their bounds."""
    m = s.max(axis=1, keepdims=True)
    with np.errstate(invalid="ignore"):
        a = np.where(np.isfinite(s), (s - m) * scale, -np.inf)
    e = np.where(np.isfinite(a), np.exp(a), 0.0)
    total = e.sum(axis=1, keepdims=True)
    p = np.divide(e, total, out=np.zeros_like(e), where=total > 0)
    size = np.where(np.isfinite(a), np.abs(a), 0.0)
    R = 2.0**-24 * (3 * size + 3 * (p * size).sum(axis=1, keepdims=True) + s.shape[1] + FEW)
    return p, R


def chosen(s, slots):
    """Experts by falling score, the lower first among equals, -1 where none is left."""
    order = np.argsort(-s, axis=1, kind="stable")
    order = np.pad(order, ((0, 0), (0, max(0, slots - s.shape[1]))))[:, :slots]
    left = np.arange(slots) < np.minimum((s > -np.inf).sum(axis=1), s.shape[1])[:, None]
    return np.where(left, order, -1)


def weights(s, scale, expert, renormalize):
    """(w, bound) of the chosen experts."""
    p, R = softmax(s, scale)
    i, on = np.maximum(expert, 0), expert >= 0
    w = np.where(on, np.take_along_axis(p, i, 1), 0.0)
    r = np.take_along_axis(R, i, 1)
    if renormalize:
        # a softmax over the chosen alone; its own maximum and sum
        own = np.where(on, np.take_along_axis(s, i, 1), -np.inf)
        w, r = softmax(own, scale)
    return w, w * r + 2.0**-126


def balance(s, scale, expert):
    """(count with n, prob, loss), bounds of prob and loss, for rows without NaN."""
    experts, slots = s.shape[1], expert.shape[1]
    p, R = softmax(s, scale)
    n = int((s > -np.inf).any(axis=1).sum())
    count = np.array([(expert == e).sum() for e in range(experts)] + [n])
    prob = p.sum(axis=0) / max(n, 1)
    # a lane adds its tokens one after the other
    lim = (p * R).sum(axis=0) / max(n, 1) + (n + FEW) * 2.0**-24 * prob + 2.0**-126
    f = count[:-1] / max(1, n * slots)
    loss = experts * (f * prob).sum()
    return count, prob, loss, lim, experts * (f * lim).sum() + 2.0**-22 * loss


def gradient(s, scale, expert, renormalize, gw=None, count=None, gl=None):
    """(ds, bound), rows without NaN; count as balance gives it."""
    tokens, experts = s.shape
    p, R = softmax(s, scale)
    dz, lim = np.zeros_like(p), np.zeros_like(p)
    if count is not None and count[-1] > 0:
        f = count[:-1] / (count[-1] * expert.shape[1])
        c = gl * experts / count[-1]
        dot = (p * f).sum(axis=1, keepdims=True)
        dz += c * p * (f - dot)
        dot_lim = (p * f * R).sum(axis=1, keepdims=True) + experts * 2.0**-24 * dot
        lim += abs(c) * p * ((R + FEW * 2.0**-24) * (f + dot) + dot_lim)
    if gw is not None:
        on = (expert >= 0) & (expert < experts)
        g, times = np.zeros_like(p), np.zeros_like(p)
        size = np.zeros_like(p)
        for j in range(expert.shape[1]):
            at = np.nonzero(on[:, j])[0]
            e = expert[at, j]
            g[at, e] += gw[at, j]
            size[at, e] += np.abs(gw[at, j])
            times[at, e] += 1
        w, r = p, R
        if renormalize:
            own, r = softmax(np.where(times > 0, s, -np.inf), scale)
            total = (times * own).sum(axis=1, keepdims=True)
            w = np.divide(own, total, out=np.zeros_like(own), where=total > 0)
            # the sum counts an expert as often as it is named
            r = r + (w * times * r).sum(axis=1, keepdims=True) + expert.shape[1] * 2.0**-24
        else:
            times = np.ones_like(p)
        mean = (w * g).sum(axis=1, keepdims=True)
        spread = (w * size).sum(axis=1, keepdims=True)
        mean_lim = (w * size * r).sum(axis=1, keepdims=True) + (experts + expert.shape[1]) * 2.0**-24 * spread
        dz += w * (g - times * mean)
        lim += w * ((r + (FEW + expert.shape[1]) * 2.0**-24) * (size + times * spread) + times * mean_lim)
    return scale * dz, scale * (lim + 2.0**-120)
