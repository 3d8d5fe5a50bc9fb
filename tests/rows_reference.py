"""Plain 64-bit implementations of the row operators, one row at a time (numpy)."""

import numpy as np


def in_order(v):
    """Columns of a row in top-k order: larger first, equal ones (-0 == +0) by lower column."""
    return np.lexsort((np.arange(len(v)), -(v + 0.0)))


def sample_row(x, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(ids, probabilities, kept) of one row of float64 scores."""
    valid = np.flatnonzero(x > -np.inf)
    n = len(uniforms)
    if len(valid) == 0:
        return np.full(n, -1, np.int64), np.zeros(n), 0
    walk = valid[in_order(x[valid])]
    best = x[walk[0]]
    if not temperature > 0:
        return np.full(n, walk[0], np.int64), np.ones(n), 1
    with np.errstate(all="ignore"):
        d = np.where(x[walk] == best, 0.0, x[walk] - best)
        w = np.where(d == 0, 1.0, np.exp(d / temperature))
    w = np.where(np.isnan(w), 0.0, w)  # +inf beside finite scores at an infinite temperature
    # The contract's resolution: multiples of 2^-frac of the row's largest. It shows where u is 0
    # and the temperature small: exp(-7 / 1e-3) is no weight to draw, though above 0 in 64 bits.
    frac = min(50, 62 - int(np.ceil(np.log2(len(x)))))
    w = np.rint(w * 2.0 ** frac) / 2.0 ** frac
    end = len(walk)
    if 0 < top_k < end:
        end = int(top_k)
    sums = np.cumsum(w)
    if top_p < 1:
        want = max(float(top_p), 0.0) * sums[end - 1]
        end = min(end, int(np.searchsorted(sums[:end], want, side="left")) + 1)
    if min_p > 0:
        with np.errstate(all="ignore"):
            edge = best + temperature * np.log(min(float(min_p), 1.0))
        if not np.isnan(edge):
            end = min(end, int(np.count_nonzero(x[valid] >= edge)))
    keep = np.zeros(len(x))
    keep[walk[:end]] = w[:end]
    run = np.cumsum(keep)
    u = np.where(uniforms > 0, np.minimum(uniforms, np.float32(1 - 2.0 ** -24)), 0.0)
    ids = np.searchsorted(run, u.astype(np.float64) * run[-1], side="right")
    return ids.astype(np.int64), keep[ids] / run[-1], end


def sample(x, uniforms, temperature=None, top_k=None, top_p=None, min_p=None):
    x = np.asarray(x, np.float64)
    rows = len(x)
    temperature = np.ones(rows) if temperature is None else np.asarray(temperature, np.float64)
    top_k = np.zeros(rows, int) if top_k is None else top_k
    top_p = np.ones(rows) if top_p is None else np.asarray(top_p, np.float64)
    min_p = np.zeros(rows) if min_p is None else np.asarray(min_p, np.float64)
    got = [sample_row(x[r], uniforms[r], temperature[r], top_k[r], top_p[r], min_p[r])
           for r in range(rows)]
    return (np.stack([g[0] for g in got]), np.stack([g[1] for g in got]),
            np.array([g[2] for g in got], np.int32))


def scores_row(x, score):
    valid = x > -np.inf
    if not valid.any():
        return np.zeros(len(x))
    with np.errstate(all="ignore"):
        if score == "sigmoid":
            s = 1.0 / (1.0 + np.exp(-x))
        else:
            best = x[valid].max()
            s = np.where(x == best, 1.0, np.exp(np.where(valid, x, 0.0) - best))
            s = s / s[valid].sum()
    return np.where(valid, s, 0.0)


def ratio_row(x, ids, score):
    """Chosen scores over their sum, from exponentials relative to the largest of them."""
    v = x[ids]
    top = v.max()
    with np.errstate(all="ignore"):
        if score == "sigmoid":
            base = min(top, 0.0)
            r = 1.0 / (np.exp(base) + np.where(v == base, 1.0, np.exp(base - v)))
        else:
            r = np.where(v == top, 1.0, np.exp(v - top))
    return r / r.sum()


def route_row(x, k, bias=None, score="softmax", groups=1, topk_groups=1, group_rule="max",
              renormalize=True, scale=1.0):
    """(ids, weights, scores) of one token's float64 logits."""
    n = len(x)
    s = scores_row(x, score)
    choice = x.copy() if bias is None else s + bias
    choice = np.where((x > -np.inf) & (choice > -np.inf), choice, -np.inf)
    if groups > 1:
        value = np.full(groups, -np.inf)
        for g in range(groups):
            at = np.arange(g * (n // groups), (g + 1) * (n // groups))
            at = at[choice[at] > -np.inf]
            if len(at) == 0:
                continue
            if group_rule == "max":
                value[g] = choice[at].max()
            else:
                best = np.sort(s[at] if bias is None else choice[at])[::-1][:2]
                value[g] = best.sum()
        stands = np.zeros(groups, bool)
        stands[in_order(value)[:topk_groups]] = True
        choice = np.where(np.repeat(stands, n // groups), choice, -np.inf)
    walk = in_order(choice)
    ids = walk[choice[walk] > -np.inf][:k]
    w = np.zeros(k)
    if len(ids):
        w[: len(ids)] = ratio_row(x, ids, score) if renormalize else s[ids]
    return np.concatenate([ids, np.full(k - len(ids), -1)]).astype(np.int32), w * scale, s


def route(x, k, **how):
    got = [route_row(row, k, **how) for row in np.asarray(x, np.float64)]
    return tuple(np.stack([g[i] for g in got]) for i in range(3))


def route_backward_row(x, ids, dweights, score="softmax", renormalize=True, scale=1.0,
                       dscores=None):
    """(gradient, sum of the magnitudes that were added up for it) of one token's logits."""
    n = len(x)
    valid = x > -np.inf
    s = scores_row(x, score)
    dw = np.where((ids >= 0) & (ids < n), dweights, 0.0) * scale
    live = np.array([0 <= i < n and valid[i] for i in ids], bool)
    ids, dw = ids[live], dw[live]
    d = np.zeros(n) if dscores is None else np.where(valid, dscores, 0.0)
    slope = s * (1 - s) if score == "sigmoid" else s
    grad, size = d * slope, np.abs(d) * slope
    if score == "softmax":
        grad = grad - s * (d * s).sum()
        size = size + s * (np.abs(d) * s).sum()
    if len(ids):
        if renormalize:
            r = ratio_row(x, ids, score)
            own = r * (dw - (r * dw).sum())
            mag = r * (np.abs(dw) + (r * np.abs(dw)).sum())
        else:
            own, mag = s[ids] * dw, s[ids] * np.abs(dw)
        if score == "sigmoid":
            own, mag = own * (1 - s[ids]), mag * (1 - s[ids])
        elif not renormalize:
            grad = grad - s * own.sum()
            size = size + s * mag.sum()
        np.add.at(grad, ids, own)
        np.add.at(size, ids, mag)
    return np.where(valid, grad, 0.0), np.where(valid, size, 0.0)


def route_backward(x, ids, dweights, dscores=None, **how):
    got = [route_backward_row(row, ids[t], dweights[t].astype(np.float64),
                              dscores=None if dscores is None else dscores[t].astype(np.float64),
                              **how)
           for t, row in enumerate(np.asarray(x, np.float64))]
    return np.stack([g[0] for g in got]), np.stack([g[1] for g in got])


def plan(ids, experts, align, capacity):
    """(offsets, order, position) of the flat ids."""
    ids = np.asarray(ids).reshape(-1)
    offsets = np.zeros(experts + 1, np.int32)
    order = np.full(capacity, -1, np.int32)
    position = np.full(len(ids), -1, np.int32)
    for e in range(experts):
        pairs = np.flatnonzero(ids == e)
        offsets[e + 1] = offsets[e] + -(-len(pairs) // align) * align
        order[offsets[e]: offsets[e] + len(pairs)] = pairs
        position[pairs] = offsets[e] + np.arange(len(pairs))
    return offsets, order, position
