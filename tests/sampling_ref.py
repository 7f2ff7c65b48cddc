"""Plain restatements, on the CPU in 64 bits and more, of what ``mzoo_amd.sampling`` computes.

Tokens are whole numbers and have to be equal.  The kernels' running sums, as shares of a row's sum W, are off by less than
2^-29 (``csrc/sampling.hip`` adds up of what): 2^-44 of each weight, 2^-52 ln 2 / 20 of its distance in bins from where the row's bins are
counted from, half a unit of each bin or value, of which 2^42 and more are the largest weight, and what is below 2^-51 of
that.  ``clear`` says whether no border of a row lies within 2^-28 W of what is looked for; random inputs of a fixed seed are (a
border among N at distance 2^-28 has probability N 2^-28 at most).  Where all weights are equal, sums of them are exact on both sides.
"""

import numpy as np


def weights(logits, temperature):
    """A row's tokens in their order, and their weights."""
    x = np.asarray(logits, np.float64).copy()
    big = float(np.finfo(np.float32).max)
    x[np.isnan(x)] = -np.inf
    x[x == np.inf] = big
    x = x + 0.0
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if order.size == 0:
        return order, np.zeros(0, np.longdouble)
    t = float(np.float32(temperature))
    d = (x[order] - x[order[0]]).astype(np.longdouble)
    with np.errstate(over="ignore", invalid="ignore"):
        w = np.exp(d / np.longdouble(t)) if 0 < t < np.inf else np.ones(order.size, np.longdouble)
    if not t > 0:
        return order, np.concatenate([[1.0], np.zeros(order.size - 1)]).astype(np.longdouble)
    return order, w


def kept(logits, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(the kept tokens in their order, their weights, whether no border is near)."""
    order, w = weights(logits, temperature)
    clear = True
    if order.size == 0:
        return order, w, clear
    n = order.size
    if not float(np.float32(temperature)) > 0:
        return order[:1], w[:1], clear
    if 0 < top_k < n:
        n = int(top_k)
    p = float(np.float32(top_p))
    if p < 1:
        sums = np.cumsum(w[:n])
        x = np.longdouble(max(p, 0.0)) * sums[-1]
        m = int((sums < x).sum()) + 1
        equal = bool((w[:n] == w[0]).all())
        clear &= equal or p <= 0 or float(np.abs(sums[:-1] - x).min(initial=1.0)) > 2.0 ** -28 * float(sums[-1])
        n = min(n, m)
    f = float(np.float32(min_p))
    if f > 0:
        # in logarithms: a weight of 1 - 1e-42 is not 1
        x = np.asarray(logits, np.float64)[order]
        top = float(np.finfo(np.float32).max)
        d = (np.minimum(x, top) - min(x[0], top)).astype(np.longdouble) / np.longdouble(float(np.float32(temperature)))
        edge = np.log(np.longdouble(min(f, 1.0)))
        m = int((d[:n] >= edge).sum())
        clear &= f >= 1 or float(np.abs(d - edge).min()) > 2.0 ** -45
        n = max(1, min(n, m))
    return order[:n], w[:n], clear


def pick(order, w, u):
    """(the token at u of the running sum, whether no border is near)."""
    if order.size == 0:
        return -1, True
    sums = np.cumsum(w)
    u = float(u)
    u = 0.0 if not u > 0 else min(u, 1 - 2.0 ** -24)
    x = np.longdouble(u) * sums[-1]
    some = np.flatnonzero(w > 0)
    at = min(int((sums <= x).sum()), int(some[-1]))
    equal = bool((w[some] == w[0]).all())
    near = float(np.abs(sums[:-1] - x).min(initial=1.0)) <= 2.0 ** -28 * float(sums[-1])
    # a sum that is not reached by rounding alone: u 0 is before every border
    return int(order[at]), equal or u == 0.0 or not near


def sample(logits, u, **filters):
    """(token, log probability, clear)."""
    order, w, clear = kept(logits, **filters)
    token, sure = pick(order, w, u)
    if token < 0:
        return -1, -np.inf, True
    at = int(np.flatnonzero(order == token)[0])
    return token, float(np.log(w[at] / w.sum())), clear and sure


def verify(logits, tokens, u, draw, probs=None, **filters):
    """One sequence: rows of logits, the tokens that they follow.  (accepted, next, clear)."""
    n = len(tokens)
    if n == 0:
        return 0, -1, True
    clear = True
    v = logits.shape[1]
    for i in range(n):
        f = {k: x[i] if isinstance(x, (list, np.ndarray)) else x for k, x in filters.items()}
        order, w, sure = kept(logits[i], **f)
        clear &= sure
        if i == n - 1:
            break
        d = int(tokens[i + 1])
        p = np.zeros(v, np.longdouble)
        if order.size:
            p[order] = w / w.sum()
        pd = p[d] if 0 <= d < v else np.longdouble(0)
        q = 1.0 if probs is None else float(probs[i][d]) if 0 <= d < v else 1.0
        a = np.longdouble(float(np.float32(u[i]))) * np.longdouble(q)
        if pd > 0 and float(abs(a - pd)) <= 2.0 ** -28 and not (pd == 1 and q == 1):
            clear = False
        if a < pd:
            continue
        if probs is None:
            if 0 <= d < v and pd < 1:
                w = w[order != d]
                order = order[order != d]
        else:
            left = np.maximum(p - np.maximum(np.nan_to_num(np.asarray(probs[i], np.float64), nan=0.0), 0.0).astype(np.longdouble), 0)
            if left.sum() > 0:
                order, w = np.arange(v), left
        break
    token, sure = pick(order, w, draw)
    return i, token, clear and sure


def beams(logits, scores, width, keep):
    """(parents, tokens, scores float64) of all groups."""
    rows, v = logits.shape
    out = []
    for g in range(rows // width):
        cand = []
        for r in range(g * width, (g + 1) * width):
            if not scores[r] > -np.inf:
                continue
            order, w = weights(logits[r], 1.0)
            if order.size == 0:
                continue
            x = np.asarray(logits[r], np.float64)
            x = np.minimum(x[order], float(np.finfo(np.float32).max))
            val = (np.longdouble(float(scores[r])) + (x - x[0]).astype(np.longdouble) - np.log(w.sum()))[:keep]
            cand += [(-float(val[j]), -val[j], r, int(order[j])) for j in range(len(val))]
        cand.sort(key=lambda c: (c[1], c[2], c[3]))
        cand = cand[:keep] + [(np.inf, 0, -1, -1)] * (keep - min(keep, len(cand)))
        out += [(c[2], c[3], -c[0]) for c in cand]
    a = list(zip(*out))
    return np.array(a[0]), np.array(a[1]), np.array(a[2])
