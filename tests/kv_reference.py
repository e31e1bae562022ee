"""Plain restatements in 64 bits of the paged cache's attention and of the expert router, for the GPU tests."""

import numpy as np

F64 = np.float64


def softmax_attention(q, k, v, scale):
    """q [D], k, v [n, D] -> (out [D], the largest error a float32 evaluation may have [D])."""
    D, n = q.shape[0], k.shape[0]
    q, k, v = q.astype(F64), k.astype(F64), v.astype(F64)
    s = (k @ q) * scale
    w = np.exp(s - s.max())
    w /= w.sum()
    out = w @ v
    # q enters with 22 bits, a score is a chain of D / 16 accumulations rounded to float32 (each at most one unit, 2^-23, of
    # what the sum's magnitudes come to) and three roundings more: an error of delta in every score changes a weight by at
    # most exp(2 delta) - 1. The exponential, the weight's 22 bits and the division add some 2^-22 each (2^-20 for all), and
    # the running sums one rounding per 16 positions and for each of the up to 32 partial results that are joined.
    delta = abs(scale) * (np.abs(k) @ np.abs(q)).max() * (D / 16 + 4) * 2.0 ** -23
    size = w @ np.abs(v)
    return out, size * (np.expm1(2 * delta) + 2.0 ** -20 + (n / 16 + 32) * 2.0 ** -24)


def attention(q, keys, values, lens, scale):
    """q [S][n][H][D]; keys, values: per sequence [len][Hkv][D]. Returns out and its bound, both [S][n][H][D]."""
    S, n, H, D = q.shape
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for s in range(S):
        group = H // max(1, keys[s].shape[1])
        for r in range(n):
            seen = lens[s] - n + r + 1
            if seen <= 0:
                continue
            for h in range(H):
                out[s, r, h], tol[s, r, h] = softmax_attention(q[s, r, h], keys[s][:seen, h // group], values[s][:seen, h // group], scale)
    return out, tol


def route(logits, top_k, bias=None, score="softmax", n_group=1, topk_group=1, group_top=1, renorm=True, scale=1.0):
    """Row by row: ids int32 and w in 64 bits."""
    T, E = logits.shape
    ids, w = np.zeros((T, top_k), np.int32), np.zeros((T, top_k))
    for t in range(T):
        x = logits[t].astype(F64).copy()
        x[np.isnan(x)] = -np.inf
        with np.errstate(over="ignore", invalid="ignore"):
            if score == "sigmoid":
                p = np.where(x == -np.inf, 0.0, 1.0 / (1.0 + np.exp(-x)))
            else:
                e = np.where(x == -np.inf, 0.0, np.where(x == x.max(), 1.0, np.exp(x - x.max())))
                p = e / e.sum() if e.sum() > 0 else e
        c = x if bias is None and n_group == 1 else p + (bias.astype(F64) if bias is not None else 0.0)
        c = np.where(np.isnan(c), -np.inf, c)
        left = list(range(E))
        if n_group > 1:
            size = E // n_group
            best = [np.sort(c[g * size:(g + 1) * size])[::-1][:group_top].sum() for g in range(n_group)]
            kept = sorted(range(n_group), key=lambda g: (-best[g], g))[:topk_group]
            left = [e for e in left if e // size in kept]
        ids[t] = sorted(left, key=lambda e: (-c[e], e))[:top_k]
        w[t] = p[ids[t]]
        if renorm:
            w[t] = w[t] / w[t].sum() if w[t].sum() > 0 else 0.0
    return ids, w * scale
