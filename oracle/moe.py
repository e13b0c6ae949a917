"""A layer of experts and the product's epilogue in 64 bits (numpy): what the plugin's moe_route, qmatmul_experts, moe_combine and qmatmul_epi are tested against."""
import numpy as np

NONE, RELU, SILU, GELU, GELU_TANH = range(5)


def _erfc(v):
    from math import erfc
    return np.vectorize(erfc, otypes=[np.float64])(v)


def act(kind, v):
    v = np.asarray(v, np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        if kind == RELU:
            return np.where(v > 0, v, 0.0 * v if np.isnan(v).any() else 0.0)
        if kind == SILU:
            return v / (1 + np.exp(-v))
        if kind == GELU:
            return 0.5 * v * _erfc(-v / np.sqrt(2))
        if kind == GELU_TANH:
            return 0.5 * v * (1 + np.tanh(np.sqrt(2 / np.pi) * (v + 0.044715 * v ** 3)))
    return v


def sigmoid(v):
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-np.asarray(v, np.float64)))


def route(logits, k, softmax=True, renorm=True, scale=1.0, bias=None):
    """(ids, weights) of logits [T][E] as fp64."""
    v = np.asarray(logits, np.float64)
    T, E = v.shape
    key = v if bias is None else sigmoid(v) + np.asarray(bias, np.float64)
    ok = (v > -np.inf) & (key > -np.inf)
    ids, w = np.full((T, k), -1, np.int32), np.zeros((T, k))
    for t in range(T):
        best = sorted(np.flatnonzero(ok[t]), key=lambda e: (-key[t, e], e))[:k]
        ids[t, :len(best)] = best
        if not best:
            continue
        if softmax:
            top = v[t, best[0]]
            with np.errstate(invalid="ignore"):
                p = np.where(v[t] == top, 1.0, np.exp(v[t] - top))
            p[~(v[t] > -np.inf)] = 0
            total = p.sum()
        else:
            p, total = sigmoid(v[t]), 1.0
        got = p[best]
        if renorm:
            total = got.sum()
        w[t, :len(best)] = scale * got / total if total > 0 else 0
    return ids, w


def sort(ids, E):
    """(order without its unset end, pos, offsets)."""
    flat = ids.reshape(-1)
    lists = [np.flatnonzero(flat == e) for e in range(E)]
    order = np.concatenate(lists).astype(np.int32) if lists else np.zeros(0, np.int32)
    pos = np.full(flat.size, -1, np.int32)
    pos[order] = np.arange(order.size)
    return order, pos, np.concatenate([[0], np.cumsum([len(x) for x in lists])]).astype(np.int32)


def product(x, w, bias=None):
    """(sums, sums of magnitudes) of x [M][K] and w [N][K], both values."""
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    v, s = x @ w.T, np.abs(x) @ np.abs(w).T
    if bias is not None:
        v, s = v + np.asarray(bias, np.float64), s + np.abs(np.asarray(bias, np.float64))
    return v, s


U = 2.0 ** -24


def epilogue(v, s, K, kind, gated, residual=None):
    """(value, tolerance in fp32) of an activation over sums v of K products whose magnitudes sum to s.  The sum is off by no more than K + 2
    roundings of partial sums (U each of s: none exceeds it); the slopes of the activations stay below 1.2, their own error below 8 U |v| (a
    handful of roundings of values no larger than |v|; 1 + erf and 1 + tanh lose no more than U of 1)."""
    d = (K + 2) * U * s
    if gated:
        f = v.shape[-1] // 2
        g, up, dg, du = v[..., :f], v[..., f:], d[..., :f], d[..., f:]
        a = act(kind, g)
        da = 1.2 * dg + 8 * U * np.abs(g)
        r = a * up
        tol = da * (np.abs(up) + du) + np.abs(a) * du + U * np.abs(r)
    else:
        r = act(kind, v)
        tol = 1.2 * d + (8 * U * np.abs(v) if kind else 0)
    if residual is not None:
        r = r + np.asarray(residual, np.float64)
        tol = tol + U * np.abs(r)
    return r, tol
