"""Float64 restatement of sampling and of speculative sampling (test infrastructure only, see oracle/__init__.py): one
row at a time, in plain numpy, as include/nvattn.h states the rules."""
import numpy as np


def kept_weights(logits, t, top_k=0, top_p=1.0, min_p=0.0):
    """The weights of one row [V] after every setting (t > 0), float64."""
    x = np.asarray(logits, dtype=np.float64).copy()
    x[np.isnan(x)] = -np.inf
    m = x.max()
    with np.errstate(over="ignore", invalid="ignore"):
        w = np.where(x == m, 1.0, np.exp((x - m) / np.float64(np.float32(t))))
    w[np.isnan(w)] = 0.0
    if min_p > 0:
        w[w < min(np.float64(np.float32(min_p)), 1.0)] = 0.0
    order = np.argsort(-x, kind="stable")
    if 0 < top_k < len(x):
        w[order[top_k:]] = 0.0
    if top_p < 1:
        s = w[order]
        before = np.concatenate([[0.0], np.cumsum(s)[:-1]])
        gone = before >= np.float64(np.float32(top_p)) * s.sum()
        gone[0] = False
        w[order[gone]] = 0.0
    return w


def argmax(logits):
    x = np.asarray(logits, dtype=np.float64)
    nan = np.flatnonzero(np.isnan(x))
    return int(nan[0]) if len(nan) else int(np.argmax(x))


def draw(w, u):
    """(index, distance of u * sum from the nearest running sum, over the sum)."""
    c = np.cumsum(w)
    at = u * c[-1]
    i = int(np.searchsorted(c, at, side="right"))
    return min(i, int(np.flatnonzero(w)[-1])), float(np.abs(c - at).min() / c[-1])


def sample(logits, t, u, top_k=0, top_p=1.0, min_p=0.0):
    """(token, margin): the margin says how near another token was."""
    if not t > 0:
        return argmax(logits), 1.0
    return draw(kept_weights(logits, t, top_k, top_p, min_p), u)


def verify(logits, drafts, num_drafts, t, accept_u, u, top_k=0, top_p=1.0, min_p=0.0):
    """One sequence: logits [K + 1, V], drafts [K] -> (accepted, next token)."""
    K, V = len(drafts), logits.shape[1]
    for j in range(K + 1):
        d = int(drafts[j]) if j < K and j < num_drafts else -1
        if not t > 0:
            best = argmax(logits[j])
            if d < 0 or d != best:
                return j, best
            continue
        w = kept_weights(logits[j], t, top_k, top_p, min_p)
        wd = w[d] if 0 <= d < V else 0.0
        if d >= 0 and accept_u[j] * w.sum() < wd:
            continue
        if 0 <= d < V:
            w[d] = 0.0
        return j, draw(w, u)[0]
