"""Test infrastructure: draws from exponentiated returns and gradient clipping restated in numpy, in 64 bits, from their
definitions (one row, one sample after the other's weight; nothing shared with the kernels)."""
import numpy as np


def kept_weights(R, kappa=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Weight of every sample of one row, zero where a filter drops it."""
    R = np.asarray(R, dtype=np.float64)
    out = np.zeros(len(R))
    fine = np.flatnonzero(np.isfinite(R))
    if not len(fine) or not (0.0 <= kappa < np.inf):
        return out
    order = fine[np.lexsort((fine, -R[fine]))]
    best = R[order[0]]
    if top_k > 0:
        order = order[:top_k]
    with np.errstate(over="ignore", under="ignore"):
        w = np.exp(-kappa * (best - R[order])) if kappa > 0.0 else np.ones(len(order))
    upto = np.cumsum(w, dtype=np.longdouble)
    before = np.concatenate(([0.0], upto[:-1]))
    keep = (before < np.longdouble(np.float64(top_p) * np.float64(upto[-1]))) & (w >= min_p)
    if top_p >= 1.0:
        keep = w >= min_p
    out[order[keep]] = w[keep]
    return out


def draw(R, u, kappa=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(index, weight) of the draws u from one row."""
    w = kept_weights(R, kappa, top_k, top_p, min_p)
    u = np.asarray(u, dtype=np.float64)
    if not w.any():
        return np.full(u.shape, -1, dtype=np.int64), np.zeros(u.shape)
    upto = np.cumsum(w, dtype=np.longdouble)
    last = int(np.flatnonzero(w)[-1])
    u = np.clip(np.nan_to_num(u, nan=0.0), 0.0, 1.0)
    index = np.minimum(np.searchsorted(upto, u * upto[-1], side="right"), last)
    return index.astype(np.int64), w[index] / np.float64(upto[-1])


def norm(grads, kind="l2"):
    grads = [np.asarray(g, dtype=np.float64).ravel() for g in grads]
    if kind == "max":
        return max([0.0] + [np.abs(g).max() if g.size else 0.0 for g in grads])
    return float(np.sqrt(sum(np.dot(g, g) for g in grads)))


def clip(grads, max_norm, kind="l2"):
    """(norm before, clipped gradients in 64 bits)."""
    total = norm(grads, kind)
    s = max_norm / total if np.isfinite(total) and total > max_norm else 1.0
    return total, [np.asarray(g, dtype=np.float64) * s if s != 1.0 else np.asarray(g, dtype=np.float64) for g in grads]
