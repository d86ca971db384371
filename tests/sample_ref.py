"""Sampling by its definition, one row at a time on the CPU: weights and their
sums in numpy's long double (64 bits of mantissa), a full sort."""
import numpy as np


def draw(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, probability) of one row: logits float64 [V] as the GPU sees them."""
    x = np.asarray(logits, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    x = np.minimum(x, float(np.finfo(np.float32).max)) + 0.0
    if x.max() == -np.inf:
        return -1, 0.0
    order = np.argsort(-x, kind="stable")
    if not temperature > 0:
        return int(order[0]), 1.0
    with np.errstate(all="ignore"):
        z = (x.astype(np.longdouble) - x.max()) / np.longdouble(np.float32(temperature))
        w = np.exp(np.where(np.isnan(z), -np.inf, z))
    w[w < np.longdouble(2.0) ** -45] = 0  # (never drawn)
    kept = order[:top_k] if 0 < top_k < len(x) else order
    mass = np.cumsum(w[kept])
    if top_p < 1:
        want = np.longdouble(np.float32(top_p)) * mass[-1]
        kept = kept[np.concatenate([[True], mass[:-1] < want])]
    if min_p > 0:
        kept = kept[w[kept] >= min(float(np.float32(min_p)), 1.0)]
    mass = np.cumsum(w[kept])
    u = 0.0 if np.isnan(u) else min(max(float(np.float32(u)), 0.0), 1 - 2.0 ** -24)
    i = int(np.searchsorted(mass, np.longdouble(u) * mass[-1], side="right"))
    return int(kept[i]), float(w[kept[i]] / mass[-1])
