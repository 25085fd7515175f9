"""The next token from its definition in 64 bits (test infrastructure)."""
import numpy as np


def pick(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """logits: a numpy row (float64); u: a float."""
    l = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64))
    order = np.lexsort((np.arange(len(l)), -l))  # larger first, equal ones by number
    top = l[order[0]]
    if top == -np.inf:
        return -1
    if not temperature > 0:
        return int(order[0])
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        w = np.where(l[order] == top, 1.0, np.exp((l[order] - top) / temperature))
    w[np.isnan(w)] = 0.0
    if top_k > 0:
        w[top_k:] = 0.0
    running = np.cumsum(w)
    before = np.concatenate(([0.0], running[:-1]))
    keep = w >= min_p
    if top_p < 1:
        keep &= before < top_p * running[-1]
    keep[0] = True
    w = np.where(keep, w, 0.0)
    running = np.cumsum(w)
    past = (running > u * running[-1]) & (w > 0)
    return int(order[np.argmax(past)]) if past.any() else int(order[np.flatnonzero(w)[-1]])
