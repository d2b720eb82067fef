"""Token sampling in float64, one row at a time (numpy; what the CUDA kernel is compared with)."""

from __future__ import annotations

import numpy as np


def kept(logits, temperature, top_k, top_p, min_p):
    """Masses of the tokens that a draw can give (zeros elsewhere), or None where there are none."""
    x = np.asarray(logits, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    top = x.max()
    if top == -np.inf:
        return None
    order = np.argsort(-x, kind="stable")  # by logit, ties by index
    mass = np.zeros_like(x)
    if not temperature > 0 or top_k == 1 or not top_p > 0 or not min_p <= 1:
        mass[order[0]] = 1.0
        return mass
    with np.errstate(invalid="ignore"):
        all_mass = np.where(x == top, 1.0, np.exp((x - top) / temperature))
    ranked = all_mass[order]
    if top_k > 0:
        ranked = ranked[:top_k]
    if top_p < 1:
        before = np.cumsum(ranked) - ranked
        ranked = ranked[:max(1, int((before < top_p * ranked.sum()).sum()))]
    stays = ranked >= min_p
    stays[0] = True
    mass[order[:len(ranked)][stays]] = ranked[stays]
    return mass


def draw(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """-> (token, how far the running mass is from the draw's border, relative to the whole)."""
    mass = kept(logits, temperature, top_k, top_p, min_p)
    if mass is None:
        return -1, 1.0
    run = np.cumsum(mass)
    target = float(u) * run[-1]
    token = int(np.argmax(run > target)) if (run > target).any() else int(np.nonzero(mass)[0][-1])
    return token, float(np.min(np.abs(run[mass > 0] - target)) / run[-1])
