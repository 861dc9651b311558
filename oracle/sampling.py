"""The sampler restated on the CPU in float64, one row at a time.

The reference's sampler (nanoserve/sampler.py:24-77) divides by the
temperature, keeps the top k, then the smallest prefix of the sorted
probabilities that reaches top_p, and draws once; min-p and a given uniform
number in the draw's place are the product's own.
"""

from __future__ import annotations

import numpy as np


def sample_row(z, u, temperature, top_k=0, top_p=1.0, min_p=0.0) -> int:
    z = np.asarray(z, dtype=np.float64)
    nan = np.flatnonzero(np.isnan(z))
    if nan.size:
        return int(nan[0])
    top = z.max()
    if not temperature > 0 or not np.isfinite(top):
        return int(np.argmax(z))
    order = np.argsort(-z, kind="stable")
    with np.errstate(invalid="ignore"):
        a = (z[order] - top) / np.float64(temperature)
    w = np.where(np.isneginf(z[order]), 0.0, np.exp(a))
    n = int(top_k) if 0 < top_k < z.size else z.size
    before = np.concatenate(([0.0], np.cumsum(w)))
    keep = np.arange(z.size) < n
    if top_p < 1:
        keep &= before[:-1] < np.float64(top_p) * before[n]
    if min_p > 0:
        keep &= w >= np.float64(min_p)
    keep[0] = True
    n = int(keep.sum())  # every filter keeps a prefix
    r = int(np.searchsorted(before[1:n + 1], max(np.float64(u), 0.0) * before[n], side="right"))
    return int(order[min(r, n - 1)])


def sample_ref(logits, uniform, temperature, top_k=None, top_p=None, min_p=None) -> list[int]:
    """Row by row; settings are sequences or None."""
    pick = lambda v, i, off: off if v is None else float(v[i])  # noqa: E731
    return [sample_row(z, float(uniform[i]), float(temperature[i]), int(pick(top_k, i, 0)), pick(top_p, i, 1.0),
                       pick(min_p, i, 0.0)) for i, z in enumerate(np.asarray(logits, dtype=np.float64))]
