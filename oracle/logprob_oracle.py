"""Log probabilities, entropy and alternatives of rows of logits in 64 bits -- TEST
INFRASTRUCTURE ONLY. numpy float64, from the definitions in include/ribn_amd.h."""
from __future__ import annotations

import numpy as np


def logprobs(logits, targets=None, top=0):
    """logits [rows][tokens]: (log probabilities of targets, entropy, top tokens, their log probabilities)."""
    x = np.asarray(logits, np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    rows, n = x.shape
    lp = np.full((rows, n), -np.inf)
    entropy = np.zeros(rows)
    for r in range(rows):
        most = x[r].max()
        if most == -np.inf:
            continue
        t = np.where(x[r] == most, 0.0, -np.inf) if most == np.inf else x[r] - most
        others = np.exp(t)
        others[int(x[r].argmax())] = 0.0
        rest = np.log1p(others.sum())  # the likeliest token's 1 aside: exact near 0
        lp[r] = t - rest
        live = t > -np.inf
        p = np.exp(lp[r][live])
        entropy[r] = rest - (p * t[live]).sum()
    given = None
    if targets is not None:
        at = np.asarray(targets, np.int64) & 0xffffffff
        given = np.array([lp[r, t] if t < n else -np.inf for r, t in enumerate(at)])
    order = np.argsort(-x, axis=1, kind="stable")[:, :top]
    return given, entropy, order, np.take_along_axis(lp, order, 1)
