"""Verification of drafted tokens in 64 bits, one sequence at a time (numpy).  Test infrastructure."""
from __future__ import annotations

import numpy as np

NONE = 0xFFFFFFFF


def probabilities(logits, temperature):
    """softmax(logits / T) in 64 bits: NaN as minus infinity, infinity as the largest number; zeros
    where nothing is left."""
    with np.errstate(invalid="ignore", over="ignore", under="ignore"):
        l = np.where(np.isnan(logits), -np.inf, np.minimum(logits, np.finfo(np.float32).max)).astype(np.float64)
        if l.max() == -np.inf:
            return np.zeros(len(l))
        e = np.exp((l - l.max()) / temperature)
        return e / e.sum()


def greedy(logits):
    l = np.where(np.isnan(logits), -np.inf, np.minimum(logits, np.finfo(np.float32).max))
    return int(l.argmax()) if l.max() > -np.inf else NONE


def drawn(weights, u):
    total = weights.cumsum()
    if not total[-1] > 0:
        return NONE
    return min(int(np.searchsorted(total, u * total[-1], side="right")), int(np.flatnonzero(weights > 0)[-1]))


def verify(logits, starts, drafts, temperature, probs=None, accept_u=None, sample_u=None, ids=None):
    """(accepted [seqs], ids [rows]); `ids` holds what rows of no sequence keep."""
    vocab, seqs = logits.shape[1], len(starts) - 1
    ids = ids.copy()
    accepted = np.zeros(seqs, np.uint32)
    for s in range(seqs):
        t0, n = int(starts[s]), int(starts[s + 1]) - int(starts[s])
        if n == 0:
            continue
        taken, token = 0, NONE
        while taken < n - 1:
            x = int(drafts[t0 + taken])
            row = logits[t0 + taken]
            if x >= vocab:
                break
            if not temperature:
                if greedy(row) != x:
                    break
            else:
                q = max(0.0, np.nan_to_num(float(probs[t0 + taken, x]))) if probs is not None else 1.0
                if not float(accept_u[t0 + taken]) * q < probabilities(row, temperature)[x]:
                    break
            taken += 1
        row = logits[t0 + taken]
        if not temperature:
            token = greedy(row)
        else:
            p = probabilities(row, temperature)
            left = p
            if taken < n - 1:
                if probs is not None:
                    left = np.maximum(p - np.maximum(np.nan_to_num(probs[t0 + taken].astype(np.float64)), 0.0), 0.0)
                elif drafts[t0 + taken] < vocab:
                    left = p.copy()
                    left[drafts[t0 + taken]] = 0.0
                if not left.sum() > 0:
                    left = p
            token = drawn(left, float(sample_u[s]))
        accepted[s] = taken
        ids[t0:t0 + n] = NONE
        ids[t0:t0 + taken] = drafts[t0:t0 + taken]
        ids[t0 + taken] = token
    return accepted, ids
