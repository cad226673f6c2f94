"""Routing of rows to experts in 64 bits: the choice, the weights and their gradient."""
from __future__ import annotations

import numpy as np


def scores(logits, scoring):
    l = np.asarray(logits, dtype=np.float64)
    with np.errstate(all="ignore"):
        if scoring == "sigmoid":
            return 1.0 / (1.0 + np.exp(-l))
        top = np.nanmax(np.where(np.isnan(l), -np.inf, l), axis=1, keepdims=True)
        e = np.where(np.isneginf(top), 0.0, np.exp(l - np.where(np.isfinite(top), top, 0.0)))
        e = np.where(np.isposinf(top), np.isposinf(l), np.where(np.isnan(l), 0.0, e))
        return e / np.maximum(e.sum(1, keepdims=True), 1e-300)


def choose(logits, k, scoring, bias=None, groups=1, kept=1, padded=None):
    """ids [M, k]: E where nothing is left."""
    l = np.asarray(logits, dtype=np.float64)
    m, e = l.shape
    s = scores(l, scoring)
    b = np.zeros(e) if bias is None else np.asarray(bias, dtype=np.float64)
    with np.errstate(all="ignore"):
        c = s + b
    c[~(l > -np.inf) | ~(b > -np.inf)] = -np.inf
    ids = np.full((m, k), e)
    for r in range(m):
        if padded is not None and padded[r]:
            continue
        row = c[r]
        if kept < groups:
            best = np.sort(row.reshape(groups, -1), axis=1)[:, ::-1]
            total = best[:, 0] + (0.0 if best.shape[1] == 1 else np.where(np.isneginf(best[:, 1]), 0.0, best[:, 1]))
            out = np.argsort(-total, kind="stable")[kept:]
            row = row.copy()
            row.reshape(groups, -1)[out] = -np.inf
        rank = l[r] if bias is None else row  # without a bias the scores grow with the logits (and may saturate)
        order = [i for i in np.argsort(-np.where(np.isnan(rank), -np.inf, rank), kind="stable") if row[i] > -np.inf]
        ids[r, :min(k, len(order))] = order[:k]
    return ids


def weights(logits, ids, scoring, renormalize, scale):
    """Of the chosen experts, relative to the largest where they are renormalized (so that small ones keep their ratio)."""
    l = np.asarray(logits, dtype=np.float64)
    m, e = l.shape
    real = ids < e
    at = np.where(real, ids, 0)
    mine = np.where(real, np.take_along_axis(l, at, 1), -np.inf)
    with np.errstate(all="ignore"):
        if renormalize:
            top = np.where(real.any(1, keepdims=True), mine.max(1, keepdims=True), 0.0)
            w = np.exp(mine - top)
            if scoring == "sigmoid":
                w = np.where(top < 0, w / (1 + np.exp(mine)), 1 / (1 + np.exp(-mine)))
            w = np.where(real, w, 0.0)
            w = np.where(real, w / w.sum(1, keepdims=True), 0.0)
        else:
            w = np.where(real, np.take_along_axis(scores(l, scoring), at, 1), 0.0)
    return w * scale


def grad(dweights, logits, ids, scoring, renormalize, scale):
    l = np.asarray(logits, dtype=np.float64)
    m, e = l.shape
    out = np.zeros((m, e))
    for r in range(m):
        slots = [j for j in range(ids.shape[1]) if 0 <= ids[r, j] < e]
        if not slots:
            continue
        at = ids[r, slots]
        dw = np.asarray(dweights, dtype=np.float64)[r, slots] * scale
        if renormalize:
            w = weights(l[r:r + 1], at[None], scoring, True, 1.0)[0]
            g = w * (dw - (dw * w).sum())
            if scoring == "sigmoid":
                g = g / (1 + np.exp(l[r, at]))
            np.add.at(out[r], at, g)
        elif scoring == "sigmoid":
            s = 1 / (1 + np.exp(-l[r, at]))
            np.add.at(out[r], at, dw * s * (1 - s))
        else:
            s = scores(l[r:r + 1], scoring)[0]
            np.add.at(out[r], at, dw * s[at])
            out[r] -= s * (dw * s[at]).sum()
    return out
