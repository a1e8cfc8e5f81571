"""Norms, 8-bit rows, products and the draw of a token -- TEST INFRASTRUCTURE ONLY.

Plain restatements in float64 of ``flashnext_b200.dense`` and
``flashnext_b200.sampling``.  The reference leaves these steps to mlx, so there
is no file of its own to follow; the formulas are the definitions.
"""
from __future__ import annotations

import math

import numpy as np

TINY = 2.0 ** -100
TOP = {"int8": 127.0, "e4m3": 448.0}


def add_rms_norm(x, weight, residual=None, eps=1e-6, unit_offset=False):
    """(y, s) of rows in float64."""
    s = x.astype(np.float64) if residual is None else x.astype(np.float64) + residual.astype(np.float64)
    w = weight.astype(np.float64) + (1.0 if unit_offset else 0.0)
    with np.errstate(invalid="ignore", divide="ignore"):
        return s / np.sqrt((s * s).mean(1, keepdims=True) + eps) * w, s


def row_scales(y, kind):
    return np.maximum(np.abs(y).max(1), TINY) / TOP[kind]


def linear(x, weight, bias=None, act=None, residual=None, x_scale=None, weight_scale=None):
    """(out, magnitude) in float64; magnitude is the sum of the products' magnitudes before the activation."""
    x, w = x.astype(np.float64), weight.astype(np.float64)
    a = x @ w.T  # codes: whole numbers, exact
    magnitude = np.abs(x) @ np.abs(w).T
    if x_scale is not None:
        both = x_scale.astype(np.float64)[:, None] * weight_scale.astype(np.float64)
        a, magnitude = a * both, magnitude * both
    if bias is not None:
        a = a + bias.astype(np.float64)
    if act == "silu":
        a = a / (1.0 + np.exp(-np.clip(a, -700, None)))
    elif act == "gelu":
        a = a * 0.5 * np.vectorize(math.erfc)(-a / math.sqrt(2.0))
    elif act == "relu":
        a = np.maximum(a, 0.0)
    return (a if residual is None else a + residual.astype(np.float64)), magnitude


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log-probability) of one row, in float64; settings are float32 values."""
    z = [float(v) for v in logits]
    live = [i for i, v in enumerate(z) if v > -math.inf]
    if not live:
        return -1, 0.0
    top = max(z[i] for i in live)
    if not temperature > 0 or top_k == 1 or not top_p > 0:
        return next(i for i in live if z[i] == top), 0.0
    x = {i: 0.0 if z[i] == top else (z[i] - top) / float(temperature) for i in live}
    w = {i: math.exp(x[i]) if x[i] > -745 else 0.0 for i in live}
    ranked = sorted(live, key=lambda i: (-z[i], i))
    if 0 < top_k:
        ranked = ranked[:top_k]
    if top_p < 1:
        total, before, kept = math.fsum(w[i] for i in ranked), 0.0, []
        for i in ranked:
            if kept and not before < top_p * total:
                break
            kept.append(i)
            before += w[i]
        ranked = kept
    if min_p > 0:
        ranked = [i for i in ranked if w[i] >= min(min_p, 1.0)]
    kept = sorted(ranked)
    total = math.fsum(w[i] for i in kept)
    want, upto, token = (u if u > 0 else 0.0) * total, 0.0, None
    for i in kept:
        if w[i] > 0:
            token = i
        upto += w[i]
        if upto > want:
            break
    return token, x[token] - math.log(total)
