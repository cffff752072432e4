"""General expert router and its gradient in numpy -- TEST INFRASTRUCTURE ONLY.

  s = sigmoid(x) or softmax(x)   exponentials in float64, rounded to fp32 (the sigmoid's add and divide are fp32)
  v = s + bias                   fp32
  group score = the sum (fp32) of the group's one or two largest v; a closed second place adds nothing
  picks = the top_k largest v of the best groups, ties to the lower index, listed ascending

Experts whose logit or v is -inf or NaN are closed.  Weights and gradients are float64, from the exact formulas on the
same picks.
"""

from __future__ import annotations

import numpy as np

from .numerics import sigmoid


def scores(x: np.ndarray, scoring: str):
    """(s fp32, open) of fp32 logits."""
    with np.errstate(invalid="ignore", over="ignore"):
        open_ = x > -np.inf
        if scoring == "sigmoid":
            s = sigmoid(x)
        else:
            e = _softmax_terms(x, open_)
            total = e.sum(1, keepdims=True)
            s = (e / np.where(total > 0, total, 1.0)).astype(np.float32)
    return np.where(open_, s, np.float32(0.0)), open_


def _softmax_terms(x: np.ndarray, open_: np.ndarray) -> np.ndarray:
    m = np.where(open_, x, -np.inf).max(1, keepdims=True)
    d = np.where(x == m, 0.0, x.astype(np.float64) - m.astype(np.float64))
    return np.where(open_, np.exp(np.where(open_, d, 0.0)), 0.0)


def exact_scores(x: np.ndarray, scoring: str) -> np.ndarray:
    with np.errstate(invalid="ignore", over="ignore"):
        open_ = x > -np.inf
        if scoring == "sigmoid":
            return np.where(open_, 1.0 / (1.0 + np.exp(-x.astype(np.float64))), 0.0)
        e = _softmax_terms(x, open_)
        total = e.sum(1, keepdims=True)
        return e / np.where(total > 0, total, 1.0)


def route(x, bias, top_k, scoring, n_group=1, topk_group=None, group_top=2, renormalize=True, scale=1.0):
    """(weights float64 [T, k], ids int32 [T, k])."""
    x = np.asarray(x, np.float32)
    T, E = x.shape
    topk_group = n_group if topk_group is None else topk_group
    s, open_ = scores(x, scoring)
    with np.errstate(invalid="ignore"):
        v = s if bias is None else (s + np.asarray(bias, np.float32)).astype(np.float32)
        v = np.where(open_ & (v > -np.inf), v, np.float32(-np.inf))
    if n_group > 1:
        best = -np.sort(-v.reshape(T, n_group, -1), axis=2)
        score = best[:, :, 0]
        if group_top == 2 and best.shape[2] > 1:
            score = np.where(best[:, :, 1] > -np.inf, (best[:, :, 0] + best[:, :, 1]).astype(np.float32), score)
        kept = np.argsort(-score, axis=1, kind="stable")[:, :topk_group]
        mask = np.zeros((T, n_group), bool)
        np.put_along_axis(mask, kept, True, axis=1)
        v = np.where(np.repeat(mask, E // n_group, axis=1), v, np.float32(-np.inf))
    order = np.argsort(-v, axis=1, kind="stable")[:, :top_k]
    there = np.take_along_axis(v, order, 1) > -np.inf
    ids = np.sort(np.where(there, order, E), axis=1)
    there = ids < E
    ids = np.where(there, ids, -1).astype(np.int32)
    w = np.where(there, np.take_along_axis(exact_scores(x, scoring), np.where(there, ids, 0), 1), 0.0)
    if renormalize:
        w = w / (w.sum(1, keepdims=True) + 1e-20)
    return w * scale, ids


def weights_of(x, ids, scoring, renormalize=True, scale=1.0):
    """The weights of given picks as a function of the logits, float64 (for differences)."""
    there = ids >= 0
    w = np.where(there, np.take_along_axis(exact_scores(np.asarray(x), scoring), np.where(there, ids, 0), 1), 0.0)
    if renormalize:
        w = w / (w.sum(1, keepdims=True) + 1e-20)
    return w * scale


def route_backward(grad, x, ids, scoring, renormalize=True, scale=1.0):
    """(gradient of the logits, its scale): the second is the sum of the magnitudes that the formula adds up, by which
    a 32-bit evaluation's error is measured."""
    x, g = np.asarray(x, np.float64), np.asarray(grad, np.float64)
    there = (ids >= 0) & (ids < x.shape[1])
    at = np.where(there, ids, 0)
    s = exact_scores(x, scoring)
    p = np.where(there, np.take_along_axis(s, at, 1), 0.0)
    g = np.where(there, g, 0.0) * scale
    mag = np.abs(g)
    if renormalize:
        total = p.sum(1, keepdims=True) + 1e-20
        mag = np.where(there, (mag + (mag * p).sum(1, keepdims=True) / total) / total, 0.0)
        g = np.where(there, (g - (g * p).sum(1, keepdims=True) / total) / total, 0.0)
    d, m = np.zeros_like(x), np.zeros_like(x)
    rows = np.arange(x.shape[0])[:, None]
    np.add.at(d, (rows, at), np.where(there, g, 0.0))
    np.add.at(m, (rows, at), mag)
    if scoring == "sigmoid":
        slope = s * np.where(x > -np.inf, 1.0 / (1.0 + np.exp(np.minimum(x, 700.0))), 0.0)
        return d * slope, m * slope
    return (s * (d - (d * s).sum(1, keepdims=True)), s * (m + (m * s).sum(1, keepdims=True)))
