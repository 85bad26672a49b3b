"""Plain models, in 64 bits, of entries grouped by index, a router, the experts' products and low-rank
adapters, written from their definitions."""
from __future__ import annotations

import numpy as np

from np_decode import decode


def grouped(ids, groups):
    """(offsets, order): entries sorted by id (stable), those outside [0, groups) last."""
    key = np.where((ids >= 0) & (ids < groups), ids, groups)
    order = np.argsort(key, kind="stable").astype(np.int32)
    offsets = np.searchsorted(key[order], np.arange(groups + 1)).astype(np.int32)
    return offsets, order


def route(z, top_k, bias=None, sigmoid=False, normalise=True, scale=1.0, parts=1, top_parts=1):
    """ids (-1: none) and weights of rows of logits."""
    z = np.where(np.isnan(z), -np.inf, z.astype(np.float64))
    m, experts = z.shape
    ids = np.full((m, top_k), -1, np.int32)
    w = np.zeros((m, top_k))
    for r in range(m):
        x = z[r]
        live = x > -np.inf
        if not live.any():
            continue
        with np.errstate(over="ignore"):
            if sigmoid:
                s = np.where(live, 1 / (1 + np.exp(np.where(live, -x, 0))), 0)
            else:
                top = x.max()
                s = np.where(x == top, 1.0, np.exp(np.where(x == top, -np.inf, x) - (top if np.isfinite(top) else 0)))
                s = np.where((x < top) & np.isinf(top), 0, s)
        total = s.sum()
        key = x
        if bias is not None:
            key = (s if sigmoid else s / total) + bias.astype(np.float64)
            key = np.where(live & ~np.isnan(key), key, -np.inf)
        if parts > 1:
            g = key.reshape(parts, -1)
            best = -np.sort(-g, axis=1)
            score = best[:, 0] if bias is None or g.shape[1] == 1 else best[:, 0] + best[:, 1]
            keep = np.argsort(-score, kind="stable")[:top_parts]
            mask = np.zeros(parts, bool)
            mask[keep] = True
            key = np.where(mask[:, None], g, -np.inf).reshape(-1)
        pick = np.argsort(-key, kind="stable")[:top_k]
        pick = pick[key[pick] > -np.inf]
        ids[r, :len(pick)] = pick
        p = s[pick]
        if normalise:
            total = p.sum()
        elif sigmoid:
            total = 1.0
        if total > 0:
            w[r, :len(pick)] = p / total * scale
    return ids, w


def expert_values(w, t, experts, n, k):
    """(values, magnitudes) [experts][n][k] of GGUF blocks, in 64 bits: magnitudes count a K-quant's two
    terms apart, as a kernel adds them."""
    q, s, mn = decode(w, t, experts * n, k)
    v = s * q
    return (v - mn).reshape(experts, n, k), (np.abs(v) + np.abs(mn)).reshape(experts, n, k)


def q8_values(orc, x):
    """The values of the rows' Q8_0 blocks (codes and scales of the reference's quantization)."""
    qs, sc, _ = orc.quantize(np.ascontiguousarray(x, np.float32))
    m, k = x.shape
    return (qs.reshape(m, -1, 32).astype(np.float64) * sc.reshape(m, -1, 1).astype(np.float64)).reshape(m, k)


def product_bound(mag, x, k):
    """How far fp32 sums of products may be off, element by element: mag [n][k] magnitudes of the
    weights' terms, x [m][k] values of the rows.
      an activation is rounded once to fp32 (2^-24) and stands as fp16 hi + lo (lo's rounding: 2^-22), its
      smallest parts as subnormals of 2^-14 against a row maximum of 2^13 and more (2^-27 of that);
      every matrix instruction adds to a running sum (a step of 2^-23 of the magnitudes so far): up
      to 26 a super-block of 256, one multiply-add each after it, and the waves' and parts' sums."""
    s = np.abs(x) @ mag.T
    top = np.abs(x).max(1, keepdims=True) * mag.sum(1)[None]
    chunks = (k + 255) // 256
    return s * (2.0 ** -22 + 2.0 ** -24 + (26 + chunks + 10) * 2.0 ** -23) + top * 2.0 ** -27


def silu(g):
    with np.errstate(over="ignore"):
        return g / (1 + np.exp(-g))
