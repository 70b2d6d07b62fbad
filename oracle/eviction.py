"""ORACLE — rotated append and attention-weight eviction restated on the CPU.

Test infrastructure only; float64 numpy from the definitions.

* ``norm_rotate_fp64`` — x * weight / sqrt(mean(x^2) + eps), then the rotation
  of the first rotary_dim elements by position * frequency, pairs (i, i +
  rotary_dim / 2) or (2 i, 2 i + 1);
* ``attention_mass_fp64`` — per KV head and cached token, the sum over the
  head's query rows of softmax(q k^T / sqrt(D)) under the window's causal mask;
* ``select_kept`` — the first tokens, the last ones and the heaviest of the
  rest, ties to the lower index.
"""

from __future__ import annotations

import math

import numpy as np


def norm_rotate_fp64(x, positions, inv_freq, weight=None, eps=1e-6, interleaved=False):
    """x ``[..., tokens, heads, D]``, positions ``[..., tokens]``; returns the
    rotated heads and, per element, the sum of the magnitudes of the (up to
    two) normalised elements that form it (rounding errors scale with it)."""
    x = np.asarray(x, dtype=np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(axis=-1, keepdims=True) + eps) * np.asarray(weight, dtype=np.float64)
    half = len(inv_freq)
    theta = np.asarray(positions, dtype=np.float64)[..., None, None] * np.asarray(inv_freq, dtype=np.float64)
    first = np.arange(half) * 2 if interleaved else np.arange(half)
    second = first + 1 if interleaved else first + half
    out, span = x.copy(), np.abs(x)
    a, b = x[..., first], x[..., second]
    out[..., first] = a * np.cos(theta) - b * np.sin(theta)
    out[..., second] = b * np.cos(theta) + a * np.sin(theta)
    span[..., first] = span[..., second] = np.abs(a) + np.abs(b)
    return out, span


def attention_mass_fp64(q, keys):
    """q ``[Hq, window, D]``, keys ``[T, Hkv, D]`` float64 -> ``[Hkv, T]``."""
    q = np.asarray(q, dtype=np.float64)
    Hq, window, D = q.shape
    T, Hkv, _ = keys.shape
    group = Hq // Hkv
    visible = np.arange(T)[None, :] <= np.arange(T - window, T)[:, None]
    mass = np.zeros((Hkv, T))
    for h in range(Hq):
        s = np.where(visible, q[h] @ keys[:, h // group].T / math.sqrt(D), -np.inf)
        p = np.exp(s - s.max(axis=1, keepdims=True))
        mass[h // group] += (p / p.sum(axis=1, keepdims=True)).sum(axis=0)
    return mass


def select_kept(mass, budget, recent, sinks):
    """mass ``[T]`` float32 -> int32 ``[budget]``, ascending, -1 past T."""
    T = len(mass)
    if T <= budget:
        return np.concatenate([np.arange(T), np.full(budget - T, -1)]).astype(np.int32)
    middle = np.arange(sinks, T - recent)
    m = np.asarray(mass, dtype=np.float64)[middle]
    # heaviest first, NaN before everything, the lower index first among equals
    rank = np.lexsort((middle, -np.where(np.isnan(m), 0.0, m), ~np.isnan(m)))
    chosen = middle[rank[:budget - recent - sinks]]
    return np.concatenate([np.arange(sinks), np.sort(chosen), np.arange(T - recent, T)]).astype(np.int32)
