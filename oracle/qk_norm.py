"""Norm of each head's query or key and its rotation by position, in float64. The reference rotates in its QKV epilogue
(foidfinder/backends/cuda/csrc/gemm.cuh:140-151) and has no head norm."""

from __future__ import annotations

import numpy as np

NONE, RMS, LAYER = 0, 1, 2


def head_norm(x: np.ndarray, norm: int, gamma: np.ndarray | None, beta: np.ndarray | None, eps: float) -> np.ndarray:
    x = x.astype(np.float64)
    if norm == LAYER:
        x = x - x.mean(-1, keepdims=True)
    if norm != NONE:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gamma.astype(np.float64)
    return x + beta.astype(np.float64) if norm == LAYER else x


def rotate(x: np.ndarray, cos: np.ndarray, sin: np.ndarray, pairs: bool) -> tuple[np.ndarray, np.ndarray]:
    """x [T, heads, D] turned by the angles of cos/sin [T, R / 2] (its first R columns), and the sum of the magnitudes of the
    terms of each value."""
    half = cos.shape[1]
    i = np.arange(half)
    first, second = (2 * i, 2 * i + 1) if pairs else (i, i + half)
    c, s = cos.astype(np.float64)[:, None], sin.astype(np.float64)[:, None]
    out, size = x.copy(), np.abs(x)
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * c - b * s, a * s + b * c
    size[..., first], size[..., second] = np.abs(a * c) + np.abs(b * s), np.abs(a * s) + np.abs(b * c)
    return out, size


def qk_norm_rope(x: np.ndarray, norm: int, gamma, beta, eps: float, cos: np.ndarray, sin: np.ndarray,
                 positions: np.ndarray, pairs: bool, scale: float = 1.0) -> tuple[np.ndarray, np.ndarray]:
    """x [T, heads, D], tables [L, R / 2], positions [T] -> float64 result and the size of its terms; tokens whose position is
    outside the table are not numbers."""
    ok = (positions >= 0) & (positions < cos.shape[0])
    p = np.where(ok, positions, 0)
    y, size = rotate(head_norm(x, norm, gamma, beta, eps), cos[p], sin[p], pairs)
    return np.where(ok[:, None, None], y * scale, np.nan), size * abs(scale)
