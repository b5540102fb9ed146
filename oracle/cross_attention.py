"""Attention to rows of another length, behind a shared prefix, and the residual stream between two norms, in float64 from the
definitions (no counterpart in the reference)."""

from __future__ import annotations

import numpy as np


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float, seen: np.ndarray):
    """One sequence: q [L, H, D], k, v [S, KV, D], seen bool [L, S] -> o [L, H, D]; the weighted mean of |v|, which bounds what
    roundings of the weights can do; and per row [L, H, 1] the largest sum of |q k| over a seen key, which bounds the roundings
    of a score. Keys that a query does not see take no part, whatever they hold; without keys: 0."""
    L, H, D = q.shape
    group = H // k.shape[1]
    o, size, load = np.zeros((L, H, D)), np.zeros((L, H, D)), np.zeros((L, H, 1))
    for i in range(L):
        at = np.flatnonzero(seen[i])
        if at.size == 0:
            continue
        for h in range(H):
            keys, query = k[at, h // group].astype(np.float64), q[i, h].astype(np.float64)
            x = keys @ query * scale
            load[i, h] = (np.abs(keys) @ np.abs(query)).max()
            p = np.exp(x - x.max())
            p /= p.sum()
            rows = v[at, h // group].astype(np.float64)
            o[i, h], size[i, h] = p @ rows, p @ np.abs(rows)
    return o, size, load


def cross_attention(q, k, v, scale, lens=None, mask=None):
    """q [B, L, H, D], k, v [B, S, KV, D], lens [B], mask [B, S]."""
    B, L, S = q.shape[0], q.shape[1], k.shape[1]
    out = []
    for b in range(B):
        seen = np.arange(S) < (S if lens is None else min(max(int(lens[b]), 0), S))
        if mask is not None:
            seen = seen & mask[b]
        out.append(attend(q[b], k[b], v[b], scale, np.broadcast_to(seen, (L, S))))
    return tuple(np.stack(x) for x in zip(*out))


def prefix_attention(q, prefix_k, prefix_v, k, v, scale, lens=None):
    """q [B, L, H, D], the prefix [P, KV, D], k, v [B, S, KV, D]: query i sees the prefix and the own keys j < lens[b] - L + 1 + i."""
    B, L, S, P = q.shape[0], q.shape[1], k.shape[1], prefix_k.shape[0]
    out = []
    for b in range(B):
        n = S if lens is None else min(max(int(lens[b]), 0), S)
        own = np.arange(S)[None] < n - L + 1 + np.arange(L)[:, None]
        seen = np.concatenate((np.ones((L, P), bool), own), 1)
        out.append(attend(q[b], np.concatenate((prefix_k, k[b])), np.concatenate((prefix_v, v[b])), scale, seen))
    return tuple(np.stack(x) for x in zip(*out))


def norm(x, kind, gamma, beta, eps):
    """RMSNorm (1) or LayerNorm (2) of float64 rows, or the rows themselves (0)."""
    if kind == 0:
        return x
    if kind == 2:
        x = x - x.mean(-1, keepdims=True)
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gamma
    return x + beta if kind == 2 else x


def residual_norm(x, y, post, post_gamma, post_beta, pre, pre_gamma, pre_beta, gate, scale, eps):
    """x_out and h (None without a pre-norm), unrounded; gate [G, C] or None."""
    x, y = x.astype(np.float64), y.astype(np.float64)
    g = 1.0 if gate is None else np.repeat(gate.astype(np.float64), x.shape[0] // gate.shape[0], 0)
    s = x + scale * g * norm(y, post, post_gamma, post_beta, eps)
    return s, None if pre == 0 else norm(s, pre, pre_gamma, pre_beta, eps)
