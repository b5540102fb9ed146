"""MX4 (OCP microscaling, E2M1 codes with an E8M0 exponent per 32 columns): quantization with the fused norm and rotation in
numpy float32, the codes' values, and the product in float64.

Quantization restates the HIP kernel's operations one by one (each a single IEEE float32 operation, fused multiply-adds
where fma32 stands), so codes and exponents can be compared bit for bit; tests/test_mx4.py pins it against definitions in
float64. The reference has no MX4 path.
"""

from __future__ import annotations

import numpy as np

from .gemm import fma32
from .rotq8 import INV_SQRT_128, fwht_rows

F32 = np.float32
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])  # E2M1 magnitudes by code
NONE, RMS, LAYER = 0, 1, 2


def _row_sum(v: np.ndarray, step) -> np.ndarray:
    """64 partial sums a row (partial 16 (b mod 4) + c: the 8-column chunks c of the 128-column blocks b, ascending), then
    folded in halves. `step(values, acc)` adds one column to every partial sum."""
    T, C = v.shape
    lanes = np.pad(v, ((0, 0), (0, -C % 512))).reshape(T, -1, 4 * 16, 8)
    acc = np.zeros((T, 64), F32)
    for i in range(lanes.shape[1]):
        for e in range(8):
            acc = step(lanes[:, i, :, e], acc)
    n = 32
    while n:
        acc = acc[:, :n] + acc[:, n : 2 * n]
        n //= 2
    return acc[:, 0]


def norm_rows(v: np.ndarray, norm: int, c_real: int, gamma: np.ndarray, beta: np.ndarray | None, eps: float) -> np.ndarray:
    """RMSNorm or LayerNorm over the first c_real columns of float32 v; columns past them count as zeros."""
    real = np.arange(v.shape[1]) < c_real
    v = np.where(real, v, F32(0))
    if norm == LAYER:
        mean = _row_sum(v, lambda x, a: a + x) / F32(c_real)
        v = np.where(real, v - mean[:, None], F32(0))
    var = _row_sum(v, lambda x, a: fma32(x, x, a)) / F32(c_real)
    rstd = F32(1) / np.sqrt(var + F32(eps))
    return fma32(v * rstd[:, None], gamma[None], (np.zeros_like(gamma) if beta is None else beta)[None])


def encode(v: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """float32 [T, C] -> (E2M1 codes uint8 [T, C], E8M0 exponents uint8 [T, C / 32])."""
    T, C = v.shape
    b = v.reshape(T, C // 32, 32).astype(np.float64)
    with np.errstate(invalid="ignore"):
        amax = np.abs(b).max(-1)  # not a number if any is
    finite = np.isfinite(amax)
    e = np.maximum(np.frexp(np.where(finite, amax, 1.0))[1] - 3, -127)
    e = np.where(finite & (amax > 0), e, -127)
    u = np.where(finite[..., None], np.ldexp(np.where(finite[..., None], np.abs(b), 0.0), -e[..., None]), 0.0)
    code = np.where(u < 2, np.rint(u * 2), np.where(u < 4, np.rint(u) + 2, np.rint(u / 2) + 4))
    code = np.minimum(code, 7).astype(np.uint8) + np.where(np.signbit(b), 8, 0).astype(np.uint8)
    return code.reshape(T, C), np.where(finite, e + 127, 255).astype(np.uint8)


def pack(code: np.ndarray, e: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """Codes and exponents in the kernels' layout: uint8 [T, C / 2] and int32 [C / 128, T]."""
    T = code.shape[0]
    words = np.ascontiguousarray(e).view("<i4").reshape(T, -1)
    return code[:, 0::2] | (code[:, 1::2] << 4), np.ascontiguousarray(words.T)


def unpack(codes: np.ndarray, scale: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    T = codes.shape[0]
    code = np.stack([codes & 15, codes >> 4], -1).reshape(T, -1)
    return code, np.ascontiguousarray(scale.T).view(np.uint8).reshape(T, -1)


def values(codes: np.ndarray, scale: np.ndarray) -> np.ndarray:
    """float64 values of packed codes."""
    code, e = unpack(codes, scale)
    v = GRID[code & 7] * np.where(code & 8, -1.0, 1.0)
    f = np.where(e == 255, np.nan, np.ldexp(1.0, e.astype(np.int32) - 127))
    return v * np.repeat(f, 32, axis=1)


def quant_mx4(x: np.ndarray, rotate: bool = True, norm: int = NONE, c_real: int = 0, gamma: np.ndarray | None = None,
              beta: np.ndarray | None = None, eps: float = 1e-6) -> tuple[np.ndarray, np.ndarray]:
    """float32 x [T, C] (values of the input type) -> packed codes and scale."""
    T, C = x.shape
    v = x.astype(F32)
    with np.errstate(invalid="ignore", over="ignore"):
        if norm != NONE:
            v = norm_rows(v, norm, c_real or C, gamma.astype(F32), None if beta is None else beta.astype(F32), eps)
        if rotate:
            v = fwht_rows(v.reshape(-1, 128), tuple(range(7))).reshape(T, C) * INV_SQRT_128
    return pack(*encode(v))


def gemm_mx4(a: tuple, w: tuple, bias: np.ndarray | None = None) -> tuple[np.ndarray, np.ndarray]:
    """float64 y = A W^T + bias, and sum_k |A| |W| + |bias| (what a summation's rounding is relative to)."""
    av, wv = values(*a), values(*w)
    b = 0.0 if bias is None else bias.astype(np.float64)
    return av @ wv.T + b, np.abs(av) @ np.abs(wv).T + np.abs(b)
