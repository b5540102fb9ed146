"""The gfx950 kernel library behind a C ABI (include/foidfinder_rocm.h), loaded with ctypes and registered as
`torch.ops.foidfinder_rocm.*` with the reference's op schemas.

Mirrors foidfinder/backends/cuda/kernels.py:38-48 (`kernels()` -> the op namespace) and the op registration of
foidfinder/backends/cuda/csrc/kernels.cu:267-281. Every op is out-param / in-place, returns nothing, allocates
nothing and launches on the current stream, so a forward built from them can be captured in a HIP graph. Failed
preconditions raise RuntimeError, as TORCH_CHECK does in the reference.

There is no CPU fallback: without the built library every call raises.
"""

from __future__ import annotations

import ctypes
import os
from functools import cache
from pathlib import Path

import torch
from torch.autograd import forward_ad

LIB_PATH = Path(__file__).resolve().parent / "libfoidfinder_rocm.so"
ENV = "FOIDFINDER_ROCM_KERNELS"  # path to a prebuilt library (the reference's $FOIDFINDER_KERNELS)

# Epilogue codes (include/foidfinder_rocm.h); 0-2 as foidfinder/backends/cuda/engine.py:24.
EPI_QKV_ROPE, EPI_RESIDUAL, EPI_GELU_F16, EPI_SWIGLU, EPI_BIAS_F16, EPI_I32 = 0, 1, 2, 3, 4, 5

# Norm codes of quant_mx4, qk_norm_rope and residual_norm (include/foidfinder_rocm.h).
NORM_NONE, NORM_RMS, NORM_LAYER = 0, 1, 2

_vp, _i64, _f32, _int = ctypes.c_void_p, ctypes.c_int64, ctypes.c_float, ctypes.c_int
SIGNATURES = {
    "ff_abi_version": ([], _int),
    "ff_last_error": ([], ctypes.c_char_p),
    "ff_rot_q8_1024": ([_vp, _vp, _vp, _f32, _i64, _vp, _vp, _vp], _int),
    "ff_rot_q8_h128": ([_vp, _i64, _i64, _i64, _vp, _vp, _f32, _vp, _vp, _vp], _int),
    "ff_gemm_s8": ([_vp, _vp, _i64, _i64, _i64, _vp, _vp, _vp, _vp, _int, _int, _vp, _vp, _i64, _f32, _vp], _int),
    "ff_gemm_s8_variants": ([], _int),
    "ff_attention": ([_vp, _vp, _i64, _i64, _i64, _vp], _int),
    "ff_cross_attention": ([_vp, _i64, _i64, _i64] * 4 + [_int] + [_i64] * 6 + [_f32, _vp, _vp, _i64, _vp, _i64, _vp],
                           _int),
    "ff_cross_attention_work": ([_i64] * 6, _i64),
    "ff_prefix_attention": ([_vp, _i64, _i64, _i64] + [_vp, _i64, _i64] * 2 + [_vp, _i64, _i64, _i64] * 3 + [_int]
                            + [_i64] * 7 + [_f32, _vp, _vp, _i64, _vp], _int),
    "ff_prefix_attention_work": ([_i64] * 7, _i64),
    "ff_residual_norm": ([_vp, _i64] * 4 + [_int, _i64, _i64] + [_int, _vp, _vp] * 2 + [_vp, _i64, _int, _f32, _f32, _vp],
                         _int),
    "ff_resample_u8": ([_vp, _i64, _i64, _int, _vp, _vp, _i64, _i64, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _vp],
                       _int),
    "ff_bicubic_taps": ([*[_i64] * 3, _vp, _vp, *[_i64] * 4, _vp, _vp, _i64, _vp], _int),
    "ff_layer_norm2": ([_vp, _i64, _i64, _vp, _vp, _vp, _vp, _f32, _vp, _vp], _int),
    "ff_slot_weights_blocks": ([_i64], _i64),
    "ff_slot_weights": ([_vp, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _vp, _vp, _vp], _int),
    "ff_pool_weights_blocks": ([_i64], _i64),
    "ff_pool_weights": ([_vp, _vp, _i64, _vp, _i64, _vp, *[_i64] * 6, _vp, _vp, _vp], _int),
    "ff_pool_sum": ([_vp, _vp, *[_i64] * 5, _vp, _vp], _int),
    "ff_pool_values": ([_vp, _vp, _vp, _vp, *[_i64] * 5, _vp, _vp], _int),
    "ff_pool_queries": ([*[_vp] * 7, _f32, *[_i64] * 5, _vp, _vp, _vp, _vp], _int),
    "ff_pool_keys": ([_vp, _vp, _i64, _i64, _i64, _i64, _vp, _vp], _int),
    "ff_pool_tree": ([*[_vp] * 5, _i64, _f32, *[_i64] * 5, _vp, _vp], _int),
    "ff_pool_leaf": ([_vp, _vp, _vp, _i64, _i64, _i64, _i64, _vp, _vp], _int),
    "ff_patch_embed": ([_vp, _vp, _vp, _vp, _i64, _i64, _i64, _vp, _vp], _int),
    "ff_quant_mx4": ([_vp, _int, *[_i64] * 3, _int, _int, _i64, _vp, _vp, _f32, _vp, _vp, _vp], _int),
    "ff_dequant_mx4": ([_vp, _vp, _i64, _i64, _vp, _int, _vp], _int),
    "ff_gemm_mx4": ([*[_vp] * 4, *[_i64] * 3, *[_vp] * 3, _int, _int, _int, _vp], _int),
    "ff_gemm_mx4_variants": ([], _int),
    "ff_qk_norm_rope": ([*[_vp, _i64, _i64] * 4, _int, *[_i64] * 4, _int, *[_vp] * 4, _f32, _vp, _vp, _i64, _i64, _int, _vp,
                         _int, _f32, _vp], _int),
    "ff_head": ([_vp, _i64, _vp, _vp, _f32, _vp, _vp, _i64, _i64, _i64, _vp, _vp], _int),
}
ABI_VERSION = 5


@cache
def lib() -> ctypes.CDLL:
    """The loaded C library. torch is imported first so the library binds to the HIP runtime torch already loaded."""
    path = Path(os.environ.get(ENV, LIB_PATH))
    if not path.exists():
        raise RuntimeError(f"{path} is missing: build it with `python -m foidfinder_amd.build`")
    handle = ctypes.CDLL(str(path))
    for name, (args, res) in SIGNATURES.items():
        fn = getattr(handle, name)
        fn.argtypes, fn.restype = args, res
    if handle.ff_abi_version() != ABI_VERSION:
        raise RuntimeError(f"{path}: ABI {handle.ff_abi_version()}, expected {ABI_VERSION}")
    return handle


def _check(status: int) -> None:
    if status != 0:
        raise RuntimeError(lib().ff_last_error().decode())


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _run(name: str, dev: int, *args) -> None:
    """Calls a launching function of the library on device `dev`'s current stream, with that device current. A call is
    made of a few us of host work in all, so nothing is switched or built that is not needed: the device is entered only
    if it is not the current one already, and the stream comes as its raw handle."""
    fn = getattr(lib(), name)
    if torch._C._cuda_getDevice() == dev:  # a tensor on a GPU is there, so the runtime is up
        _check(fn(*args, torch._C._cuda_getCurrentRawStream(dev)))
        return
    with torch.cuda.device(dev):
        _check(fn(*args, torch._C._cuda_getCurrentRawStream(dev)))


def _require(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _on_gpu(*ts: torch.Tensor | None) -> int:
    """The device index of contiguous tensors that are all on one GPU."""
    dev = -1
    for t in ts:
        if t is None:
            continue
        d = t.get_device()  # -1 on the CPU
        if d < 0:
            raise RuntimeError("foidfinder_rocm ops take GPU tensors")
        if not t.is_contiguous():
            raise RuntimeError("foidfinder_rocm ops take contiguous tensors")
        if d != dev:
            if dev >= 0:
                raise RuntimeError("all tensors must be on one device")
            dev = d
    return dev


# ---- op implementations (raw; also callable directly, bypassing the dispatcher) ----


def rot_q8_1024(
    x: torch.Tensor,
    gamma: torch.Tensor | None,
    beta: torch.Tensor | None,
    out: torch.Tensor,
    row_scale: torch.Tensor,
    eps: float = 1e-5,
) -> None:
    """x fp16 [T, 1024] -> out int8 [T, 1024], row_scale fp32 [T]; LayerNorm(gamma, beta, eps) first if given."""
    dev = _on_gpu(x, gamma, beta, out, row_scale)
    _require(x.dim() == 2 and x.size(1) == 1024 and x.dtype == torch.float16, "x must be fp16 [T, 1024]")
    _require(out.dtype == torch.int8 and out.shape == x.shape, "out must be int8 [T, 1024]")
    _require(row_scale.dtype == torch.float32 and row_scale.numel() == x.size(0), "row_scale must be fp32 [T]")
    if gamma is not None:
        _require(beta is not None, "gamma and beta go together")
        _require(gamma.dtype == beta.dtype == torch.float32 and gamma.numel() == beta.numel() == 1024,
                 "gamma/beta must be fp32 [1024]")
    _run("ff_rot_q8_1024", dev, _ptr(x), _ptr(gamma), _ptr(beta), eps, x.size(0), _ptr(out), _ptr(row_scale))


def rot_q8_h128(
    x: torch.Tensor,
    out: torch.Tensor,
    row_scale: torch.Tensor,
    gamma: torch.Tensor | None = None,
    beta: torch.Tensor | None = None,
    c_real: int = 0,
    eps: float = 1e-6,
) -> None:
    """x fp16 [T, C] (C % 128 == 0) -> out int8 [T, C], row_scale fp32 [T]; LayerNorm over the first c_real columns
    (default: all) first if gamma is given. gamma/beta are fp32 [C] with zeros in columns >= c_real
    (`pad_norm` builds them)."""
    dev = _on_gpu(x, out, row_scale, gamma, beta)
    _require(x.dim() == 2 and x.dtype == torch.float16, "x must be fp16 [T, C]")
    _require(out.dtype == torch.int8 and out.shape == x.shape, "out must be int8 [T, C]")
    _require(row_scale.dtype == torch.float32 and row_scale.numel() == x.size(0), "row_scale must be fp32 [T]")
    C = x.size(1)
    cr = c_real or C
    if gamma is not None:
        _require(beta is not None, "gamma and beta go together")
        _require(gamma.dtype == beta.dtype == torch.float32 and gamma.numel() == beta.numel() == C,
                 "gamma/beta must be fp32 [C], zero past c_real")
    _run("ff_rot_q8_h128", dev, _ptr(x), x.size(0), C, cr, _ptr(gamma), _ptr(beta), eps, _ptr(out), _ptr(row_scale))


def pad_norm(weight: torch.Tensor, bias: torch.Tensor, C: int) -> tuple[torch.Tensor, torch.Tensor]:
    """LayerNorm gamma/beta over c_real columns -> fp32 [C] with zeros past c_real, as rot_q8_h128 takes them."""
    g = torch.zeros(C, dtype=torch.float32, device=weight.device)
    b = torch.zeros(C, dtype=torch.float32, device=weight.device)
    g[: weight.numel()] = weight.float().reshape(-1)
    b[: bias.numel()] = bias.float().reshape(-1)
    return g, b


def out_shape(M: int, N: int, epi: int) -> tuple[int, int]:
    return (M, N // 2) if epi == EPI_SWIGLU else (M, N)


def gemm_s8(
    A: torch.Tensor,
    W: torch.Tensor,
    row_scale: torch.Tensor,
    col_scale: torch.Tensor,
    bias: torch.Tensor,
    out: torch.Tensor,
    epi: int,
    stages: int,
    rope_cos: torch.Tensor | None,
    rope_sin: torch.Tensor | None,
    q_scale: float,
) -> None:
    """A int8 [M, K] x W int8 [N, K] -> epilogue into out. `stages` selects the tile variant (0 = default), the
    knob the engine autotunes (the reference's pipeline depth)."""
    dev = _on_gpu(A, W, row_scale, col_scale, bias, out, rope_cos, rope_sin)
    _require(A.dtype == W.dtype == torch.int8 and A.dim() == W.dim() == 2, "A and W must be int8 matrices")
    M, K = A.shape
    N = W.size(0)
    _require(W.size(1) == K, "A and W must share K")
    want = torch.int32 if epi == EPI_I32 else torch.float16
    shape = out_shape(M, N, epi)
    if out.dtype != want or tuple(out.shape) != shape:
        raise RuntimeError(f"out must be {want} {shape}")
    if epi != EPI_I32:
        _require(row_scale.dtype == col_scale.dtype == bias.dtype == torch.float32, "scales and bias must be fp32")
        _require(row_scale.numel() == M and col_scale.numel() == N and bias.numel() == N, "scale/bias sizes")
    rope_len = 0
    if epi == EPI_QKV_ROPE:
        _require(rope_cos is not None and rope_sin is not None, "QKV epilogue needs RoPE tables")
        _require(rope_cos.dtype == rope_sin.dtype == torch.float32 and rope_cos.shape == rope_sin.shape
                 and rope_cos.dim() == 2 and rope_cos.size(1) == 32, "RoPE tables must be fp32 [L, 32]")
        rope_len = rope_cos.size(0)
    _run("ff_gemm_s8", dev, _ptr(A), _ptr(W), M, N, K, _ptr(row_scale), _ptr(col_scale), _ptr(bias), _ptr(out), epi,
         stages, _ptr(rope_cos), _ptr(rope_sin), rope_len, q_scale)


def attention(qkv: torch.Tensor, out: torch.Tensor, seq_len: int) -> None:
    """qkv fp16 [T, 3C] (q rotated and pre-scaled, k rotated) -> out fp16 [T, C]; heads of 64, any seq_len."""
    dev = _on_gpu(qkv, out)
    _require(qkv.dtype == out.dtype == torch.float16, "qkv and out must be fp16")
    _require(qkv.dim() == 2 and qkv.size(1) % 192 == 0, "qkv must be [T, 3 * heads * 64]")
    C = qkv.size(1) // 3
    _require(out.shape == (qkv.size(0), C), "out must be [T, C]")
    _run("ff_attention", dev, _ptr(qkv), _ptr(out), qkv.size(0), C // 64, seq_len)


def resample_u8(src: torch.Tensor, axis: int, kk: torch.Tensor, bounds: torch.Tensor, row0: int, out: torch.Tensor,
                region: tuple[int, int, int, int]) -> None:
    """One Pillow resampling pass (include/foidfinder_rocm.h, ff_resample_u8): src uint8 [H, W, 3] -> out uint8
    [out_h, out_w, 3], `region` = (top, left, h, w) resampled along axis 0 (width) or 1 (height), the rest white."""
    dev = _on_gpu(src, kk, bounds, out)
    _require(src.dtype == out.dtype == torch.uint8 and src.dim() == out.dim() == 3 and src.size(2) == out.size(2) == 3,
             "src and out must be uint8 [rows, cols, 3]")
    _require(src.is_contiguous() and out.is_contiguous(), "src and out must be contiguous")
    _require(kk.dtype == bounds.dtype == torch.int32 and kk.dim() == 2 and bounds.dim() == 2 and bounds.size(1) == 2
             and kk.is_contiguous() and bounds.is_contiguous(), "kk int32 [n, ksize], bounds int32 [n, 2]")
    top, left, h, w = region
    n = w if axis == 0 else h
    _require(kk.size(0) >= n and bounds.size(0) >= n, "kk/bounds need a row per output index of the region")
    _run("ff_resample_u8", dev, _ptr(src), src.size(0), src.size(1), axis, _ptr(kk), _ptr(bounds), kk.size(1), row0,
         _ptr(out), out.size(0), out.size(1), top, left, h, w)


def bicubic_taps(width: tuple[int, int, int], height: tuple[int, int, int], kk_w: torch.Tensor, bounds_w: torch.Tensor,
                 kk_h: torch.Tensor, bounds_h: torch.Tensor) -> None:
    """Pillow's bicubic taps of both axes (include/foidfinder_rocm.h, ff_bicubic_taps): `width` and `height` are (input
    size, output size, shift); kk int32 [output size, ksize], bounds int32 [output size, 2]."""
    dev = _on_gpu(kk_w, bounds_w, kk_h, bounds_h)
    for (_, n, _), kk, bounds in ((width, kk_w, bounds_w), (height, kk_h, bounds_h)):
        _require(kk.dtype == bounds.dtype == torch.int32 and kk.dim() == 2 and kk.size(0) == n
                 and tuple(bounds.shape) == (n, 2), "kk int32 [n, ksize], bounds int32 [n, 2]")
    _run("ff_bicubic_taps", dev, width[0], width[1], kk_w.size(1), _ptr(kk_w), _ptr(bounds_w), width[2], height[0],
         height[1], kk_h.size(1), _ptr(kk_h), _ptr(bounds_h), height[2])


def layer_norm2(x: torch.Tensor, g1: torch.Tensor, b1: torch.Tensor, g2: torch.Tensor, b2: torch.Tensor, eps: float,
                out: torch.Tensor) -> None:
    """out = LN(fp16(LN(x; g1, b1)); g2, b2) over the last dimension of fp16 x [..., C] (fp16 params [C])."""
    dev = _on_gpu(x, g1, b1, g2, b2, out)
    C = x.size(-1)
    _require(x.dtype == out.dtype == torch.float16 and x.is_contiguous() and out.is_contiguous()
             and out.shape == x.shape, "x and out must be contiguous fp16 of one shape")
    _require(all(t.dtype == torch.float16 and t.numel() == C for t in (g1, b1, g2, b2)), "params must be fp16 [C]")
    _run("ff_layer_norm2", dev, _ptr(x), x.numel() // C, C, _ptr(g1), _ptr(b1), _ptr(g2), _ptr(b2), eps, _ptr(out))


def slot_weights_blocks(N: int) -> int:
    return lib().ff_slot_weights_blocks(N)


def slot_weights(logits: torch.Tensor, c: torch.Tensor, bias: torch.Tensor, heads: int, a_t: torch.Tensor,
                 partial: torch.Tensor) -> None:
    """Tree-pool weights (include/foidfinder_rocm.h, ff_slot_weights): logits fp16 [B, N, heads*M] + c fp32 ([heads*M]
    shared or [B, heads*M]) -> a_t fp16 [B, heads*M, N], partial fp32 [B, blocks, heads*M]."""
    dev = _on_gpu(logits, c, bias, a_t, partial)
    B, N, GM = logits.shape
    M = bias.numel()
    _require(logits.dtype == torch.float16 and logits.is_contiguous() and GM == heads * M, "logits fp16 [B, N, heads*M]")
    _require(c.dtype == bias.dtype == torch.float32 and c.is_contiguous() and bias.is_contiguous(), "c, bias fp32")
    _require(c.numel() in (GM, B * GM), "c must be [heads*M] or [B, heads*M]")
    _require(a_t.dtype == torch.float16 and a_t.is_contiguous() and a_t.shape == (B, GM, N), "a_t fp16 [B, heads*M, N]")
    _require(partial.dtype == torch.float32 and partial.is_contiguous()
             and partial.shape == (B, slot_weights_blocks(N), GM), "partial fp32 [B, blocks, heads*M]")
    _run("ff_slot_weights", dev, _ptr(logits), _ptr(c), 0 if c.numel() == GM else GM, _ptr(bias), B, N, heads, M,
         _ptr(a_t), _ptr(partial))


def pool_weights_blocks(N: int) -> int:
    return lib().ff_pool_weights_blocks(N)


def pool_fits(B: int, N: int, heads: int, leaves: int, dim: int) -> bool:
    """Whether the tree pool's kernels take B images of N tokens (others go to the library's products): 32-bit byte
    offsets within an image's tokens and weights (rows padded to 8 tokens), and at most 65535 launch rows of images and of
    16 (image, leaf) pairs each."""
    ldt = (N + 7) // 8 * 8
    return N * dim < 1 << 30 and heads * leaves * ldt < 1 << 30 and B <= 65535 and B * leaves <= 16 * 65535


def _half(shape: tuple, *ts: torch.Tensor) -> None:
    for t in ts:
        if t.dtype != torch.float16 or tuple(t.shape) != shape:
            raise RuntimeError(f"need fp16 {shape}")


def _float(numel: int, *ts: torch.Tensor) -> None:
    for t in ts:
        if t.dtype != torch.float32 or t.numel() != numel:
            raise RuntimeError(f"need fp32 of {numel} elements")


def pool_weights(xn: torch.Tensor, u: torch.Tensor, c: torch.Tensor, bias: torch.Tensor, heads: int, a_t: torch.Tensor,
                 partial: torch.Tensor) -> None:
    """Tree-pool weights from the tokens and the queries' u (include/foidfinder_rocm.h, ff_pool_weights): xn fp16
    [B, N, D], u fp16 [heads*M, D] (shared) or [B, heads*M, D], c fp32 [heads*M] or [B, heads*M], bias fp32 [M] -> a_t
    fp16 [B, heads*M, ldt], partial fp32 [B, blocks, heads*M]."""
    dev = _on_gpu(xn, u, c, bias, a_t, partial)
    B, N, D = xn.shape
    M = bias.numel()
    GM = heads * M
    _require(xn.dtype == torch.float16 and u.dtype == torch.float16 and tuple(u.shape[-2:]) == (GM, D)
             and (u.dim() == 2 or u.dim() == 3 and u.size(0) == B), "u must be fp16 [heads*M, D] or [B, heads*M, D]")
    _require(c.dtype == bias.dtype == torch.float32 and c.numel() in (GM, B * GM), "c must be fp32 [heads*M] or [B, heads*M]")
    _half((B, GM, a_t.size(-1)), a_t)
    _float(B * pool_weights_blocks(N) * GM, partial)
    _run("ff_pool_weights", dev, _ptr(xn), _ptr(u), 0 if u.dim() == 2 else GM * D, _ptr(c), 0 if c.numel() == GM else
         GM, _ptr(bias), B, N, heads, M, D, a_t.size(-1), _ptr(a_t), _ptr(partial))


def pool_sum(a_t: torch.Tensor, xn: torch.Tensor, pooled: torch.Tensor) -> None:
    """pooled fp16 [B, GM, D] = a_t xn over the N tokens of xn fp16 [B, N, D], a_t fp16 [B, GM, ldt] as pool_weights leaves
    it (ff_pool_sum)."""
    dev = _on_gpu(a_t, xn, pooled)
    B, N, D = xn.shape
    GM = a_t.size(1)
    _half((B, N, D), xn)
    _half((B, GM, a_t.size(-1)), a_t)
    _half((B, GM, D), pooled)
    _run("ff_pool_sum", dev, _ptr(a_t), _ptr(xn), B, N, GM, D, a_t.size(-1), _ptr(pooled))


def pool_values(pooled: torch.Tensor, wv: torch.Tensor, bv: torch.Tensor, partial: torch.Tensor, heads: int,
                z: torch.Tensor) -> None:
    """z fp16 [B, M, D] from pooled fp16 [B, heads*M, D], wv fp16 [D, D], bv fp32 [D] and the weights' partial sums."""
    dev = _on_gpu(pooled, wv, bv, partial, z)
    B, M, D = z.shape
    _half((B, M, D), z)
    _half((B, heads * M, D), pooled)
    _half((D, D), wv)
    _float(D, bv)
    _float(B * partial.size(1) * heads * M, partial)
    _run("ff_pool_values", dev, _ptr(pooled), _ptr(wv), _ptr(bv), _ptr(partial), partial.size(1), B, heads, M, D,
         _ptr(z))


def pool_queries(z: torch.Tensor, trunk_g: torch.Tensor, trunk_b: torch.Tensor, child: torch.Tensor,
                 child_g: torch.Tensor, child_b: torch.Tensor, bk: torch.Tensor, heads: int, eps: float,
                 parent: torch.Tensor, qleaf: torch.Tensor, cq: torch.Tensor) -> None:
    """z fp16 [B, C, D] -> parent fp16 [B, C, D], qleaf fp16 [B, Q, D], cq fp32 [B, heads*Q] (ff_pool_queries)."""
    dev = _on_gpu(z, trunk_g, trunk_b, child, child_g, child_b, bk, parent, qleaf, cq)
    B, C, D = z.shape
    Q = child.size(0)
    _half((B, C, D), z, parent)
    _half((B, Q, D), qleaf)
    _half((Q, D), child)
    _half((D,), trunk_g, trunk_b, child_g, child_b)
    _float(D, bk)
    _float(B * heads * Q, cq)
    _run("ff_pool_queries", dev, _ptr(z), _ptr(trunk_g), _ptr(trunk_b), _ptr(child), _ptr(child_g), _ptr(child_b),
         _ptr(bk), eps, B, C, Q, heads, D, _ptr(parent), _ptr(qleaf), _ptr(cq))


def pool_keys(qleaf: torch.Tensor, kT: torch.Tensor, u: torch.Tensor) -> None:
    """u fp16 [B, heads*Q, D] from qleaf fp16 [B, Q, D] and kT fp16 [heads, D, D / heads] (ff_pool_keys)."""
    dev = _on_gpu(qleaf, kT, u)
    B, Q, D = qleaf.shape
    heads = kT.size(0)
    _half((B, Q, D), qleaf)
    _half((heads, D, D // heads), kT)
    _half((B, heads * Q, D), u)
    _run("ff_pool_keys", dev, _ptr(qleaf), _ptr(kT), B, Q, heads, D, _ptr(u))


def pool_tree(parent: torch.Tensor, zc: torch.Tensor, g: torch.Tensor, b: torch.Tensor, partial: torch.Tensor,
              heads: int, eps: float, tree: torch.Tensor) -> None:
    """tree fp16 [Q, B, D] from parent fp16 [B, C, D], zc fp16 [B, Q, D] and the weights' partial sums (ff_pool_tree)."""
    dev = _on_gpu(parent, zc, g, b, partial, tree)
    B, Q, D = zc.shape
    _half((B, parent.size(1), D), parent)
    _half((B, Q, D), zc)
    _half((D,), g, b)
    _half((Q, B, D), tree)
    _float(B * partial.size(1) * heads * Q, partial)
    _run("ff_pool_tree", dev, _ptr(parent), _ptr(zc), _ptr(g), _ptr(b), _ptr(partial), partial.size(1), eps, B,
         parent.size(1), Q, heads, D, _ptr(tree))


def pool_leaf(tree: torch.Tensor, wl: torch.Tensor, bl: torch.Tensor, leaf: torch.Tensor) -> None:
    """leaf fp16 [B, Q*F] from tree fp16 [Q, B, D], wl fp16 [Q, F, D], bl fp16 [Q, F] (ff_pool_leaf)."""
    dev = _on_gpu(tree, wl, bl, leaf)
    Q, B, D = tree.shape
    F = wl.size(1)
    _half((Q, B, D), tree)
    _half((Q, F, D), wl)
    _half((Q, F), bl)
    _half((B, Q * F), leaf)
    _run("ff_pool_leaf", dev, _ptr(tree), _ptr(wl), _ptr(bl), B, Q, F, D, _ptr(leaf))


PATCH_COLS, PATCH_PAD = 588, 608  # 14 x 14 x 3, and the row length of patch_embed's weights


def pad_patch_weight(w: torch.Tensor) -> torch.Tensor:
    """Patch weights [N, 588] -> fp16 [N, 608] with zeros past column 588, as patch_embed takes them."""
    out = torch.zeros(w.size(0), PATCH_PAD, dtype=torch.half, device=w.device)
    out[:, :PATCH_COLS] = w
    return out


def patch_embed(img: torch.Tensor, w: torch.Tensor, bias_pos: torch.Tensor, cls: torch.Tensor, x: torch.Tensor) -> None:
    """x fp16 [B, 1 + grid^2, N]: the class row, then each 14 x 14 patch of img fp16 [B, S, S, 3] times w fp16 [N, 608]
    (pad_patch_weight) plus bias_pos fp16 [grid^2, N] (ff_patch_embed)."""
    dev = _on_gpu(img, w, bias_pos, cls, x)
    B, S = img.shape[:2]
    grid, N = S // 14, w.size(0)
    _half((B, grid * 14, grid * 14, 3), img)
    _half((N, PATCH_PAD), w)
    _half((grid * grid, N), bias_pos)
    _half((N,), cls)
    _half((B, 1 + grid * grid, N), x)
    _run("ff_patch_embed", dev, _ptr(img), _ptr(w), _ptr(bias_pos), _ptr(cls), B, grid, N, _ptr(x))


def head_fits(x: torch.Tensor, W: torch.Tensor) -> bool:
    """Whether `head` takes the rows x with W [N, K] (others go to the library's GEMM): up to 64 rows, and fp16, which a
    library product under autocast need not have left."""
    return x.size(0) <= 64 and x.dtype == torch.float16 and W.size(1) % 32 == 0 and W.size(1) <= 1280


def unfollowed(x: torch.Tensor) -> bool:
    """Whether x is a plain GPU tensor that nothing follows, so that an op here can take the place of a torch product: these
    ops go by addresses, past autograd (backward and forward), functorch's transforms, tracing and dispatch modes."""
    return (type(x) is torch.Tensor and x.is_cuda and not (x.requires_grad and torch.is_grad_enabled())
            and torch.autograd.forward_ad._current_level < 0 and not torch._C._functorch.is_functorch_wrapped_tensor(x)
            and not torch.jit.is_tracing() and not torch.compiler.is_compiling()
            and torch._C._len_torch_dispatch_stack() == 0)


def head(x: torch.Tensor, W: torch.Tensor, bias: torch.Tensor, out: torch.Tensor, gamma: torch.Tensor | None = None,
         beta: torch.Tensor | None = None, eps: float = 1e-6) -> None:
    """Tag head: out fp32 [B, N] = LN(x) W^T + bias, x fp16 [B, K] with contiguous rows (any row stride from K up that is
    a multiple of 8; rows that overlap are refused), W fp16 [N, K], bias fp16 [N]; the norm (fp32 gamma, beta [K]) only if
    given (ff_head)."""
    dev = _on_gpu(W, bias, out, gamma, beta)
    B, K = x.shape
    N = W.size(0)
    _require(x.device == W.device and x.dtype == torch.float16 and x.stride(1) == 1, "x must be fp16 rows on W's device")
    _half((N, K), W)
    _half((N,), bias)
    _require(out.dtype == torch.float32 and tuple(out.shape) == (B, N), "out must be fp32 [B, N]")
    if gamma is not None:
        _require(beta is not None, "gamma and beta go together")
        _float(K, gamma, beta)
    stride = x.stride(0) if B > 1 else K  # a single row's stride says nothing
    _run("ff_head", dev, _ptr(x), stride, _ptr(gamma), _ptr(beta), eps, _ptr(W), _ptr(bias), B, N, K,
         _ptr(out))


_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_HALVES = (torch.float16, torch.bfloat16)


def _mx4(codes: torch.Tensor, scale: torch.Tensor, name: str) -> tuple[int, int]:
    """Rows and columns of an MX4 tensor: codes uint8 [T, C / 2], scale int32 [C / 128, T]."""
    shape = codes.shape
    if codes.dtype != torch.uint8 or len(shape) != 2 or shape[1] % 64 != 0:
        raise RuntimeError(f"{name} codes must be uint8 [T, C / 2] with C a multiple of 128")
    T, C = shape[0], shape[1] * 2
    if scale.dtype != torch.int32 or scale.shape != (C // 128, T):
        raise RuntimeError(f"{name} scale must be int32 {(C // 128, T)}")
    return T, C


def _no_grad(*ts: torch.Tensor | None) -> None:
    """Refuses tensors that autograd would follow, backward or forward: these ops write into given tensors and have no
    derivative. (Forward mode does not end with torch.no_grad().)"""
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                raise RuntimeError("this op has no backward: call it under torch.no_grad() or detach its tensors")
    if forward_ad._current_level >= 0:
        for t in ts:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("this op has no derivative in forward mode: give it tensors without a tangent")


def quant_mx4(x: torch.Tensor, out: torch.Tensor, scale: torch.Tensor, rotate: bool = True, norm: int = NORM_NONE,
              gamma: torch.Tensor | None = None, beta: torch.Tensor | None = None, c_real: int = 0,
              eps: float = 1e-6) -> None:
    """x fp16 or bf16 [T, C] (C % 128 == 0; any row stride from C up that is a multiple of 8) -> MX4: out uint8 [T, C / 2],
    scale int32 [C / 128, T] (include/foidfinder_rocm.h, ff_quant_mx4). First the norm over the first c_real columns
    (default: all) with gamma, and beta for NORM_LAYER, fp32 [C] with zeros past c_real (`pad_norm` builds them); then with
    `rotate` the rotation by blockdiag(H128). Weights are prepared by the same call: rows [N, K], no norm. The outputs share no memory
    with each other or with what is read (refused)."""
    _no_grad(x, gamma, beta)
    dev = _on_gpu(out, scale, gamma, beta)
    T, C = _mx4(out, scale, "out")
    if x.get_device() != dev or x.shape != (T, C) or x.dtype not in _HALVES:
        raise RuntimeError(f"x must be fp16 or bf16 {(T, C)} on the outputs' GPU")
    stride, one = x.stride()
    _require(one == 1, "x must have contiguous rows")
    if gamma is not None:
        _float(C, gamma)
    if beta is not None:
        _float(C, beta)
    if T <= 1:
        stride = C  # a single row's stride says nothing
    _run("ff_quant_mx4", dev, x.data_ptr(), _DTYPES[x.dtype], T, C, stride, rotate, norm, c_real or C, _ptr(gamma),
         _ptr(beta), eps, out.data_ptr(), scale.data_ptr())


def dequant_mx4(codes: torch.Tensor, scale: torch.Tensor, out: torch.Tensor) -> None:
    """The values of MX4 codes into out [T, C], fp16, bf16 or fp32, in memory of its own (ff_dequant_mx4)."""
    _no_grad(out)
    dev = _on_gpu(codes, scale, out)
    T, C = _mx4(codes, scale, "the")
    if out.dtype not in _DTYPES or out.shape != (T, C):
        raise RuntimeError(f"out must be fp16, bf16 or fp32 {(T, C)}")
    _run("ff_dequant_mx4", dev, codes.data_ptr(), scale.data_ptr(), T, C, out.data_ptr(), _DTYPES[out.dtype])


def gemm_mx4(A: torch.Tensor, a_scale: torch.Tensor, W: torch.Tensor, w_scale: torch.Tensor, bias: torch.Tensor | None,
             out: torch.Tensor, epi: int, stages: int = 0, residual: torch.Tensor | None = None) -> None:
    """MX4 A [M, K] x MX4 W [N, K] + bias fp32 [N] (or None) -> epilogue into out: EPI_BIAS_F16 (out fp16, bf16 or fp32),
    EPI_GELU_F16, EPI_SWIGLU (out [M, N / 2]) or EPI_RESIDUAL (out = y + residual of out's type, which is out itself (None)
    or memory apart from it). out shares no memory with the other operands (refused). `stages` selects the tile variant (0 = by the sizes) (ff_gemm_mx4)."""
    _no_grad(bias, out, residual)
    dev = _on_gpu(A, a_scale, W, w_scale, bias, out, residual)
    M, K = _mx4(A, a_scale, "A's")
    N, KW = _mx4(W, w_scale, "W's")
    _require(KW == K, "A and W must share K")
    shape = out_shape(M, N, epi)
    if out.dtype not in _DTYPES or out.shape != shape:
        raise RuntimeError(f"out must be fp16, bf16 or fp32 {shape}")
    if bias is not None:
        _float(N, bias)
    if epi == EPI_RESIDUAL:
        residual = out if residual is None else residual
        _require(residual.dtype == out.dtype and residual.shape == out.shape, "residual must be like out")
    else:
        _require(residual is None, "a residual goes with EPI_RESIDUAL")
    _run("ff_gemm_mx4", dev, A.data_ptr(), a_scale.data_ptr(), W.data_ptr(), w_scale.data_ptr(), M, N, K, _ptr(bias),
         _ptr(residual), out.data_ptr(), _DTYPES[out.dtype], epi, stages)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_out: torch.Tensor, k_out: torch.Tensor, norm: int,
                 q_gamma: torch.Tensor | None, k_gamma: torch.Tensor | None, q_beta: torch.Tensor | None,
                 k_beta: torch.Tensor | None, rope_cos: torch.Tensor, rope_sin: torch.Tensor,
                 positions: torch.Tensor | None = None, pairs: bool = True, eps: float = 1e-6,
                 q_scale: float = 1.0) -> None:
    """Norm of each head's query and key and their rotation by position in one pass (include/foidfinder_rocm.h,
    ff_qk_norm_rope): q fp16 or bf16 [T, heads, D], k [T, kv_heads, D], views with any token and head strides (of a packed
    [T, 3 C] row, say: `qkv.view(T, 3, heads, D)[:, 0]`) -> q_out, k_out of the same shapes; an output may be its input
    itself and shares no other memory with what is read or with the other (refused). gamma (with a norm) and beta (NORM_LAYER) fp32 [D]; tables fp32 [L, R / 2];
    positions int32 or int64 [T], or None: t % L. `pairs`: columns (2 i, 2 i + 1) turn together, else (i, i + R / 2)."""
    _no_grad(q, k, q_out, k_out, q_gamma, k_gamma, q_beta, k_beta, rope_cos, rope_sin)
    dev = _on_gpu(q_gamma, k_gamma, q_beta, k_beta, rope_cos, rope_sin, positions)
    shape, k_shape, dt = q.shape, k.shape, q.dtype
    if len(shape) != 3 or len(k_shape) != 3:
        raise RuntimeError("q and k must be [T, heads, D]")
    (T, H, D), (TK, KV, DK) = shape, k_shape
    if TK != T or DK != D:
        raise RuntimeError("q and k must share T and D")
    if not (dt in _HALVES and k.dtype == q_out.dtype == k_out.dtype == dt):
        raise RuntimeError("q, k, q_out and k_out must be fp16 or bf16, of one type")
    if q_out.shape != shape or k_out.shape != k_shape:
        raise RuntimeError("q_out and k_out must have the shapes of q and k")
    if not (q.get_device() == k.get_device() == q_out.get_device() == k_out.get_device() == dev):
        raise RuntimeError("all tensors must be on one device")
    (qt, qh, q1), (kt, kh, k1), (ot, oh, o1), (pt, ph, p1) = q.stride(), k.stride(), q_out.stride(), k_out.stride()
    if not q1 == k1 == o1 == p1 == 1:
        raise RuntimeError("q, k, q_out and k_out must have contiguous columns")
    if T <= 1:  # a dimension of one has no stride
        qt = kt = ot = pt = 0
    if H == 1:
        qh = oh = 0
    if KV == 1:
        kh = ph = 0
    qp, kp, op, pp = q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr()
    if T and ((qp == op and (qt, qh) != (ot, oh)) or (kp == pp and (kt, kh) != (pt, ph))):
        raise RuntimeError("an output in its input's place must have its strides")
    table = rope_cos.shape
    if not (rope_cos.dtype == rope_sin.dtype == torch.float32 and len(table) == 2 and rope_sin.shape == table):
        raise RuntimeError("RoPE tables must be fp32 [L, R / 2]")
    _float(D, *[t for t in (q_gamma, k_gamma, q_beta, k_beta) if t is not None])
    pos64 = False
    if positions is not None:
        pos64 = positions.dtype == torch.int64
        if not (pos64 or positions.dtype == torch.int32) or positions.shape != (T,):
            raise RuntimeError(f"positions must be int32 or int64 [{T}]")
    L, half = table
    _run("ff_qk_norm_rope", dev, qp, qt, qh, kp, kt, kh, op, ot, oh, pp, pt, ph, _DTYPES[dt], T, H, KV, D, norm,
         _ptr(q_gamma), _ptr(k_gamma), _ptr(q_beta), _ptr(k_beta), eps, rope_cos.data_ptr(), rope_sin.data_ptr(), L,
         2 * half, pairs, _ptr(positions), pos64, q_scale)


def _attended(q: torch.Tensor, out: torch.Tensor, lens: torch.Tensor | None, work: torch.Tensor | None,
              *kv: torch.Tensor) -> int:
    """The device of an attention's tensors, which agree in type, device and head width; the last two are keys and values
    [B, S, kv_heads, D] of q's batch."""
    shape, dt, dev = q.shape, q.dtype, q.get_device()
    if dev < 0:
        raise RuntimeError("foidfinder_rocm ops take GPU tensors")
    if len(shape) != 4 or dt not in _HALVES or out.dtype != dt or out.shape != shape or out.get_device() != dev:
        raise RuntimeError("q and out must be fp16 or bf16 [B, L, heads, D], of one type and shape on one device")
    for t in kv:
        if t.dtype != dt or t.get_device() != dev:
            raise RuntimeError("keys and values must have q's type and device")
    B, _, _, D = shape
    kshape = kv[-2].shape
    if len(kshape) != 4 or kshape[0] != B or kshape[3] != D or kv[-1].shape != kshape:
        raise RuntimeError("keys and values must be [B, S, kv_heads, D] with q's B and D, and of one shape")
    if lens is not None and (lens.dtype != torch.int32 or lens.shape != (B,) or lens.get_device() != dev
                             or not lens.is_contiguous()):
        raise RuntimeError(f"lens must be contiguous int32 {(B,)} on the queries' GPU")
    if work is not None and (work.dtype != torch.float32 or work.get_device() != dev or not work.is_contiguous()):
        raise RuntimeError("work must be contiguous fp32 on the queries' GPU")
    return dev


def _columns(ones: tuple, *ts: torch.Tensor) -> None:
    """Refuses rows with a column stride other than 1 (no rows, no stride)."""
    for one, t in zip(ones, ts):
        if one != 1 and t.numel():
            raise RuntimeError("q, keys, values and out must have contiguous columns")


def cross_attention_work(q: torch.Tensor, k: torch.Tensor) -> int:
    """fp32 elements of the workspace that cross_attention takes for queries and keys of these shapes (0: none)."""
    B, L, H, D = q.shape
    return lib().ff_cross_attention_work(B, L, k.size(1), H, k.size(2), D)


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, scale: float,
                    lens: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                    work: torch.Tensor | None = None) -> None:
    """Attention of q [B, L, heads, D] to keys and values [B, S, kv_heads, D] of another length into out, fp16 or bf16 with
    fp32 sums (include/foidfinder_rocm.h, ff_cross_attention): any batch, token and head strides that are multiples of 16
    bytes (views of packed rows, [B, heads, L, D] transposed, rows expanded over the batch), D a multiple of 8 up to 128,
    heads a multiple of kv_heads. Keys j >= lens[b] (int32 [B]) and keys with mask[b, j] False (bool [B, S], contiguous
    columns) are not read; a query without keys gives zeros, one with a score of +inf, or of -inf alone, is not a number.
    work: fp32 of at least cross_attention_work(q, k) elements; calls that run one after another may share it. out and work
    share no memory with each other or with what is read (refused)."""
    _no_grad(q, k, v, out, work)
    dev = _attended(q, out, lens, work, k, v)
    (qb, qt, qh, q1), (kb, kt, kh, k1), (vb, vt, vh, v1), (ob, ot, oh, o1) = q.stride(), k.stride(), v.stride(), out.stride()
    if not q1 == k1 == v1 == o1 == 1:
        _columns((q1, k1, v1, o1), q, k, v, out)
    (B, L, H, D), (_, S, KV, _) = q.shape, k.shape
    mp, mb = None, 0
    if mask is not None:
        if mask.dtype != torch.bool or mask.shape != (B, S) or mask.get_device() != dev:
            raise RuntimeError(f"mask must be bool {(B, S)} on the queries' GPU")
        mb, one = mask.stride()
        if one != 1 and S > 1:
            raise RuntimeError("mask must have contiguous columns")
        mp = mask.data_ptr()
    _run("ff_cross_attention", dev, q.data_ptr(), qb, qt, qh, k.data_ptr(), kb, kt, kh, v.data_ptr(), vb, vt, vh,
         out.data_ptr(), ob, ot, oh, _DTYPES[q.dtype], B, L, S, H, KV, D, scale, None if lens is None else lens.data_ptr(), mp,
         mb, None if work is None else work.data_ptr(), 0 if work is None else work.numel())


def prefix_attention_work(q: torch.Tensor, prefix_k: torch.Tensor, k: torch.Tensor) -> int:
    """fp32 elements of the workspace that prefix_attention takes for tensors of these shapes (0: none)."""
    B, L, H, D = q.shape
    return lib().ff_prefix_attention_work(B, L, prefix_k.size(0), k.size(1), H, k.size(2), D)


def prefix_attention(q: torch.Tensor, prefix_k: torch.Tensor, prefix_v: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                     out: torch.Tensor, scale: float, lens: torch.Tensor | None = None,
                     work: torch.Tensor | None = None) -> None:
    """Attention of a batch that shares a prefix (include/foidfinder_rocm.h, ff_prefix_attention): q [B, L, heads, D] are each
    sequence's newest L tokens, prefix_k and prefix_v [P, kv_heads, D] the rows that all sequences see, read once for all of them,
    k and v [B, S, kv_heads, D] each sequence's own behind them, lens[b] of them (int32 [B]; None: S) with the new tokens' own
    last. Query i sees the prefix and the own keys j < lens[b] - L + 1 + i, and nothing of later ones, whatever they hold.
    Types, strides and work (at least prefix_attention_work(q, prefix_k, k) elements) as in cross_attention."""
    _no_grad(q, prefix_k, prefix_v, k, v, out, work)
    dev = _attended(q, out, lens, work, prefix_k, prefix_v, k, v)
    (qb, qt, qh, q1), (kb, kt, kh, k1), (vb, vt, vh, v1), (ob, ot, oh, o1) = q.stride(), k.stride(), v.stride(), out.stride()
    if not q1 == k1 == v1 == o1 == 1:
        _columns((q1, k1, v1, o1), q, k, v, out)
    (B, L, H, D), (_, S, KV, _), pshape = q.shape, k.shape, prefix_k.shape
    if len(pshape) != 3 or pshape[1] != KV or pshape[2] != D or prefix_v.shape != pshape:
        raise RuntimeError("prefix_k and prefix_v must be [P, kv_heads, D], of one shape")
    (pkt, pkh, pk1), (pvt, pvh, pv1) = prefix_k.stride(), prefix_v.stride()
    if not pk1 == pv1 == 1:
        _columns((pk1, pv1), prefix_k, prefix_v)
    _run("ff_prefix_attention", dev, q.data_ptr(), qb, qt, qh, prefix_k.data_ptr(), pkt, pkh, prefix_v.data_ptr(), pvt, pvh,
         k.data_ptr(), kb, kt, kh, v.data_ptr(), vb, vt, vh, out.data_ptr(), ob, ot, oh, _DTYPES[q.dtype], B, L, pshape[0], S,
         H, KV, D, scale, None if lens is None else lens.data_ptr(), None if work is None else work.data_ptr(),
         0 if work is None else work.numel())


def residual_norm(x: torch.Tensor, y: torch.Tensor, x_out: torch.Tensor, h: torch.Tensor | None, post: int,
                  post_gamma: torch.Tensor | None, post_beta: torch.Tensor | None, pre: int,
                  pre_gamma: torch.Tensor | None, pre_beta: torch.Tensor | None, gate: torch.Tensor | None = None,
                  scale: float = 1.0, eps: float = 1e-6) -> None:
    """A block's output into the residual stream between two norms (include/foidfinder_rocm.h, ff_residual_norm): x_out =
    x + scale * gate * N_post(y) and h = N_pre(x_out) in one pass, h from the unrounded sum. x, y, x_out, h fp16 or bf16 [T, C]
    with contiguous rows (any row stride that is a multiple of 8), C a multiple of 8 up to 16384; h only with a pre-norm (None
    otherwise); gammas and betas fp32 [C] as the norms (NORM_*) need them; gate [G, C] or [C], fp32 or of x's type, token t
    taking row t / (T / G): one row is a layer scale, one a sequence an adaptive gate. An output may be x or y itself and shares
    no other memory with what is read or with the other (refused)."""
    _no_grad(x, y, x_out, h, post_gamma, post_beta, pre_gamma, pre_beta, gate)
    shape, dt, dev = x.shape, x.dtype, x.get_device()
    if len(shape) != 2 or dt not in _HALVES:
        raise RuntimeError("x must be fp16 or bf16 [T, C]")
    if not (y.shape == x_out.shape == shape and y.dtype == x_out.dtype == dt):
        raise RuntimeError("x, y and the outputs must have one type and shape")
    if dev < 0 or y.get_device() != dev or x_out.get_device() != dev:
        raise RuntimeError("all tensors must be on one GPU")
    T, C = shape
    (xs, x1), (ys, y1), (os, o1) = x.stride(), y.stride(), x_out.stride()
    hp, hs, h1 = None, C, 1
    if h is not None:
        if h.shape != shape or h.dtype != dt or h.get_device() != dev:
            raise RuntimeError("h must have x's type, shape and device")
        hp, (hs, h1) = h.data_ptr(), h.stride()
    if not x1 == y1 == o1 == h1 == 1 and T:
        raise RuntimeError("x, y and the outputs must have contiguous rows")
    params = []
    for p in (post_gamma, post_beta, pre_gamma, pre_beta):
        if p is None:
            params.append(None)
            continue
        if p.dtype != torch.float32 or p.numel() != C or p.get_device() != dev or not p.is_contiguous():
            raise RuntimeError(f"gammas and betas must be contiguous fp32 of {C} elements on x's GPU")
        params.append(p.data_ptr())
    gp, gates, kind = None, 0, 0
    if gate is not None:
        if gate.dtype not in (dt, torch.float32) or gate.dim() not in (1, 2) or gate.size(-1) != C or T and not gate.numel():
            raise RuntimeError("gate must be fp32 or of x's type, [G, C] or [C]")
        if gate.get_device() != dev or not gate.is_contiguous():
            raise RuntimeError("gate must be contiguous on x's GPU")
        gp, gates, kind = gate.data_ptr(), gate.numel() // C, _DTYPES[gate.dtype]
    pg, pb, qg, qb = params
    _run("ff_residual_norm", dev, x.data_ptr(), xs, y.data_ptr(), ys, x_out.data_ptr(), os, hp, hs, _DTYPES[dt], T, C, post, pg,
         pb, pre, qg, qb, gp, gates, kind, scale, eps)


# ---- torch.ops.foidfinder_rocm registration (schemas as kernels.cu:268-273, plus eps / the fused norm) ----

_LIB = torch.library.Library("foidfinder_rocm", "DEF")
_LIB.define(
    "gemm_s8(Tensor A, Tensor W, Tensor row_scale, Tensor col_scale, Tensor bias, Tensor(a!) out, int epi, "
    "int stages, Tensor? rope_cos, Tensor? rope_sin, float q_scale) -> ()"
)
_LIB.define("rot_q8_1024(Tensor x, Tensor? gamma, Tensor? beta, Tensor(a!) out, Tensor(b!) row_scale, "
            "float eps=1e-05) -> ()")
_LIB.define("rot_q8_h128(Tensor x, Tensor(a!) out, Tensor(b!) row_scale, Tensor? gamma=None, Tensor? beta=None, "
            "int c_real=0, float eps=1e-06) -> ()")
_LIB.define("attention(Tensor qkv, Tensor(a!) out, int seq_len) -> ()")
_LIB.impl("gemm_s8", gemm_s8, "CUDA")
_LIB.impl("rot_q8_1024", rot_q8_1024, "CUDA")
_LIB.impl("rot_q8_h128", rot_q8_h128, "CUDA")
_LIB.impl("attention", attention, "CUDA")
# Haruka's tree pool (no reference CUDA op; out-param ops in the same style)
_LIB.define("layer_norm2(Tensor x, Tensor g1, Tensor b1, Tensor g2, Tensor b2, float eps, Tensor(a!) out) -> ()")
_LIB.define("slot_weights(Tensor logits, Tensor c, Tensor bias, int heads, Tensor(a!) a_t, Tensor(b!) partial) -> ()")
_LIB.define("pool_weights(Tensor xn, Tensor u, Tensor c, Tensor bias, int heads, Tensor(a!) a_t, Tensor(b!) partial) "
            "-> ()")
_LIB.define("pool_sum(Tensor a_t, Tensor xn, Tensor(a!) pooled) -> ()")
_LIB.define("pool_values(Tensor pooled, Tensor wv, Tensor bv, Tensor partial, int heads, Tensor(a!) z) -> ()")
_LIB.define("pool_queries(Tensor z, Tensor trunk_g, Tensor trunk_b, Tensor child, Tensor child_g, Tensor child_b, "
            "Tensor bk, int heads, float eps, Tensor(a!) parent, Tensor(b!) qleaf, Tensor(c!) cq) -> ()")
_LIB.define("pool_keys(Tensor qleaf, Tensor kT, Tensor(a!) u) -> ()")
_LIB.define("pool_tree(Tensor parent, Tensor zc, Tensor g, Tensor b, Tensor partial, int heads, float eps, "
            "Tensor(a!) tree) -> ()")
_LIB.define("pool_leaf(Tensor tree, Tensor wl, Tensor bl, Tensor(a!) leaf) -> ()")
_LIB.define("patch_embed(Tensor img, Tensor w, Tensor bias_pos, Tensor cls, Tensor(a!) x) -> ()")
_LIB.define("head(Tensor x, Tensor W, Tensor bias, Tensor(a!) out, Tensor? gamma=None, Tensor? beta=None, "
            "float eps=1e-06) -> ()")
for _fn in (pool_weights, pool_sum, pool_values, pool_queries, pool_keys, pool_tree, pool_leaf, patch_embed, head):
    _LIB.impl(_fn.__name__, _fn, "CUDA")
_LIB.impl("layer_norm2", layer_norm2, "CUDA")
# the MX4 linear and the norm of queries and keys (no reference counterpart; out-param ops in the same style)
_LIB.define("quant_mx4(Tensor x, Tensor(a!) out, Tensor(b!) scale, bool rotate=True, int norm=0, Tensor? gamma=None, "
            "Tensor? beta=None, int c_real=0, float eps=1e-06) -> ()")
_LIB.define("dequant_mx4(Tensor codes, Tensor scale, Tensor(a!) out) -> ()")
_LIB.define("gemm_mx4(Tensor A, Tensor a_scale, Tensor W, Tensor w_scale, Tensor? bias, Tensor(a!) out, int epi, "
            "int stages=0, Tensor? residual=None) -> ()")
_LIB.define("qk_norm_rope(Tensor q, Tensor k, Tensor(a!) q_out, Tensor(b!) k_out, int norm, Tensor? q_gamma, "
            "Tensor? k_gamma, Tensor? q_beta, Tensor? k_beta, Tensor rope_cos, Tensor rope_sin, Tensor? positions=None, "
            "bool pairs=True, float eps=1e-06, float q_scale=1.0) -> ()")
for _fn in (quant_mx4, dequant_mx4, gemm_mx4, qk_norm_rope):
    _LIB.impl(_fn.__name__, _fn, "CUDA")
# the decoder side: attention to other rows and the residual stream between two norms (no reference counterpart)
_LIB.define("cross_attention(Tensor q, Tensor k, Tensor v, Tensor(a!) out, float scale, Tensor? lens=None, "
            "Tensor? mask=None, Tensor(b!)? work=None) -> ()")
_LIB.define("prefix_attention(Tensor q, Tensor prefix_k, Tensor prefix_v, Tensor k, Tensor v, Tensor(a!) out, float scale, "
            "Tensor? lens=None, Tensor(b!)? work=None) -> ()")
_LIB.define("residual_norm(Tensor x, Tensor y, Tensor(a!) x_out, Tensor(b!)? h, int post, Tensor? post_gamma, "
            "Tensor? post_beta, int pre, Tensor? pre_gamma, Tensor? pre_beta, Tensor? gate=None, float scale=1.0, "
            "float eps=1e-06) -> ()")
for _fn in (cross_attention, prefix_attention, residual_norm):
    _LIB.impl(_fn.__name__, _fn, "CUDA")
_LIB.impl("slot_weights", slot_weights, "CUDA")


@cache
def kernels():
    """The op namespace, loading the library (raises if it is missing). Mirrors the reference's `kernels()`."""
    lib()
    return torch.ops.foidfinder_rocm
