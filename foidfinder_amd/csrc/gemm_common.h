// What the matrix products share (gemm_s8.hip, gemm_mx4.hip): buffer accesses with a range and the activations of the
// epilogues.
#pragma once

#include "common.h"

namespace ff {

constexpr uint32_t RSRC_WORD3 = 0x00020000;  // buffer descriptor word 3: raw dword access (gfx9 family)

// Raw buffer loads and stores through a descriptor over [base, base + nbytes): an access past the range reads zeros
// or is dropped, so bounds need no clamped addresses or branches, and the 32-bit lane offset plus a scalar base
// replaces 64-bit address arithmetic per access. Plain functions, so the descriptor type never appears in a
// template-dependent expression (the host pass of a template drops its kernel stubs otherwise). An offset of
// OOB_OFFSET is always out of range (nbytes <= INT32_MAX).
constexpr uint32_t OOB_OFFSET = 0x80000000u;
__device__ __forceinline__ int buf_bytes(int64_t bytes) {
  return static_cast<int>(bytes < 0 ? 0 : (bytes < 0x7fffffff ? bytes : 0x7fffffff));
}
__device__ __forceinline__ float4_t buf_load_f4(const void* base, int nbytes, uint32_t voff) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, nbytes, RSRC_WORD3);
  return __builtin_bit_cast(float4_t, __builtin_amdgcn_raw_buffer_load_b128(r, voff, 0, 0));
}
__device__ __forceinline__ float buf_load_f1(const void* base, int nbytes, uint32_t voff) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, nbytes, RSRC_WORD3);
  return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, voff, 0, 0));
}
__device__ __forceinline__ half8_t buf_load_h8(const void* base, int nbytes, uint32_t voff) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, nbytes, RSRC_WORD3);
  return __builtin_bit_cast(half8_t, __builtin_amdgcn_raw_buffer_load_b128(r, voff, 0, 0));
}
__device__ __forceinline__ void buf_store_h8(half8_t v, void* base, int nbytes, uint32_t voff) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(base, 0, nbytes, RSRC_WORD3);
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(int4_t, v), r, voff, 0, 0);
}

// silu(g) = g / (1 + e^-g) from the hardware transcendental units: e^-g = v_exp_f32(-g log2 e) and the quotient as
// g * v_rcp_f32(1 + e^-g), each about 1 ulp, so silu(g) * value lands within one fp16 ulp of the correctly rounded
// result (the reference's own exp is a platform library call, mlx/kernels.py:45-49). Limits: g -> -inf gives
// e^-g = inf, rcp = 0, silu = -0; g -> +inf gives g.
__device__ __forceinline__ float silu(float g) {
  const float e = __builtin_amdgcn_exp2f(-g * 1.44269504088896341f);
  return g * __builtin_amdgcn_rcpf(1.f + e);
}

// The tanh GELU 0.5 y (1 + tanh(u)), u = sqrt(2/pi) (y + 0.044715 y^3), in the exactly equal form y / (1 + e^(-2u)),
// from the hardware exp2 and reciprocal (each about 1 ulp): within a few fp32 ulp of the exact value for every y (the
// form 0.5 y (1 + tanh(u)) cancels for negative y), where the reference itself evaluates tanh with a hardware
// approximation (common.cuh:50-56); ~8 instructions instead of a library tanhf with branches. Limits: y -> -inf
// gives e^(-2u) = inf, rcp = 0, gelu = -0; y -> +inf gives y.
__device__ __forceinline__ float gelu_tanh(float y) {
  constexpr float K1 = -2.f * 1.4426950408889634f * 0.7978845608f;  // -2 sqrt(2/pi) log2(e)
  constexpr float K3 = K1 * 0.044715f;
  const float t = __builtin_fmaf(K3, y * y, K1) * y;  // -2u log2(e)
  return y * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(t));
}

typedef __attribute__((address_space(3))) void lds_void;

// One 16-byte-per-lane buffer load into LDS through a raw descriptor of `nbytes` bytes at `base` (loads past it read
// zeros). A plain function, so the descriptor type never appears in a template-dependent expression: the host pass
// of HIP cannot instantiate those and would silently drop the kernel's launch stub.
__device__ __forceinline__ void buffer_to_lds(const void* base, int nbytes, uint8_t* lds_dst, uint32_t voff) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, nbytes, RSRC_WORD3);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)lds_dst, 16, voff, 0, 0, 0);
}

}  // namespace ff
