// What the Walsh-Hadamard rotations share (rotq8.hip, quant_mx4.hip). The cross-lane butterflies: lane l of a 16-lane DPP row owns
// column chunk gray(l) = l ^ (l >> 1), so the partners for chunk bits 0..3 are lanes l ^ 1, ^ 3, ^ 7, ^ 15.
#pragma once

#include "common.h"

namespace ff {

// Sign-tracked butterfly across lanes, u = fma(p, s, u) with partner p, own u, s = +1 (column bit 0) or -1 (column
// bit 1), as one v_fmac_f32_dpp (DPP on the multiplicand: the partner's u). The compiler only emits it as
// v_mov_b32_dpp + v_fmac_f32, so it is written out; one stage is one call over all of a lane's values, which are
// distinct registers, so the only VALU-write -> DPP-read hazard (2 wait states) is with whatever wrote them before
// the stage: the leading s_nop covers it. DPP controls: l^1 quad_perm [1,0,3,2], l^3 quad_perm [3,2,1,0], l^7
// row_half_mirror, l^15 row_mirror (all partners are inside the 16-lane DPP row, so bound_ctrl never applies).
#define FF_FMAC_DPP(CTL) "v_fmac_f32_dpp %0, %0, %1 " CTL " row_mask:0xf bank_mask:0xf bound_ctrl:1"
template <int CTRL, int N>
__device__ __forceinline__ void bfly_stage(float (&v)[N], float s) {
  asm volatile("s_nop 1" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (CTRL == DPP_XOR1)
      asm volatile(FF_FMAC_DPP("quad_perm:[1,0,3,2]") : "+v"(v[i]) : "v"(s));
    else if constexpr (CTRL == DPP_XOR3)
      asm volatile(FF_FMAC_DPP("quad_perm:[3,2,1,0]") : "+v"(v[i]) : "v"(s));
    else if constexpr (CTRL == DPP_XOR7)
      asm volatile(FF_FMAC_DPP("row_half_mirror") : "+v"(v[i]) : "v"(s));
    else
      asm volatile(FF_FMAC_DPP("row_mirror") : "+v"(v[i]) : "v"(s));
  }
}

__device__ __forceinline__ float gray_sign(int bit) { return bit ? -1.f : 1.f; }

// An fp16 value folded into its first fp32 operation with v_fma_mix_f32, whose f16 source converts exactly and whose result
// rounds once, so it equals the fp32 addition of the converted value: half HI of h2 plus s.
template <int HI>
__device__ __forceinline__ float add_h(uint32_t h2, float s) {
  float r;
  if constexpr (HI)
    asm("v_fma_mix_f32 %0, %1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h2), "v"(s));
  else
    asm("v_fma_mix_f32 %0, %1, 1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h2), "v"(s));
  return r;
}

}  // namespace ff
