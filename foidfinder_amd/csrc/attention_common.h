// What the attention kernels share (attention.hip, cross_attention.hip).
#pragma once

#include "common.h"

namespace ff {

// ds_read_b64_tr_b16 as inline asm. The compiler's wait-insertion pass treats the builtin as possibly reading LDS
// that in-flight buffer->LDS loads are writing and drains them all (s_waitcnt vmcnt(0)) before it, which would
// serialize the LDS ring; this form is invisible to that pass. Ordering: "memory" keeps it after the barrier that
// publishes the tile; the caller waits for the data (s_waitcnt lgkmcnt(0) tied to the result registers).
template <int OFF, typename V>
__device__ __forceinline__ void tr_read(V& v, uint32_t lds_addr) {
  static_assert(sizeof(V) == 8, "four 16-bit values");
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(v) : "v"(lds_addr), "n"(OFF) : "memory");
}

}  // namespace ff
