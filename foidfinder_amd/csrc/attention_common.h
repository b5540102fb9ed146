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

// Four reads STEP bytes apart, of one address or of two, and the wait for them in one block.
template <int OFF, int STEP, typename V>
__device__ __forceinline__ void tr_read4(V (&x)[4], uint32_t at) {
  static_assert(sizeof(V) == 8, "four 16-bit values");
  asm volatile(
      "ds_read_b64_tr_b16 %0, %4 offset:%5\n\t"
      "ds_read_b64_tr_b16 %1, %4 offset:%6\n\t"
      "ds_read_b64_tr_b16 %2, %4 offset:%7\n\t"
      "ds_read_b64_tr_b16 %3, %4 offset:%8\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3])
      : "v"(at), "n"(OFF), "n"(OFF + STEP), "n"(OFF + 2 * STEP), "n"(OFF + 3 * STEP)
      : "memory");
}
template <int OFF, int STEP, typename V>
__device__ __forceinline__ void tr_read4(V (&x)[4], uint32_t at, V (&y)[4], uint32_t to) {
  static_assert(sizeof(V) == 8, "four 16-bit values");
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8 offset:%10\n\t"
      "ds_read_b64_tr_b16 %4, %9 offset:%10\n\t"
      "ds_read_b64_tr_b16 %1, %8 offset:%11\n\t"
      "ds_read_b64_tr_b16 %5, %9 offset:%11\n\t"
      "ds_read_b64_tr_b16 %2, %8 offset:%12\n\t"
      "ds_read_b64_tr_b16 %6, %9 offset:%12\n\t"
      "ds_read_b64_tr_b16 %3, %8 offset:%13\n\t"
      "ds_read_b64_tr_b16 %7, %9 offset:%13\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(y[0]), "=&v"(y[1]), "=&v"(y[2]), "=&v"(y[3])
      : "v"(at), "v"(to), "n"(OFF), "n"(OFF + STEP), "n"(OFF + 2 * STEP), "n"(OFF + 3 * STEP)
      : "memory");
}

}  // namespace ff
