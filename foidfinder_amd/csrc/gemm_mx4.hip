// The product of two MX4 matrices (quant_mx4.hip) on gfx950's scaled MFMA, with the epilogue fused.
//
// y[m, n] = sum over blocks b of 32 columns of 2^(ea[m, b] + ew[n, b]) sum_k a[m, k] w[n, k], + bias[n], in fp32: the
// products of two E2M1 codes are exact, and v_mfma_scale_f32_32x32x64_f8f6f4 applies both exponents to its 32-column
// partial sums. The instruction does 64 columns of K in the time that int8's 32x32x32 does 32, from the same 16 bytes a
// lane and operand.
//
// K is walked in units of 128 columns: 64 bytes of codes and one 32-bit word of exponents a row. Which columns go into
// which k slot of the MFMA is free as long as both operands agree, so lane half h of step s takes the block 2 h + s of the
// unit: its 32 bytes of a unit are contiguous, and its exponents are the bytes 2 h and 2 h + 1 of the row's word.
//
// The product is computed transposed (W is the row operand), so that a lane holds one output row m and runs of four
// consecutive columns n: column pairs (SwiGLU) are in-lane and stores are whole runs.
//
// Five tile shapes, by an estimate of their times (pick_variant). 32 x 32 blocks with K over the four waves and fragments
// straight from memory serve few rows and few columns: one row x 2304 x 768 takes 3.9 us. 64 x 64 tiles serve what leaves
// CUs idle otherwise: 1025 x 1024 x 2816 with a residual 7.6 us (272 tiles, 22 units each: neither more slots nor K on two
// groups of waves is faster); 16 x 98 782 x 1152 14 us, 4.8 TB/s, the weights' bytes. 128 x 128, 256 x 128 and 256 x 256
// tiles read each operand less often: 5184 x 4736 x 1024 GELU 25-26 us (1.9-2.0 PFLOP/s with 49 MB of stores), 32 800 x
// 5632 x 1024 SwiGLU 131-140 us (2.7-2.9 PFLOP/s), 32 768 x 4096 x 4096 282 us (3.9 PFLOP/s). The instruction alone reaches
// 6.1 PFLOP/s on random codes (8.5 on zeros: power). At K = 1024 the products take 82 of 131 us, the ring's loads add 23 and
// the epilogue 25: a tile's parts run in turn, the MFMAs busy 35 % of the time, at a clock that falls with their share (1.93
// GHz; 1.66 at the 53 % of 32 768 x 4096 x 4096). Measured and not kept: W as a stream past persistent waves for few rows (16.8
// us against 14), workgroups whose ring runs on across tiles (132-134 us against 132-136, spills with a residual, slower for
// few tiles; their epilogue still stood between two tiles' products), slots of two units for the large tiles, loads spread
// between the products.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.h"
#include "gemm_common.h"

namespace ff {

struct Mx4Args {
  const uint8_t* A;        // codes [M, K / 2]
  const uint32_t* a_scale; // [K / 128, M]
  const uint8_t* W;        // codes [N, K / 2]
  const uint32_t* w_scale; // [K / 128, N]
  int M, N, K;
  const float* bias;     // [N] or null
  const void* residual;  // [M, N], RESIDUAL
  void* out;             // [M, N], [M, N / 2] for SWIGLU
};

__device__ __forceinline__ int4_t buf_load_i4(const void* base, int nbytes, uint32_t voff) {
  return __builtin_bit_cast(int4_t, buf_load_f4(base, nbytes, voff));
}
__device__ __forceinline__ uint32_t buf_load_u32(const void* base, int nbytes, uint32_t voff) {
  return __builtin_bit_cast(uint32_t, buf_load_f1(base, nbytes, voff));
}

__device__ __forceinline__ uint16_t buf_load_u16(const void* base, int nbytes, uint32_t voff) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, nbytes, RSRC_WORD3);
  return __builtin_amdgcn_raw_buffer_load_b16(r, voff, 0, 0);
}
__device__ __forceinline__ void buf_store_u32(uint32_t v, void* base, int nbytes, uint32_t voff) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(base, 0, nbytes, RSRC_WORD3);
  __builtin_amdgcn_raw_buffer_store_b32(v, r, voff, 0, 0);
}
__device__ __forceinline__ void buf_store_u16(uint16_t v, void* base, int nbytes, uint32_t voff) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(base, 0, nbytes, RSRC_WORD3);
  __builtin_amdgcn_raw_buffer_store_b16(v, r, voff, 0, 0);
}

// A store that does not stay in L2 ahead of other lines: the outputs are larger than what the tiles read again (32800 x 5632 x
// 1024 SwiGLU 141 -> 134 us, 5184 x 4736 26.3 -> 25.8; what reads the output next is no slower).
__device__ __forceinline__ void buf_stream_i4(int4_t v, void* base, int nbytes, uint32_t voff) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(base, 0, nbytes, RSRC_WORD3);
  __builtin_amdgcn_raw_buffer_store_b128(v, r, voff, 0, 2);
}

// One lane's run (16, 4 or 2 bytes) through a descriptor.
template <typename R>
__device__ __forceinline__ R buf_load_run(const void* base, int nbytes, uint32_t voff) {
  if constexpr (sizeof(R) == 16)
    return __builtin_bit_cast(R, buf_load_f4(base, nbytes, voff));
  else if constexpr (sizeof(R) == 4)
    return __builtin_bit_cast(R, buf_load_f1(base, nbytes, voff));
  else
    return __builtin_bit_cast(R, buf_load_u16(base, nbytes, voff));
}
template <typename R>
__device__ __forceinline__ void buf_store_run(R v, void* base, int nbytes, uint32_t voff) {
  if constexpr (sizeof(R) == 16)
    buf_stream_i4(__builtin_bit_cast(int4_t, v), base, nbytes, voff);
  else if constexpr (sizeof(R) == 4)
    buf_store_u32(__builtin_bit_cast(uint32_t, v), base, nbytes, voff);
  else
    buf_store_u16(__builtin_bit_cast(uint16_t, v), base, nbytes, voff);
}

// D += W-fragment x A-fragment over 64 columns; S: the byte of the exponent words that holds this step's block.
template <int S>
__device__ __forceinline__ float16_t mfma_mx4(int4_t w, int4_t a, float16_t c, uint32_t ws, uint32_t as) {
  const int8_t_v wv = {w[0], w[1], w[2], w[3], 0, 0, 0, 0}, av = {a[0], a[1], a[2], a[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv, av, c, 4, 4, S, static_cast<int>(ws), S,
                                                         static_cast<int>(as));
}

// The epilogue of four consecutive columns n .. n + 3 of row m (n % 4 == 0, n < N): y holds the sums. One rounding, at the
// store. Columns past N are not touched; runs inside the row go at once where its start is 4-byte aligned.
template <int EPI, typename T>
__device__ __forceinline__ void finish4(const Mx4Args& args, int m, int n, float4_t y) {
  const int N = args.N;
  const bool inside = n + 4 <= N;
  if (args.bias) {
    if (inside) {
      const float4_t b = *reinterpret_cast<const float4_t*>(args.bias + n);
#pragma unroll
      for (int t = 0; t < 4; ++t) y[t] = y[t] + b[t];
    } else {
#pragma unroll
      for (int t = 0; t < 4; ++t) y[t] = y[t] + (n + t < N ? args.bias[n + t] : 0.f);
    }
  }
  if constexpr (EPI == FF_EPI_SWIGLU) {
    T* o = static_cast<T*>(args.out) + static_cast<int64_t>(m) * (N >> 1) + (n >> 1);
    const T h0 = static_cast<T>(silu(y[0]) * y[1]), h1 = static_cast<T>(silu(y[2]) * y[3]);
    o[0] = h0;
    if (n + 2 < N) o[1] = h1;  // N is even
  } else {
    const bool run = inside && (sizeof(T) == 4 || (N & 1) == 0);
    const int64_t at = static_cast<int64_t>(m) * N + n;
    T* o = static_cast<T*>(args.out) + at;
    if constexpr (EPI == FF_EPI_RESIDUAL) {
      const T* r = static_cast<const T*>(args.residual) + at;
      vec4_t<T> x = {};
      if (run) {
        __builtin_memcpy(&x, r, sizeof(x));
      } else {
#pragma unroll
        for (int t = 0; t < 4; ++t)
          if (n + t < N) x[t] = r[t];
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) y[t] = y[t] + static_cast<float>(x[t]);
    }
    if constexpr (EPI == FF_EPI_GELU_F16) {
#pragma unroll
      for (int t = 0; t < 4; ++t) y[t] = gelu_tanh(y[t]);
    }
    vec4_t<T> h;
#pragma unroll
    for (int t = 0; t < 4; ++t) h[t] = static_cast<T>(y[t]);
    if (run) {
      __builtin_memcpy(o, &h, sizeof(h));
    } else {
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (n + t < N) o[t] = h[t];
    }
  }
}

// ---------------- 32 x 32 blocks, K split over the four waves ----------------
//
// Few rows: the fragments come straight from global memory (no staging: a block's rows are read once), four units in flight
// a wave, and the waves' partial sums are added through LDS in a fixed order.
constexpr int SP_UNITS = 4;   // units a wave loads at once
constexpr int SP_ROW = 36;    // floats of a partial sum's row in LDS: 32 and a pad of one 16-byte store

template <int EPI, typename T>
__global__ __launch_bounds__(256) void gemm_mx4_split_kernel(const Mx4Args args) {
  __shared__ __attribute__((aligned(16))) float part[4 * 32 * SP_ROW];
  const int tid = threadIdx.x, lane = tid & 63, fr = lane & 31, fh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tiles_n = (args.N + 31) / 32;
  const int t = xcd_remap(blockIdx.x, gridDim.x);
  const int m0 = t / tiles_n * 32, n0 = t % tiles_n * 32;
  const int kb = args.K >> 1, units = args.K >> 7;
  const uint8_t* a0 = args.A + static_cast<int64_t>(m0) * kb;
  const uint8_t* w0 = args.W + static_cast<int64_t>(n0) * kb;
  const int64_t a_rows = static_cast<int64_t>(args.M - m0) * kb, w_rows = static_cast<int64_t>(args.N - n0) * kb;
  const uint32_t off = static_cast<uint32_t>(fr * kb + 32 * fh), soff = 4u * fr;
  float16_t acc = {};
  for (int u0 = wave; u0 < units; u0 += 4 * SP_UNITS) {
    int4_t a[SP_UNITS][2], w[SP_UNITS][2];
    uint32_t as[SP_UNITS], ws[SP_UNITS];
#pragma unroll
    for (int j = 0; j < SP_UNITS; ++j) {
      const int u = u0 + 4 * j;  // units past the last read nothing: their descriptors are empty
      const bool in = u < units;
      const int uu = in ? u : 0;
      const int an = in ? buf_bytes(a_rows - 64 * uu) : 0, wn = in ? buf_bytes(w_rows - 64 * uu) : 0;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        w[j][s] = buf_load_i4(w0 + 64 * uu, wn, off + 16 * s);
        a[j][s] = buf_load_i4(a0 + 64 * uu, an, off + 16 * s);
      }
      ws[j] = buf_load_u32(args.w_scale + static_cast<int64_t>(uu) * args.N + n0, in ? 4 * (args.N - n0) : 0, soff);
      as[j] = buf_load_u32(args.a_scale + static_cast<int64_t>(uu) * args.M + m0, in ? buf_bytes(4ll * (args.M - m0)) : 0,
                           soff);
    }
#pragma unroll
    for (int j = 0; j < SP_UNITS; ++j) {
      const uint32_t wsh = ws[j] >> (16 * fh), ash = as[j] >> (16 * fh);
      acc = mfma_mx4<0>(w[j][0], a[j][0], acc, wsh, ash);
      acc = mfma_mx4<1>(w[j][1], a[j][1], acc, wsh, ash);
    }
  }
  // acc[4 q + i]: row fr of A, column 8 q + 4 fh + i
  float* mine = part + (wave * 32 + fr) * SP_ROW;
#pragma unroll
  for (int q = 0; q < 4; ++q)
    *reinterpret_cast<float4_t*>(mine + 8 * q + 4 * fh) =
        float4_t{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
  __syncthreads();
  const int r = tid >> 3, c = 4 * (tid & 7);
  if (m0 + r >= args.M || n0 + c >= args.N) return;
  float4_t y = *reinterpret_cast<const float4_t*>(part + r * SP_ROW + c);
#pragma unroll
  for (int w = 1; w < 4; ++w) {
    const float4_t p = *reinterpret_cast<const float4_t*>(part + (w * 32 + r) * SP_ROW + c);
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = y[i] + p[i];
  }
  finish4<EPI, T>(args, m0 + r, n0 + c, y);
}

// ---------------- tiles from an LDS ring ----------------
//
// BM x BN tiles, WAVES_M x WAVES_N waves, a ring of S slots that hold U units of the tile's rows: 64 U bytes of codes a row,
// in 16-byte chunks swizzled against bank conflicts, and the units' exponent words behind them. Buffer loads fill the slots
// without passing through registers; rows past the matrix read as zeros.
template <int BM, int BN, int U>
constexpr int slot_bytes() {
  return (BM + BN) * 68 * U;
}

// Physical 16-byte chunk of a row's chunk c: the 16 rows that one read pass touches land in 16 distinct slots of 256 bytes.
template <int U>
__device__ __forceinline__ int mx4_swz(int row, int c) {
  if constexpr (U == 1)
    return row * 64 + ((c ^ ((row >> 2) & 3)) << 4);
  else
    return row * 128 + ((c ^ ((row >> 1) & 7)) << 4);
}

__device__ __forceinline__ void buffer_to_lds_at(const void* base, int nbytes, uint8_t* lds_dst, uint32_t voff, int soff) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, nbytes, RSRC_WORD3);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)lds_dst, 16, voff, soff, 0, 0);
}
__device__ __forceinline__ void word_to_lds(const void* base, int nbytes, uint8_t* lds_dst, uint32_t voff) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, nbytes, RSRC_WORD3);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)lds_dst, 4, voff, 0, 0, 0);
}

// The epilogue of one wave's rows m_base .. and columns n_base ..: acc[i][j][4 q + t] is row m_base + 32 j + lane % 32, column
// n_base + 32 i + 8 q + 4 (lane / 32) + t. 32 rows at a time the results go through the wave's own LDS (`stage`), so that
// global accesses are runs of a row, 16 bytes a lane.
template <int EPI, typename T, int NI>
constexpr int mx4_stage_row() {
  return (EPI == FF_EPI_SWIGLU ? NI * 16 : NI * 32) * static_cast<int>(sizeof(T)) + 16;
}

// Rows past M are dropped by the descriptor's range. WHOLE: the tile's columns lie inside the rows and these are 4-byte
// aligned; otherwise the columns are taken one a lane.
template <int EPI, typename T, int NI, int MI, bool WHOLE>
__device__ __forceinline__ void store_tile(const float16_t (&acc)[NI][MI], int m_base, int n_base, int lane,
                                           const Mx4Args& args, uint8_t* stage) {
  constexpr bool SWI = EPI == FF_EPI_SWIGLU;
  constexpr int RB = mx4_stage_row<EPI, T, NI>(), COLS = SWI ? NI * 16 : NI * 32;
  constexpr int E = WHOLE ? 16 / static_cast<int>(sizeof(T)) : 1;  // values of a lane's run
  constexpr int LPR = COLS / E < 64 ? COLS / E : 64;               // lanes a row
  constexpr int RPP = 64 / LPR, PASSES = 32 / RPP;                 // rows a pass
  static_assert(COLS / E <= 64, "a row fits a pass");
  typedef T run_t __attribute__((ext_vector_type(E)));
  const int fr = lane & 31, fh = lane >> 5;
  const int ld = SWI ? args.N >> 1 : args.N, n0 = SWI ? n_base >> 1 : n_base;
  const int c0 = (lane % LPR) * E, r0 = lane / LPR;
  const int64_t first = static_cast<int64_t>(m_base) * ld;
  const int bytes = buf_bytes((static_cast<int64_t>(args.M) * ld - first) * static_cast<int64_t>(sizeof(T)));
  T* out = static_cast<T*>(args.out) + first;
  const T* res = static_cast<const T*>(args.residual) + first;
  const uint32_t pitch = static_cast<uint32_t>(ld) * sizeof(T);  // at most 2^23: a wave's rows stay below 2^31 bytes
  const uint32_t off = WHOLE || n0 + c0 < ld ? r0 * pitch + (n0 + c0) * static_cast<uint32_t>(sizeof(T)) : OOB_OFFSET;
  auto at = [&](int j, int p) __attribute__((always_inline)) { return off + (32 * j + p * RPP) * pitch; };
  T* const own = reinterpret_cast<T*>(stage + r0 * RB) + c0;  // the lane's run of a pass, RPP rows apart
  // The residual's rows of block j, as the store phase walks them; they go through the staging area into the lanes that hold
  // the sums, so that sum and residual are rounded once.
  run_t x[PASSES];
  auto load_residual = [&](int j) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < PASSES; ++p) x[p] = buf_load_run<run_t>(res, bytes, at(j, p));
  };
  if constexpr (EPI == FF_EPI_RESIDUAL) load_residual(0);
#pragma unroll
  for (int j = 0; j < MI; ++j) {
    if constexpr (EPI == FF_EPI_RESIDUAL) {
#pragma unroll
      for (int p = 0; p < PASSES; ++p)
        *reinterpret_cast<run_t*>(reinterpret_cast<uint8_t*>(own) + p * RPP * RB) = x[p];
      if (j + 1 < MI) load_residual(j + 1);
    }
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = 32 * i + 8 * q + 4 * fh;
        float y[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          y[t] = acc[i][j][4 * q + t];
          if constexpr (EPI == FF_EPI_GELU_F16) y[t] = gelu_tanh(y[t]);
        }
        if constexpr (SWI) {
          typedef T two_t __attribute__((ext_vector_type(2)));
          *reinterpret_cast<two_t*>(stage + fr * RB + c) =
              two_t{static_cast<T>(silu(y[0]) * y[1]), static_cast<T>(silu(y[2]) * y[3])};
        } else {
          vec4_t<T>* to = reinterpret_cast<vec4_t<T>*>(stage + fr * RB + c * static_cast<int>(sizeof(T)));
          if constexpr (EPI == FF_EPI_RESIDUAL) {
            const vec4_t<T> r = *to;
#pragma unroll
            for (int t = 0; t < 4; ++t) y[t] = y[t] + static_cast<float>(r[t]);
          }
          *to = vec4_t<T>{static_cast<T>(y[0]), static_cast<T>(y[1]), static_cast<T>(y[2]), static_cast<T>(y[3])};
        }
      }
#pragma unroll
    for (int p = 0; p < PASSES; ++p)
      buf_store_run(*reinterpret_cast<const run_t*>(reinterpret_cast<const uint8_t*>(own) + p * RPP * RB), out, bytes,
                    at(j, p));
  }
}

template <int EPI, typename T, int BM, int BN, int WAVES_M, int WAVES_N, int U, int S, int OCC>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N, OCC) void gemm_mx4_ring_kernel(const Mx4Args args) {
  constexpr int WAVES = WAVES_M * WAVES_N, WM = BM / WAVES_M, WN = BN / WAVES_N, MI = WM / 32, NI = WN / 32;
  constexpr int ROW = 64 * U, SLOT = slot_bytes<BM, BN, U>(), CODES = (BM + BN) * ROW;
  constexpr int CPR = ROW / 16;                                    // 16-byte chunks of a row
  constexpr int BLOCKS = CODES / 1024, A_BLOCKS = BM * ROW / 1024;  // 1 KB blocks of a slot; A's come first
  constexpr int LOADS = BLOCKS / WAVES;                            // of them a wave loads
  constexpr int RUNS = (BM + BN) / 64, WORDS = U * RUNS;           // 64-row runs of exponent words, plane by plane
  constexpr int WLOADS = (WORDS + WAVES - 1) / WAVES;
  static_assert(BLOCKS % WAVES == 0 && BM % 64 == 0 && BN % 64 == 0, "even shares");
  constexpr int STAGE = 32 * mx4_stage_row<EPI, T, NI>();
  static_assert(WAVES * STAGE <= S * SLOT, "staging must fit in the ring");
  __shared__ __attribute__((aligned(1024))) uint8_t smem[S * SLOT];
  const int tid = threadIdx.x, lane = tid & 63, fr = lane & 31, fh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WAVES_N, wn = wave % WAVES_N;
  const int M = args.M, N = args.N;
  // tiles in groups of 8 row tiles by all column tiles, so that what runs at once on an XCD shares rows and columns
  const int tiles_m = (M + BM - 1) / BM, tiles_n = (N + BN - 1) / BN;
  const int t = xcd_remap(blockIdx.x, gridDim.x);
  const int g = t / (8 * tiles_n), in_g = t % (8 * tiles_n), gm = min(8, tiles_m - 8 * g);
  const int m0 = (8 * g + in_g % gm) * BM, n0 = in_g / gm * BN;
  const int kb = args.K >> 1, units = args.K >> 7, slots = (units + U - 1) / U;

  uint32_t voff[LOADS];
#pragma unroll
  for (int p = 0; p < LOADS; ++p) {
    const int blk = wave * LOADS + p, row = (blk < A_BLOCKS ? blk : blk - A_BLOCKS) * (1024 / ROW) + lane / CPR;
    voff[p] = static_cast<uint32_t>(row * kb + mx4_swz<U>(row, lane % CPR) - row * ROW);
  }
  // The tile's rows through one descriptor an operand (at most 256 rows of 2^21 bytes), a slot by the scalar offset: rows past
  // the matrix lie past the descriptor's end. (Behind the last unit of an odd count a slot holds what follows the row, which
  // is never used.) The exponent words' plane of a unit has a base of its own.
  const uint8_t* a_base = args.A + static_cast<int64_t>(m0) * kb;
  const uint8_t* w_base = args.W + static_cast<int64_t>(n0) * kb;
  const int a_bytes = min(BM, M - m0) * kb, w_bytes = min(BN, N - n0) * kb;
  const int a_words = min(BM, M - m0) * 4, w_words = min(BN, N - n0) * 4;
  const uint32_t* a_plane = args.a_scale + m0;
  const uint32_t* w_plane = args.w_scale + n0;
  int next = 0, next_slot = 0;  // the slot to be loaded next, and its LDS offset
  auto issue = [&]() __attribute__((always_inline)) {
    uint8_t* st = smem + next_slot;
#pragma unroll
    for (int p = 0; p < LOADS; ++p) {
      const int blk = wave * LOADS + p;
      buffer_to_lds_at(blk < A_BLOCKS ? a_base : w_base, blk < A_BLOCKS ? a_bytes : w_bytes, st + blk * 1024, voff[p],
                       ROW * next);
    }
#pragma unroll
    for (int p = 0; p < WLOADS; ++p) {
      const int i = min(wave * WLOADS + p, WORDS - 1);  // a run past the last loads the last one once more
      const int plane = i / RUNS, run = i % RUNS;
      const bool a = run < BM / 64, in = U * next + plane < units;  // planes past the last are empty
      word_to_lds((a ? a_plane : w_plane) + (in ? static_cast<int64_t>(plane) * (a ? M : N) : 0),
                  in ? (a ? a_words : w_words) : 0, st + CODES + i * 256, 4u * ((a ? run : run - BM / 64) * 64 + lane));
    }
    a_plane += static_cast<int64_t>(U) * M;
    w_plane += static_cast<int64_t>(U) * N;
    ++next;
    next_slot = next_slot == (S - 1) * SLOT ? 0 : next_slot + SLOT;
  };

  // The sums start from the bias: acc[i][j][4 q + t] is row 32 j + fr, column 32 i + 8 q + 4 fh + t of the wave's tile.
  float16_t acc[NI][MI];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int n = n0 + wn * WN + 32 * i + 8 * q + 4 * fh;
      float4_t b = {};
      if (args.bias) {
        if ((N & 3) == 0) {
          b = buf_load_f4(args.bias, 4 * N, 4u * n);
        } else {
#pragma unroll
          for (int t = 0; t < 4; ++t) b[t] = buf_load_f1(args.bias, 4 * N, 4u * (n + t));
        }
      }
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < MI; ++j) acc[i][j][4 * q + t] = b[t];
    }
#pragma unroll
  for (int s = 0; s < S - 1; ++s)
    if (s < slots) issue();

  int4_t xw[2][NI], ya[2][MI];
  uint32_t sw[NI], sa[MI];
  // the fragments of half unit k of a slot
  auto read_frags = [&](const uint8_t* st, int k) __attribute__((always_inline)) {
    const int c = 4 * (k >> 1) + 2 * fh + (k & 1);
#pragma unroll
    for (int i = 0; i < NI; ++i)
      xw[k & 1][i] = *reinterpret_cast<const int4_t*>(st + BM * ROW + mx4_swz<U>(wn * WN + 32 * i + fr, c));
#pragma unroll
    for (int j = 0; j < MI; ++j)
      ya[k & 1][j] = *reinterpret_cast<const int4_t*>(st + mx4_swz<U>(wm * WM + 32 * j + fr, c));
  };
  // the two exponents of the lane's half in a unit of a slot
  auto read_words = [&](const uint8_t* slot, int unit, uint32_t (&w)[NI],
                        uint32_t (&a)[MI]) __attribute__((always_inline)) {
    const uint8_t* st = slot + CODES + unit * RUNS * 256 + 2 * fh;
#pragma unroll
    for (int i = 0; i < NI; ++i) w[i] = *reinterpret_cast<const uint16_t*>(st + 4 * (BM + wn * WN + 32 * i + fr));
#pragma unroll
    for (int j = 0; j < MI; ++j) a[j] = *reinterpret_cast<const uint16_t*>(st + 4 * (wm * WM + 32 * j + fr));
  };
  auto mfmas = [&](auto step) __attribute__((always_inline)) {
    constexpr int b = decltype(step)::value;
#pragma unroll
    for (int j = 0; j < MI; ++j)
#pragma unroll
      for (int i = 0; i < NI; ++i) acc[i][j] = mfma_mx4<b>(xw[b][i], ya[b][j], acc[i][j], sw[i], sa[j]);
  };
  auto interleave = [](auto per) __attribute__((always_inline)) {  // `per` LDS reads after each product
    constexpr int n = NI + MI < NI * MI ? NI + MI : NI * MI;
#pragma unroll
    for (int x = 0; x < n; ++x) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                    // 1 MFMA
      __builtin_amdgcn_sched_group_barrier(0x100, decltype(per)::value, 0);  // DS reads
    }
    __builtin_amdgcn_sched_group_barrier(0x008, NI * MI - n, 0);
  };
  if (slots >= S - 1)
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 2) * (LOADS + WLOADS)) : "memory");
  else
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  read_frags(smem, 0);
  read_words(smem, 0, sw, sa);
  // One slot: each half unit's fragments are read under the products of the half before it, a unit's exponents under the
  // unit before it, and the next slot's first ones (after its barrier) under this slot's last products. On the last slot
  // that reads a stale slot and is not used.
  int slot = 0;
  auto step = [&](auto kc, auto steady) __attribute__((always_inline)) {
    constexpr int k = decltype(kc)::value;
    uint32_t nw[NI], na[MI];
    if constexpr (k + 1 < 2 * U) {
      if constexpr (k & 1) read_words(smem + slot, (k + 1) / 2, nw, na);
      read_frags(smem + slot, k + 1);
    } else {
      // The next slot has landed once at most the loads of the newer slots are outstanding; lgkmcnt(0): this wave's reads of
      // older slots are complete, so that after the barrier any of them may be refilled.
      if constexpr (decltype(steady)::value)
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((S - 2) * (LOADS + WLOADS)) : "memory");
      else
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      slot = slot == (S - 1) * SLOT ? 0 : slot + SLOT;
      read_words(smem + slot, 0, nw, na);
      read_frags(smem + slot, 0);
    }
    mfmas(std::integral_constant<int, k & 1>{});
    interleave(std::integral_constant<int, (k & 1) + 1>{});
    if constexpr (k & 1) {
#pragma unroll
      for (int i = 0; i < NI; ++i) sw[i] = nw[i];
#pragma unroll
      for (int j = 0; j < MI; ++j) sa[j] = na[j];
    }
  };
  auto whole = [&](auto steady) __attribute__((always_inline)) {
    if constexpr (decltype(steady)::value) issue();
    step(std::integral_constant<int, 0>{}, steady);
    step(std::integral_constant<int, 1>{}, steady);
    if constexpr (U == 2) {
      step(std::integral_constant<int, 2>{}, steady);
      step(std::integral_constant<int, 3>{}, steady);
    }
  };
  int u = 0;
  for (; u + S - 1 < slots; ++u) whole(std::true_type{});
  for (; u < units / U; ++u) whole(std::false_type{});
  if constexpr (U == 2) {
    if (u < slots) {  // an odd unit
      step(std::integral_constant<int, 0>{}, std::false_type{});
      step(std::integral_constant<int, 1>{}, std::false_type{});
    }
  }
  __syncthreads();  // every wave is done with the ring: it becomes the staging area
  const int ld = EPI == FF_EPI_SWIGLU ? N >> 1 : N;
  if (n0 + BN <= N && (ld & (4 / static_cast<int>(sizeof(T)) - 1)) == 0)
    store_tile<EPI, T, NI, MI, true>(acc, m0 + wm * WM, n0 + wn * WN, lane, args, smem + wave * STAGE);
  else
    store_tile<EPI, T, NI, MI, false>(acc, m0 + wm * WM, n0 + wn * WN, lane, args, smem + wave * STAGE);
}

template <int EPI, typename T, int BM, int BN, int WAVES_M, int WAVES_N, int U, int S, int OCC>
static int launch_ring(const Mx4Args& a, hipStream_t st) {
  const int64_t tiles = static_cast<int64_t>((a.M + BM - 1) / BM) * ((a.N + BN - 1) / BN);
  gemm_mx4_ring_kernel<EPI, T, BM, BN, WAVES_M, WAVES_N, U, S, OCC>
      <<<dim3(static_cast<unsigned>(tiles)), 64 * WAVES_M * WAVES_N, 0, st>>>(a);
  return check_launch("gemm_mx4");
}

// The tile shape without a chosen one: the lowest estimated time. The estimate (us) is fixed + the larger (a 4-norm) of what
// one tile takes after another, rounds (first + unit u), and what a CU takes for its tiles, each tile + tile_unit u, with u
// units of K, plus the outputs' share. Fitted to the times of 300 products (1 .. 33 000 rows, 32 .. 9000 columns, K 128 ..
// 5120); on 196 others its pick is 1.4 % slower than the fastest shape on average and 12 % at worst, where the 64 x 64
// tiles alone are 9 % slower on average, the 256 x 128 tiles alone 74 %.
struct Mx4Cost {
  int bm, bn, threads, resident;  // tile, threads of a workgroup, workgroups a CU holds
  bool whole;                     // rounds count whole (few tiles a CU) or as a fraction
  double fixed, first, unit, tile, tile_unit, out;
};
constexpr Mx4Cost MX4_COSTS[5] = {
    {32, 32, 256, 4, false, 3.158, 0.607, 0.0353, 0.144, 0.0972, 1.149},
    {64, 64, 256, 3, true, 2.968, 0.504, 0.1246, 0.0, 0.1097, 0.586},
    {128, 128, 256, 3, true, 3.740, 0.528, 0.0971, 0.0, 0.2919, 0.376},
    {256, 128, 256, 2, false, 3.725, 1.567, 0.1800, 0.674, 0.4621, 0.365},
    {256, 256, 512, 1, false, 1.317, 4.798, 0.2753, 3.826, 0.6012, 0.389},
};
static int64_t tiles_of(const Mx4Cost& c, int M, int N) {
  return static_cast<int64_t>((M + c.bm - 1) / c.bm) * ((N + c.bn - 1) / c.bn);
}
static bool launchable(const Mx4Cost& c, int M, int N) {  // a launch has fewer than 2^32 threads
  return tiles_of(c, M, N) <= 0xffffffffll / c.threads;
}
static int pick_variant(int M, int N, int K) {
  const double u = K / 128;
  int best = 5;
  double least = HUGE_VAL;
  for (int v = 0; v < 5; ++v) {
    const Mx4Cost& c = MX4_COSTS[v];
    const double tiles = static_cast<double>(tiles_of(c, M, N));
    double rounds = tiles / (256.0 * c.resident);
    rounds = c.whole ? std::ceil(rounds) : std::max(1.0, rounds);
    const double one = rounds * (c.first + c.unit * u), all = std::ceil(tiles / 256.0) * (c.tile + c.tile_unit * u);
    const double t = c.fixed + std::sqrt(std::sqrt(one * one * one * one + all * all * all * all)) + c.out * 1e-6 * M * N;
    if (launchable(c, M, N) && t < least) {
      least = t;
      best = v + 1;
    }
  }
  return best;
}

template <int EPI, typename T>
static int launch_mx4(const Mx4Args& a, int variant, hipStream_t st) {
  switch (variant) {
    case 2: return launch_ring<EPI, T, 64, 64, 2, 2, 2, 3, 3>(a, st);
    case 3: return launch_ring<EPI, T, 128, 128, 2, 2, 1, 3, 3>(a, st);
    case 4: return launch_ring<EPI, T, 256, 128, 2, 2, 1, 3, 2>(a, st);
    case 5: return launch_ring<EPI, T, 256, 256, 2, 4, 1, 3, 2>(a, st);
    default: break;
  }
  const int64_t blocks = static_cast<int64_t>((a.M + 31) / 32) * ((a.N + 31) / 32);
  gemm_mx4_split_kernel<EPI, T><<<dim3(static_cast<unsigned>(blocks)), 256, 0, st>>>(a);
  return check_launch("gemm_mx4");
}

template <typename T>
static int launch_mx4_epi(const Mx4Args& a, int epi, int variant, hipStream_t st) {
  switch (epi) {
    case FF_EPI_RESIDUAL: return launch_mx4<FF_EPI_RESIDUAL, T>(a, variant, st);
    case FF_EPI_GELU_F16: return launch_mx4<FF_EPI_GELU_F16, T>(a, variant, st);
    case FF_EPI_SWIGLU: return launch_mx4<FF_EPI_SWIGLU, T>(a, variant, st);
    default: return launch_mx4<FF_EPI_BIAS_F16, T>(a, variant, st);
  }
}

}  // namespace ff

using namespace ff;

extern "C" int ff_gemm_mx4(const uint8_t* A, const uint32_t* a_scale, const uint8_t* W, const uint32_t* w_scale, int64_t M,
                           int64_t N, int64_t K, const float* bias, const void* residual, void* out, int dtype, int epi,
                           int variant, void* stream) {
  clear_error();
  if (epi < FF_EPI_RESIDUAL || epi > FF_EPI_BIAS_F16)
    return fail(FF_EINVAL, "gemm_mx4: epilogue must be residual, GELU, SwiGLU or bias");
  if (dtype != FF_F16 && dtype != FF_BF16 && !(dtype == FF_F32 && epi == FF_EPI_BIAS_F16))
    return fail(FF_EINVAL, "gemm_mx4: out must be fp16 or bf16 (or fp32, bias epilogue only)");
  if (variant < 0 || variant > ff_gemm_mx4_variants()) return fail(FF_EINVAL, "gemm_mx4: unknown variant");
  if (K <= 0 || K % 128 != 0) return fail(FF_EINVAL, "gemm_mx4: K must be a positive multiple of 128");
  if (N <= 0 || (epi == FF_EPI_SWIGLU && N % 2 != 0))
    return fail(FF_EINVAL, "gemm_mx4: N must be positive, and even for SwiGLU");
  if (M < 0 || M > 0x7fffff00 || N > (1 << 21) || K > (1 << 22))
    return fail(FF_EINVAL, "gemm_mx4: need M >= 0, N <= 2^21, K <= 2^22; larger is not supported");
  if (M == 0) return FF_OK;
  if (!A || !a_scale || !W || !w_scale || !out || (epi == FF_EPI_RESIDUAL && !residual))
    return fail(FF_EINVAL, "gemm_mx4: null pointer");
  auto low = [](const void* p) { return reinterpret_cast<uintptr_t>(p) & 15; };
  if (low(A) || low(W) || low(out) || low(bias) || (epi == FF_EPI_RESIDUAL && low(residual)) || (low(a_scale) & 3) ||
      (low(w_scale) & 3))
    return fail(FF_EINVAL, "gemm_mx4: misaligned pointer");
  const Extent to = range(out, M * (epi == FF_EPI_SWIGLU ? N / 2 : N) * (dtype == FF_F32 ? 4 : 2));
  // elements are read and written by different workgroups, in no order
  if (epi == FF_EPI_RESIDUAL && residual != out && !clear_of(to, range(residual, to.len)))
    return fail(FF_EINVAL, "gemm_mx4: residual overlaps out in part");
  if (variant == 0) variant = pick_variant(static_cast<int>(M), static_cast<int>(N), static_cast<int>(K));
  if (!launchable(MX4_COSTS[variant - 1], static_cast<int>(M), static_cast<int>(N)))
    return fail(FF_EINVAL, "gemm_mx4: too many tiles for this variant");
  for (const Extent& e : {range(A, M * (K / 2)), range(a_scale, M * (K / 32)), range(W, N * (K / 2)),
                          range(w_scale, N * (K / 32)), range(bias, 4 * N)})
    if (e.at != 0 && !clear_of(to, e)) return fail(FF_EINVAL, "gemm_mx4: out overlaps an operand");
  const Mx4Args a{A, a_scale, W, w_scale, static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), bias, residual,
                  out};
  const hipStream_t st = as_stream(stream);
  if (dtype == FF_F16) return launch_mx4_epi<half_t>(a, epi, variant, st);
  if (dtype == FF_BF16) return launch_mx4_epi<bf16_t>(a, epi, variant, st);
  return launch_mx4<FF_EPI_BIAS_F16, float>(a, variant, st);
}

extern "C" int ff_gemm_mx4_variants(void) { return 5; }
