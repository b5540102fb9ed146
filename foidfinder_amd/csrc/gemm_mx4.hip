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
#include <algorithm>
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

// D += W-fragment x A-fragment over 64 columns; S: the byte of the exponent words that holds this step's block.
template <int S>
__device__ __forceinline__ float16_t mfma_mx4(int4_t w, int4_t a, float16_t c, uint32_t ws, uint32_t as) {
  const int8_t_v wv = {w[0], w[1], w[2], w[3], 0, 0, 0, 0}, av = {a[0], a[1], a[2], a[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv, av, c, 4, 4, S, static_cast<int>(ws), S,
                                                         static_cast<int>(as));
}

// The epilogue of four consecutive columns n .. n + 3 of row m (n % 4 == 0, n < N): y holds the sums. One rounding, at the
// store. Columns past N are not touched; whole runs are stored at once when N % 4 == 0 keeps them aligned.
template <int EPI, typename T>
__device__ __forceinline__ void finish4(const Mx4Args& args, int m, int n, float4_t y) {
  const int N = args.N;
  const bool whole = (N & 3) == 0;
  if (args.bias) {
    if (whole) {
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
    const int64_t at = static_cast<int64_t>(m) * N + n;
    T* o = static_cast<T*>(args.out) + at;
    if constexpr (EPI == FF_EPI_RESIDUAL) {
      const T* r = static_cast<const T*>(args.residual) + at;
      if (whole) {
        const vec4_t<T> x = *reinterpret_cast<const vec4_t<T>*>(r);
#pragma unroll
        for (int t = 0; t < 4; ++t) y[t] = y[t] + static_cast<float>(x[t]);
      } else {
#pragma unroll
        for (int t = 0; t < 4; ++t)
          if (n + t < N) y[t] = y[t] + static_cast<float>(r[t]);
      }
    }
    if constexpr (EPI == FF_EPI_GELU_F16) {
#pragma unroll
      for (int t = 0; t < 4; ++t) y[t] = gelu_tanh(y[t]);
    }
    vec4_t<T> h;
#pragma unroll
    for (int t = 0; t < 4; ++t) h[t] = static_cast<T>(y[t]);
    if (whole) {
      *reinterpret_cast<vec4_t<T>*>(o) = h;
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
// BM x BN tiles, WAVES_M x WAVES_N waves, a ring of S slots that hold one unit (128 columns of K) of the tile's rows: 64
// bytes of codes a row, in 16-byte chunks swizzled against bank conflicts, and the rows' exponent words behind them. Buffer
// loads fill the slots without passing through registers; rows past the matrix read as zeros.
template <int BM, int BN>
constexpr int slot_bytes() {
  return (BM + BN) * 68;
}

// Physical 16-byte chunk of a row's chunk c: the 16 rows that one read pass touches land in 16 distinct slots of 256 bytes.
__device__ __forceinline__ int mx4_swz(int row, int c) { return row * 64 + ((c ^ ((row >> 2) & 3)) << 4); }

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

template <int EPI, typename T, int NI, int MI>
__device__ __forceinline__ void store_tile(const float16_t (&acc)[NI][MI], int m_base, int n_base, int lane,
                                           const Mx4Args& args, uint8_t* stage, const float* bias) {
  constexpr bool SWI = EPI == FF_EPI_SWIGLU;
  constexpr int RB = mx4_stage_row<EPI, T, NI>(), COLS = SWI ? NI * 16 : NI * 32;
  constexpr int E = 16 / static_cast<int>(sizeof(T));  // values of a 16-byte run
  constexpr int LPR = COLS / E, RPP = 64 / LPR;        // lanes a row, rows a pass
  typedef T run_t __attribute__((ext_vector_type(E)));
  const int fr = lane & 31, fh = lane >> 5;
  const int ld = SWI ? args.N >> 1 : args.N, n0 = SWI ? n_base >> 1 : n_base;
  const int n = n0 + (lane % LPR) * E, r0 = lane / LPR;
  const bool runs = (ld & (4 / sizeof(T) - 1)) == 0 && n + E <= ld;  // 4-byte aligned rows, the run inside them
  float4_t b[NI][4];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) b[i][q] = *reinterpret_cast<const float4_t*>(bias + 32 * i + 8 * q + 4 * fh);
#pragma unroll
  for (int j = 0; j < MI; ++j) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float y[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          y[t] = acc[i][j][4 * q + t] + b[i][q][t];
          if constexpr (EPI == FF_EPI_GELU_F16) y[t] = gelu_tanh(y[t]);
        }
        const int c = 32 * i + 8 * q + 4 * fh;
        if constexpr (SWI) {
          typedef T two_t __attribute__((ext_vector_type(2)));
          *reinterpret_cast<two_t*>(stage + fr * RB + c) =
              two_t{static_cast<T>(silu(y[0]) * y[1]), static_cast<T>(silu(y[2]) * y[3])};
        } else if constexpr (EPI == FF_EPI_RESIDUAL) {
          // y itself: the sum with the residual is rounded once
          *reinterpret_cast<float4_t*>(stage + fr * (NI * 128 + 16) + 4 * c) = float4_t{y[0], y[1], y[2], y[3]};
        } else {
          *reinterpret_cast<vec4_t<T>*>(stage + fr * RB + c * static_cast<int>(sizeof(T))) =
              vec4_t<T>{static_cast<T>(y[0]), static_cast<T>(y[1]), static_cast<T>(y[2]), static_cast<T>(y[3])};
        }
      }
#pragma unroll
    for (int p = 0; p < 32 / RPP; ++p) {
      const int r = p * RPP + r0, m = m_base + 32 * j + r;
      run_t h;
      if (m < args.M && n < ld) {
        const int64_t at = static_cast<int64_t>(m) * ld + n;
        T* o = static_cast<T*>(args.out) + at;
        if constexpr (EPI == FF_EPI_RESIDUAL) {
          const float* y = reinterpret_cast<const float*>(stage + r * (NI * 128 + 16)) + (lane % LPR) * E;
          const T* x = static_cast<const T*>(args.residual) + at;
          if (runs) {
            run_t xv;
            __builtin_memcpy(&xv, x, 16);
#pragma unroll
            for (int e = 0; e < E; ++e) h[e] = static_cast<T>(y[e] + static_cast<float>(xv[e]));
          } else {
#pragma unroll
            for (int e = 0; e < E; ++e) h[e] = static_cast<T>(y[e] + (n + e < ld ? static_cast<float>(x[e]) : 0.f));
          }
        } else {
          h = *reinterpret_cast<const run_t*>(stage + r * RB + (lane % LPR) * 16);
        }
        if (runs) {
          __builtin_memcpy(o, &h, 16);
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (n + e < ld) o[e] = h[e];
        }
      }
    }
  }
}

template <int EPI, typename T, int BM, int BN, int WAVES_M, int WAVES_N, int S>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N, 2) void gemm_mx4_ring_kernel(const Mx4Args args) {
  constexpr int WAVES = WAVES_M * WAVES_N, WM = BM / WAVES_M, WN = BN / WAVES_N, MI = WM / 32, NI = WN / 32;
  constexpr int SLOT = slot_bytes<BM, BN>(), CODES = (BM + BN) * 64;
  constexpr int BLOCKS = CODES / 1024, A_BLOCKS = BM * 64 / 1024;  // 1 KB blocks (16 rows) of a slot; A's come first
  constexpr int LOADS = BLOCKS / WAVES;                            // of them a wave loads
  constexpr int WORDS = (BM + BN) / 64, WLOADS = (WORDS + WAVES - 1) / WAVES;  // 64-row runs of exponent words
  static_assert(BLOCKS % WAVES == 0 && BM % 64 == 0 && BN % 64 == 0, "even shares");
  constexpr int STAGE = 32 * (EPI == FF_EPI_RESIDUAL ? NI * 128 + 16 : mx4_stage_row<EPI, T, NI>());
  static_assert(WAVES * STAGE + BN * 4 <= S * SLOT, "staging must fit in the ring");
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
  const int kb = args.K >> 1, units = args.K >> 7;

  uint32_t voff[LOADS];
#pragma unroll
  for (int p = 0; p < LOADS; ++p) {
    const int blk = wave * LOADS + p, row = (blk < A_BLOCKS ? blk : blk - A_BLOCKS) * 16 + (lane >> 2);
    voff[p] = static_cast<uint32_t>(row * kb + mx4_swz(row, lane & 3) - row * 64);
  }
  const int64_t a_rows = static_cast<int64_t>(M - m0) * kb, w_rows = static_cast<int64_t>(N - n0) * kb;
  const int a_words = buf_bytes(4ll * (M - m0)), w_words = buf_bytes(4ll * (N - n0));
  auto issue = [&](int u) __attribute__((always_inline)) {
    uint8_t* st = smem + (u % S) * SLOT;
    const uint8_t* ab = args.A + static_cast<int64_t>(m0) * kb + 64 * u;
    const uint8_t* wb = args.W + static_cast<int64_t>(n0) * kb + 64 * u;
    const int an = buf_bytes(a_rows - 64 * u), wn_ = buf_bytes(w_rows - 64 * u);
#pragma unroll
    for (int p = 0; p < LOADS; ++p) {
      const int blk = wave * LOADS + p;
      buffer_to_lds(blk < A_BLOCKS ? ab : wb, blk < A_BLOCKS ? an : wn_, st + blk * 1024, voff[p]);
    }
    const uint32_t* as = args.a_scale + static_cast<int64_t>(u) * M + m0;
    const uint32_t* ws = args.w_scale + static_cast<int64_t>(u) * N + n0;
#pragma unroll
    for (int p = 0; p < WLOADS; ++p) {
      const int i = min(wave * WLOADS + p, WORDS - 1);  // a run past the last loads the last one once more
      const bool a = i < BM / 64;
      word_to_lds(a ? as : ws, a ? a_words : w_words, st + CODES + i * 256, 4u * ((a ? i : i - BM / 64) * 64 + lane));
    }
  };

  float16_t acc[NI][MI] = {};
#pragma unroll
  for (int s = 0; s < S - 1; ++s)
    if (s < units) issue(s);

  int4_t xw[2][NI], ya[2][MI];
  uint32_t sw[NI], sa[MI];
  auto read_frags = [&](const uint8_t* st, int step, int b) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
      xw[b][i] = *reinterpret_cast<const int4_t*>(st + BM * 64 + mx4_swz(wn * WN + 32 * i + fr, 2 * fh + step));
#pragma unroll
    for (int j = 0; j < MI; ++j)
      ya[b][j] = *reinterpret_cast<const int4_t*>(st + mx4_swz(wm * WM + 32 * j + fr, 2 * fh + step));
  };
  auto read_words = [&](const uint8_t* slot) __attribute__((always_inline)) {  // the two exponents of the lane's half
    const uint8_t* st = slot + CODES + 2 * fh;
#pragma unroll
    for (int i = 0; i < NI; ++i) sw[i] = *reinterpret_cast<const uint16_t*>(st + 4 * (BM + wn * WN + 32 * i + fr));
#pragma unroll
    for (int j = 0; j < MI; ++j) sa[j] = *reinterpret_cast<const uint16_t*>(st + 4 * (wm * WM + 32 * j + fr));
  };
  auto mfmas = [&](auto step) __attribute__((always_inline)) {
    constexpr int b = decltype(step)::value;
#pragma unroll
    for (int j = 0; j < MI; ++j)
#pragma unroll
      for (int i = 0; i < NI; ++i) acc[i][j] = mfma_mx4<b>(xw[b][i], ya[b][j], acc[i][j], sw[i], sa[j]);
  };
  auto interleave = [] __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < NI + MI; ++x) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // 1 MFMA
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // 1 DS read
    }
    __builtin_amdgcn_sched_group_barrier(0x008, NI * MI - (NI + MI), 0);
  };
  if (units >= S - 1)
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 2) * (LOADS + WLOADS)) : "memory");
  else
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  read_frags(smem, 0, 0);
  read_words(smem);
  // One unit: the second half's fragments are read under the first half's products, the next unit's first half (after its
  // barrier) under the second half's. On the last unit that reads a stale slot and is not used.
  auto unit = [&](int u, auto steady) __attribute__((always_inline)) {
    if constexpr (decltype(steady)::value) issue(u + S - 1);
    read_frags(smem + u % S * SLOT, 1, 1);
    mfmas(std::integral_constant<int, 0>{});
    interleave();
    // Slot u + 1 has landed once at most the loads of the newer slots are outstanding; lgkmcnt(0): this wave's reads of older
    // slots are complete, so that after the barrier any of them may be refilled.
    if constexpr (decltype(steady)::value)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((S - 2) * (LOADS + WLOADS)) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    read_frags(smem + (u + 1) % S * SLOT, 0, 0);
    mfmas(std::integral_constant<int, 1>{});
    interleave();
    read_words(smem + (u + 1) % S * SLOT);
  };
  int u = 0;
  for (; u + S - 1 < units; ++u) unit(u, std::true_type{});
  for (; u < units; ++u) unit(u, std::false_type{});
  __syncthreads();  // every wave is done with the ring: it becomes the staging area, with the tile's bias behind it
  float* bias = reinterpret_cast<float*>(smem + WAVES * STAGE);
  for (int i = tid; i < BN; i += 64 * WAVES) bias[i] = args.bias && n0 + i < N ? args.bias[n0 + i] : 0.f;
  __syncthreads();
  store_tile<EPI, T, NI, MI>(acc, m0 + wm * WM, n0 + wn * WN, lane, args, smem + wave * STAGE, bias + wn * WN);
}

template <int EPI, typename T, int BM, int BN, int WAVES_M, int WAVES_N, int S>
static int launch_ring(const Mx4Args& a, hipStream_t st) {
  const int64_t tiles = static_cast<int64_t>((a.M + BM - 1) / BM) * ((a.N + BN - 1) / BN);
  if (tiles > 0x7fffffff) return fail(FF_EINVAL, "gemm_mx4: too many tiles");
  gemm_mx4_ring_kernel<EPI, T, BM, BN, WAVES_M, WAVES_N, S>
      <<<dim3(static_cast<unsigned>(tiles)), 64 * WAVES_M * WAVES_N, 0, st>>>(a);
  return check_launch("gemm_mx4");
}

template <int EPI, typename T>
static int launch_mx4(const Mx4Args& a, int variant, hipStream_t st) {
  if (variant == 2 || (variant == 0 && a.M > 256)) return launch_ring<EPI, T, 256, 128, 2, 2, 3>(a, st);
  const int64_t blocks = static_cast<int64_t>((a.M + 31) / 32) * ((a.N + 31) / 32);
  if (blocks > 0x7fffffff) return fail(FF_EINVAL, "gemm_mx4: too many tiles");
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
  const Mx4Args a{A, a_scale, W, w_scale, static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), bias, residual,
                  out};
  const hipStream_t st = as_stream(stream);
  if (dtype == FF_F16) return launch_mx4_epi<half_t>(a, epi, variant, st);
  if (dtype == FF_BF16) return launch_mx4_epi<bf16_t>(a, epi, variant, st);
  return launch_mx4<FF_EPI_BIAS_F16, float>(a, variant, st);
}

extern "C" int ff_gemm_mx4_variants(void) { return 2; }
