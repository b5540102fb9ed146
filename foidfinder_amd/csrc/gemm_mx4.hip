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

template <int EPI, typename T>
static int launch_mx4(const Mx4Args& a, hipStream_t st) {
  const int64_t blocks = static_cast<int64_t>((a.M + 31) / 32) * ((a.N + 31) / 32);
  if (blocks > 0x7fffffff) return fail(FF_EINVAL, "gemm_mx4: too many tiles");
  gemm_mx4_split_kernel<EPI, T><<<dim3(static_cast<unsigned>(blocks)), 256, 0, st>>>(a);
  return check_launch("gemm_mx4");
}

template <typename T>
static int launch_mx4_epi(const Mx4Args& a, int epi, hipStream_t st) {
  switch (epi) {
    case FF_EPI_RESIDUAL: return launch_mx4<FF_EPI_RESIDUAL, T>(a, st);
    case FF_EPI_GELU_F16: return launch_mx4<FF_EPI_GELU_F16, T>(a, st);
    case FF_EPI_SWIGLU: return launch_mx4<FF_EPI_SWIGLU, T>(a, st);
    default: return launch_mx4<FF_EPI_BIAS_F16, T>(a, st);
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
  if (dtype == FF_F16) return launch_mx4_epi<half_t>(a, epi, st);
  if (dtype == FF_BF16) return launch_mx4_epi<bf16_t>(a, epi, st);
  return launch_mx4<FF_EPI_BIAS_F16, float>(a, st);
}

extern "C" int ff_gemm_mx4_variants(void) { return 1; }
