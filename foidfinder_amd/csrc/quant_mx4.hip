// MX4 (OCP microscaling, E2M1 elements with one E8M0 exponent per 32 columns): a row's norm, the block-diagonal H128
// rotation and the 4-bit codes in one pass, and the values back from the codes.
//
// Per block of 32 columns: e = floor(log2(max |v|)) - 2, so the largest value lands in [4, 8), code = E2M1(v 2^-e) to
// nearest with ties to even, saturating at 6 (the format's own rule); e is clamped at -127, and a block with a value that is
// not finite gets the exponent 255, which makes all of it not a number, so that a fault shows in the product instead of
// turning into a plausible code. One 32-bit word holds the exponents of a row's 128 columns (the byte i of columns 32 i ..),
// and the words of one 128-column block are contiguous over the rows (scale [C / 128, T]): the product's lanes then load
// their rows' words as one contiguous run, where row-major exponents would cost a cache line per row.
//
// Layout: 16 lanes (one DPP row) own a 128-column block, 8 columns a lane in Gray order (rotate.h), so the rotation's
// lane butterflies and the maximum over a 32-column block (a quad of lanes) are DPP operations; four such groups of a wave
// take blocks 4 i + g of one row.
//
// Every step is one IEEE fp32 operation in a stated order, so codes and exponents can be checked bit for bit:
//  * sums (of x, then of (x - mean)^2 by fused multiply-adds): 64 partial sums a row, partial 16 (b mod 4) + c over the
//    columns 8 c .. 8 c + 7 of the blocks b, ascending; then folded in halves (32, 16, 8, 4, 2, 1);
//  * the norm ((x - mean) rstd) gamma + beta with a fused last step; for the RMS norm mean = beta = 0;
//  * the rotation's stages over column bits 0..6 ascending, then one multiplication by fp32(1 / sqrt(128)).
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "rotate.h"

namespace ff {

constexpr float ROOT128 = 0.08838834764831845f;

// The larger of |a|, |b|, |c|; not a number if any is (v_maximum3_f32).
__device__ __forceinline__ float amax3(float a, float b, float c) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(__builtin_fabsf(a), __builtin_fabsf(b)),
                                       __builtin_fabsf(c));
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xF, 0xF, false));
}

// The lane's columns of N blocks (v[8 i + e], Gray chunk gl), rotated if `rotate`, to codes[i] (8 codes, the first column in
// the low bits) and words[i] (the block's exponents, in each of its 16 lanes).
template <int N>
__device__ __forceinline__ void encode_blocks(float (&v)[8 * N], bool rotate, int gl, uint32_t (&codes)[N],
                                              uint32_t (&words)[N]) {
  if (rotate) {
#pragma unroll
    for (int h = 1; h < 8; h <<= 1)
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (!(e & h)) {
            const float a = v[8 * i + e], b = v[8 * i + e + h];
            v[8 * i + e] = a + b;
            v[8 * i + e + h] = a - b;
          }
    bfly_stage<DPP_XOR1>(v, gray_sign(gl & 1));
    bfly_stage<DPP_XOR3>(v, gray_sign(gl & 2));
    bfly_stage<DPP_XOR7>(v, gray_sign(gl & 4));
    bfly_stage<DPP_XOR15>(v, gray_sign(gl & 8));
    // the sign that the lane butterflies left (rounding is sign-symmetric) goes with the factor
    const float f = __builtin_popcount(gl) & 1 ? -ROOT128 : ROOT128;
#pragma unroll
    for (int i = 0; i < 8 * N; ++i) v[i] = v[i] * f;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float m = amax3(amax3(v[8 * i], v[8 * i + 1], v[8 * i + 2]), v[8 * i + 3], v[8 * i + 4]);
    m = amax3(amax3(m, v[8 * i + 5], v[8 * i + 6]), v[8 * i + 7], 0.f);
    m = __builtin_elementwise_maximum(m, dpp<DPP_XOR1>(m));
    m = __builtin_elementwise_maximum(m, dpp<DPP_XOR3>(m));
    const uint32_t field = (__builtin_bit_cast(uint32_t, m) >> 23) & 0xff;
    const uint32_t eb = field == 255 ? 255 : (field > 2 ? field - 2 : 0);
    const float s = __builtin_bit_cast(float, eb << 23);  // read by its exponent alone: 0 stands for 2^-127
    uint32_t q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[8 * i], v[8 * i + 1], s, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[8 * i + 2], v[8 * i + 3], s, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[8 * i + 4], v[8 * i + 5], s, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[8 * i + 6], v[8 * i + 7], s, 3);
    codes[i] = q;
    uint32_t w = eb << (8 * (gl >> 2));  // lanes l ^ 7 and l ^ 15 lie in the other quads
    w |= dpp_u32<DPP_XOR7>(w);
    w |= dpp_u32<DPP_XOR15>(w);
    words[i] = w;
  }
}

// Without a norm the blocks are independent: a wave takes four blocks of one row at a time, waves stride over all of them.
// 5184 x 4736 bf16 15 us, 4.1 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void quant_mx4_kernel(const T* __restrict__ x, int64_t x_stride, int64_t rows, int C,
                                                        bool rotate, uint8_t* __restrict__ out,
                                                        uint32_t* __restrict__ scale) {
  const int nb = C >> 7, per = (nb + 3) >> 2;  // steps of four blocks a row
  const int lane = threadIdx.x & 63, g = lane >> 4, l16 = lane & 15, gl = l16 ^ (l16 >> 1);
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  // the wave's first step and its stride in whole rows and steps: one 32-bit division each, none in the loop
  const int waves = static_cast<int>(gridDim.x) * 4, first = static_cast<int>(blockIdx.x) * 4 + wave;
  const int row_step = waves / per, step = waves - row_step * per;
  int64_t row = first / per;
  int i = first - static_cast<int>(row) * per;
  while (row < rows) {
    const int b = 4 * i + g;
    float v[8] = {};
    if (b < nb) {
      const vec8_t<T> h = *reinterpret_cast<const vec8_t<T>*>(x + row * x_stride + b * 128 + 8 * gl);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = static_cast<float>(h[e]);
    }
    uint32_t q[1], w[1];
    encode_blocks<1>(v, rotate, gl, q, w);
    if (b < nb) {
      *reinterpret_cast<uint32_t*>(out + row * (C >> 1) + b * 64 + 4 * gl) = q[0];
      if (l16 == 0) scale[b * rows + row] = w[0];
    }
    row += row_step;
    i += step;
    if (i >= per) {
      i -= per;
      ++row;
    }
  }
}

// a / n for a whole number n > 0, inv = 1 / n rounded: the quotient corrected by its exact remainder is the rounded one
// (Markstein; quotients of normal size), in three operations instead of a division's ten.
__device__ __forceinline__ float divide_by(float a, float n, float inv) {
  const float q = a * inv;
  const float c = __builtin_fmaf(__builtin_fmaf(-q, n, a), inv, q);
  return __builtin_isfinite(q) ? c : q;
}

// Column e of the lane's eight (packed in pairs, two bytes each) plus s, in fp32 with one rounding.
template <typename T, int E>
__device__ __forceinline__ float plus(const uint32_t (&w)[4], float s) {
  if constexpr (std::is_same_v<T, half_t>)
    return add_h<E & 1>(w[E >> 1], s);
  else
    return __builtin_bit_cast(float, E & 1 ? w[E >> 1] & 0xffff0000u : w[E >> 1] << 16) + s;
}

// With a norm: a row on G groups of 16 lanes, 4 / G rows a wave; lane group g takes blocks G i + g. The row stays in registers
// as it was loaded, two columns a register, and wide rows form their fp32 values anew in each pass (the sum, the squares, the
// norm's last step): that costs one operation a column, an addition that also converts, where held values spilled (4736
// columns of bf16: 31 us, held 46; 2816 columns: 32.6, held 33.5). gamma and beta (zeros without one) sit in LDS for the
// workgroup's rows, zero past c_real; the first rows load ahead of them. The arithmetic bounds it: 386 vector operations a
// row of 1024 (16 columns a lane at 14 each, 7 of them butterflies; the rest for sums, root, exponents and addresses) keep
// the SIMDs 75 % busy, 27.5 us at 32 800 rows where the rows' bytes take 16. At 2816 columns (5125 rows: 18 us) its 106
// registers leave four waves a SIMD, so 5125 rows are a round and a quarter; and the padding's masks, which the compiler forms
// ahead of the row loop, spill 74 scalar registers into lanes of vector ones: 1297 vector operations a row with what stands
// before the loop, where columns and sums need about 770.
template <typename T, int NI, int G>
__global__ __launch_bounds__(256) void quant_mx4_norm_kernel(const T* __restrict__ x, int64_t x_stride, int64_t rows, int C,
                                                             int c_real, const float* __restrict__ gamma,
                                                             const float* __restrict__ beta, bool centre, float eps,
                                                             bool rotate, uint8_t* __restrict__ out,
                                                             uint32_t* __restrict__ scale) {
  constexpr int RPW = 4 / G, ACCS = 4 / G;  // rows a wave; partial sums a lane
  // gamma as C / 4 float4, the even ones first, then the odd ones (a lane's two lie apart and 16 lanes read 256 bytes in a
  // row, free of bank conflicts), then beta
  extern __shared__ float4_t gb[];
  const int n4 = C >> 2, n8 = C >> 3, nb = C >> 7;
  const int lane = threadIdx.x & 63, g = (lane >> 4) & (G - 1), l16 = lane & 15, gl = l16 ^ (l16 >> 1);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 4 * RPW;
  int64_t row = (static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6)) * RPW + lane / (16 * G);
  uint32_t w[NI][4];
  auto load = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int b = G * i + g;  // lanes past the row hold zeros
      const int4_t h = G == 1 || b < nb ? *reinterpret_cast<const int4_t*>(x + row * x_stride + b * 128 + 8 * gl) : int4_t{};
#pragma unroll
      for (int k = 0; k < 4; ++k) w[i][k] = static_cast<uint32_t>(h[k]);
    }
  };
  if (row < rows) load();
  for (int i = threadIdx.x; i < n4; i += 256) {
    gb[(i & 1) * n8 + (i >> 1)] = reinterpret_cast<const float4_t*>(gamma)[i];
    gb[n4 + (i & 1) * n8 + (i >> 1)] = beta ? reinterpret_cast<const float4_t*>(beta)[i] : float4_t{};
  }
  __syncthreads();
  const float n = static_cast<float>(c_real), inv_n = 1.f / n;
  const int real = c_real - g * 128 - 8 * gl;  // the lane's columns of block G i + g below c_real: real - 128 G i, 0 .. 8
  // x + s for the lane's columns of block group i into d, zero past c_real; only groups that reach past it mask (uniform)
  auto shifted = [&](int i, float s, float (&d)[8]) __attribute__((always_inline)) {
    d[0] = plus<T, 0>(w[i], s), d[1] = plus<T, 1>(w[i], s), d[2] = plus<T, 2>(w[i], s), d[3] = plus<T, 3>(w[i], s);
    d[4] = plus<T, 4>(w[i], s), d[5] = plus<T, 5>(w[i], s), d[6] = plus<T, 6>(w[i], s), d[7] = plus<T, 7>(w[i], s);
    if ((G * i + G) * 128 > c_real) {
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = e < real - 128 * G * i ? d[e] : 0.f;
    }
  };
  // Hides that the words are the previous pass's: without it the compiler keeps that pass's fp32 values in registers.
  auto anew = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) asm("" : "+v"(w[i][k]));
  };
  // the 64 partial sums of a row folded in halves
  auto fold = [](const float (&a)[ACCS]) __attribute__((always_inline)) {
    float t;
    if constexpr (G == 1) {
      t = (a[0] + a[2]) + (a[1] + a[3]);
    } else if constexpr (G == 2) {
      t = a[0] + a[1];
      t = t + swz_xor16(t);
    } else {
      t = a[0] + xor_shuffle(a[0], 32);
      t = t + swz_xor16(t);
    }
    t = t + dpp<DPP_XOR15>(t);
    t = t + dpp<DPP_XOR7>(t);
    t = t + dpp<DPP_XOR3>(t);
    return t + dpp<DPP_XOR1>(t);
  };
  while (row < rows) {
    float minus = 0.f;  // minus the mean
    if (centre) {
      float s[ACCS] = {};
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        float& a = s[i % ACCS];
        if ((G * i + G) * 128 > c_real) {
          float d[8];
          shifted(i, 0.f, d);
#pragma unroll
          for (int e = 0; e < 8; ++e) a = a + d[e];
        } else {
          a = plus<T, 0>(w[i], a), a = plus<T, 1>(w[i], a), a = plus<T, 2>(w[i], a), a = plus<T, 3>(w[i], a);
          a = plus<T, 4>(w[i], a), a = plus<T, 5>(w[i], a), a = plus<T, 6>(w[i], a), a = plus<T, 7>(w[i], a);
        }
      }
      minus = -divide_by(fold(s), n, inv_n);
      anew();
    }
    float sq[ACCS] = {};
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      float d[8];
      shifted(i, minus, d);
#pragma unroll
      for (int e = 0; e < 8; ++e) sq[i % ACCS] = __builtin_fmaf(d[e], d[e], sq[i % ACCS]);
    }
    const float rstd = 1.f / sqrtf(divide_by(fold(sq), n, inv_n) + eps);
    if constexpr (NI > 4) anew();  // up to 32 columns a lane stay in fp32: no gain from more waves there
    int first = g * 16 + gl;  // the lane's even float4 of its first block; opaque: else gamma and beta stay in registers
    asm volatile("" : "+v"(first));
    // two block groups at a time (one at the end of an odd count): the butterflies' wait states are shared
    auto finish = [&](auto count, int i0) __attribute__((always_inline)) {
      constexpr int N = decltype(count)::value;
      float v[8 * N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int b = G * (i0 + j) + g;
        float d[8];
        shifted(i0 + j, minus, d);
        const int c = G == 1 || b < nb ? first + 16 * G * (i0 + j) : 0;
        const float4_t g0 = gb[c], g1 = gb[n8 + c], b0 = gb[n4 + c], b1 = gb[n4 + n8 + c];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[8 * j + e] = __builtin_fmaf(d[e] * rstd, g0[e], b0[e]);
          v[8 * j + 4 + e] = __builtin_fmaf(d[4 + e] * rstd, g1[e], b1[e]);
        }
      }
      uint32_t q[N], word[N];
      encode_blocks<N>(v, rotate, gl, q, word);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int b = G * (i0 + j) + g;
        if (G == 1 || b < nb) {
          *reinterpret_cast<uint32_t*>(out + row * (C >> 1) + b * 64 + 4 * gl) = q[j];
          if (l16 == 0) scale[b * rows + row] = word[j];
        }
      }
    };
#pragma unroll
    for (int i = 0; i + 1 < NI; i += 2) finish(std::integral_constant<int, 2>{}, i);
    if constexpr (NI & 1) finish(std::integral_constant<int, 1>{}, NI - 1);
    row += stride;
    if (row < rows) load();
  }
}

// 2^(e - 127) of an exponent byte, by its bits; 255 is not a number.
__device__ __forceinline__ float e8m0(uint32_t e) {
  return __builtin_bit_cast(float, e == 255 ? 0x7fc00000u : (e == 0 ? 0x00400000u : e << 23));
}

// The values of the codes: each thread 8 columns of a row, in stores that stream past L2 (32 800 x 1024 with the quantization
// before it 43.9 -> 41.2 us; the codes' own stores do not: 4 bytes a lane run slower so). Bound by its bytes: 85 MB in 15 us.
template <typename T>
__global__ __launch_bounds__(256) void dequant_mx4_kernel(const uint8_t* __restrict__ codes,
                                                          const uint32_t* __restrict__ scale, int64_t rows, int C,
                                                          T* __restrict__ out) {
  const int per = C >> 3, threads = static_cast<int>(gridDim.x) * 256;
  const int row_step = threads / per, step = threads - row_step * per;
  int64_t row = (static_cast<int>(blockIdx.x) * 256 + static_cast<int>(threadIdx.x)) / per;
  int c = static_cast<int>(blockIdx.x) * 256 + static_cast<int>(threadIdx.x) - static_cast<int>(row) * per;
  while (row < rows) {
    const int64_t i = row * per + c;
    const uint32_t q = *reinterpret_cast<const uint32_t*>(codes + 4 * i);
    const float f = e8m0((scale[(c >> 4) * rows + row] >> (8 * ((c >> 2) & 3))) & 0xff);
    vec8_t<T> o;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // magnitudes 0, 1/2, 1, 3/2, 2, 3, 4, 6: the code's bits shifted into an fp32's exponent and mantissa, times 2^126
      const uint32_t m = (q >> (4 * e)) & 7, s = (q >> (4 * e + 3)) & 1;
      const float mag = __builtin_bit_cast(float, m << 22) * 0x1p126f;
      o[e] = static_cast<T>((s ? -mag : mag) * f);
    }
    __builtin_nontemporal_store(o, reinterpret_cast<vec8_t<T>*>(out + 8 * i));
    row += row_step;
    c += step;
    if (c >= per) {
      c -= per;
      ++row;
    }
  }
}

static unsigned mx4_grid(const void* kernel, size_t smem, int64_t blocks) {
  int64_t cap = resident_blocks(kernel, 256, smem);
  if (cap <= 0) cap = 1024;
  return static_cast<unsigned>(std::min(blocks, cap));
}

template <typename T, int NI, int G>
static void launch_quant_norm(hipStream_t st, const void* x, int64_t xs, int64_t rows, int C, int c_real, const float* g,
                              const float* b, bool centre, float eps, bool rotate, uint8_t* out, uint32_t* scale) {
  const size_t smem = 2 * C * sizeof(float);
  constexpr int ROWS = 4 * (4 / G);  // of a workgroup at once
  const void* k = reinterpret_cast<const void*>(&quant_mx4_norm_kernel<T, NI, G>);
  quant_mx4_norm_kernel<T, NI, G><<<mx4_grid(k, smem, (rows + ROWS - 1) / ROWS), 256, smem, st>>>(
      static_cast<const T*>(x), xs, rows, C, c_real, g, b, centre, eps, rotate, out, scale);
}

// Lane groups a row: four (a wave a row) where the rows are few or wide, or four divides the blocks; in narrow rows two or one
// leave no group idle (768 columns of 32 800 rows: 21.2 us on two groups, 28.1 on four; 640: 16.9 on one, 23.7 on four; 2816
// columns of 12 000 rows: 32.6 on four, 34.1 on two).
static int quant_groups(int64_t rows, int nb) {
  if (rows < 4096 || nb % 4 == 0 || nb > 11) return 4;
  return nb % 2 == 0 ? 2 : 1;
}

template <typename T>
static void launch_quant(hipStream_t st, const void* x, int64_t xs, int64_t rows, int C, int c_real, int norm,
                         const float* g, const float* b, float eps, bool rotate, uint8_t* out, uint32_t* scale) {
  const int nb = C / 128;
  if (norm == FF_NORM_NONE) {
    const int64_t items = rows * ((nb + 3) / 4);
    const void* k = reinterpret_cast<const void*>(&quant_mx4_kernel<T>);
    quant_mx4_kernel<T><<<mx4_grid(k, 0, (items + 3) / 4), 256, 0, st>>>(static_cast<const T*>(x), xs, rows, C, rotate, out,
                                                                        scale);
    return;
  }
  const bool centre = norm == FF_NORM_LAYER;
  const int G = quant_groups(rows, nb);
  switch (100 * G + (nb + G - 1) / G) {
#define FF_MX4_CASE(GG, N)   case 100 * GG + N: launch_quant_norm<T, N, GG>(st, x, xs, rows, C, c_real, g, b, centre, eps, rotate, out, scale); break;
    FF_MX4_CASE(1, 1) FF_MX4_CASE(1, 3) FF_MX4_CASE(1, 5) FF_MX4_CASE(1, 7) FF_MX4_CASE(1, 9) FF_MX4_CASE(1, 11)
    FF_MX4_CASE(2, 1) FF_MX4_CASE(2, 3) FF_MX4_CASE(2, 5)
    FF_MX4_CASE(4, 1) FF_MX4_CASE(4, 2) FF_MX4_CASE(4, 3) FF_MX4_CASE(4, 4) FF_MX4_CASE(4, 5) FF_MX4_CASE(4, 6)
    FF_MX4_CASE(4, 7) FF_MX4_CASE(4, 8) FF_MX4_CASE(4, 9) FF_MX4_CASE(4, 10) FF_MX4_CASE(4, 11) FF_MX4_CASE(4, 12)
#undef FF_MX4_CASE
    default: break;
  }
}

}  // namespace ff

using namespace ff;

static bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

extern "C" int ff_quant_mx4(const void* x, int dtype, int64_t T, int64_t C, int64_t x_stride, int rotate, int norm,
                            int64_t c_real, const float* gamma, const float* beta, float eps, uint8_t* out,
                            uint32_t* scale, void* stream) {
  clear_error();
  if (dtype != FF_F16 && dtype != FF_BF16) return fail(FF_EINVAL, "quant_mx4: x must be fp16 or bf16");
  if (T < 0 || T > 0x7fffffff) return fail(FF_EINVAL, "quant_mx4: need 0 <= T < 2^31");
  if (C <= 0 || C % 128 != 0 || C > 6144)
    return fail(FF_EINVAL, "quant_mx4: C must be a positive multiple of 128, at most 6144");
  if (x_stride < C || x_stride % 8 != 0) return fail(FF_EINVAL, "quant_mx4: need x_stride >= C, a multiple of 8");
  if (rotate != 0 && rotate != 1) return fail(FF_EINVAL, "quant_mx4: rotate must be 0 or 1");
  if (norm != FF_NORM_NONE && norm != FF_NORM_RMS && norm != FF_NORM_LAYER)
    return fail(FF_EINVAL, "quant_mx4: unknown norm");
  if ((gamma != nullptr) != (norm != FF_NORM_NONE)) return fail(FF_EINVAL, "quant_mx4: gamma goes with a norm");
  if ((beta != nullptr) != (norm == FF_NORM_LAYER)) return fail(FF_EINVAL, "quant_mx4: beta goes with the LayerNorm");
  if (norm != FF_NORM_NONE && (c_real <= 0 || c_real > C)) return fail(FF_EINVAL, "quant_mx4: need 0 < c_real <= C");
  if (norm != FF_NORM_NONE && !(eps > 0.f)) return fail(FF_EINVAL, "quant_mx4: eps must be > 0");
  if (T == 0) return FF_OK;
  if (!x || !out || !scale) return fail(FF_EINVAL, "quant_mx4: null pointer");
  if (!aligned(x, 16) || !aligned(out, 4) || !aligned(scale, 4) || !aligned(gamma, 16) || !aligned(beta, 16))
    return fail(FF_EINVAL, "quant_mx4: misaligned pointer");
  // rows are read by workgroups that run while others write theirs
  const Extent codes = range(out, T * (C / 2)), words = range(scale, T * (C / 32));
  bool clear = clear_of(codes, words);
  for (const Extent& e : {Extent{reinterpret_cast<uintptr_t>(x), {T, 1}, {2 * x_stride, 0}, 2 * C}, range(gamma, 4 * C),
                          range(beta, 4 * C)})
    clear = clear && (e.at == 0 || (clear_of(codes, e) && clear_of(words, e)));
  if (!clear) return fail(FF_EINVAL, "quant_mx4: an output overlaps the other one or what is read");
  const hipStream_t st = as_stream(stream);
  const int Ci = static_cast<int>(C), cr = static_cast<int>(c_real);
  if (dtype == FF_F16)
    launch_quant<half_t>(st, x, x_stride, T, Ci, cr, norm, gamma, beta, eps, rotate != 0, out, scale);
  else
    launch_quant<bf16_t>(st, x, x_stride, T, Ci, cr, norm, gamma, beta, eps, rotate != 0, out, scale);
  return check_launch("quant_mx4");
}

extern "C" int ff_dequant_mx4(const uint8_t* codes, const uint32_t* scale, int64_t T, int64_t C, void* out, int dtype,
                              void* stream) {
  clear_error();
  if (dtype != FF_F16 && dtype != FF_BF16 && dtype != FF_F32)
    return fail(FF_EINVAL, "dequant_mx4: out must be fp16, bf16 or fp32");
  if (T < 0 || T > 0x7fffffff) return fail(FF_EINVAL, "dequant_mx4: need 0 <= T < 2^31");
  if (C <= 0 || C % 128 != 0 || C > (1 << 22))
    return fail(FF_EINVAL, "dequant_mx4: C must be a positive multiple of 128, at most 2^22");
  if (T == 0) return FF_OK;
  if (!codes || !scale || !out) return fail(FF_EINVAL, "dequant_mx4: null pointer");
  if (!aligned(codes, 4) || !aligned(scale, 4) || !aligned(out, 16))
    return fail(FF_EINVAL, "dequant_mx4: misaligned pointer");
  const Extent to = range(out, T * C * (dtype == FF_F32 ? 4 : 2));
  if (!clear_of(to, range(codes, T * (C / 2))) || !clear_of(to, range(scale, T * (C / 32))))
    return fail(FF_EINVAL, "dequant_mx4: out overlaps the codes or their scale");
  const hipStream_t st = as_stream(stream);
  const int Ci = static_cast<int>(C);
  const int64_t blocks = (T * (C / 8) + 255) / 256;
#define FF_DEQUANT(TT)                                                                                              \
  dequant_mx4_kernel<TT><<<mx4_grid(reinterpret_cast<const void*>(&dequant_mx4_kernel<TT>), 0, blocks), 256, 0, st>>>( \
      codes, scale, T, Ci, static_cast<TT*>(out))
  if (dtype == FF_F16)
    FF_DEQUANT(half_t);
  else if (dtype == FF_BF16)
    FF_DEQUANT(bf16_t);
  else
    FF_DEQUANT(float);
#undef FF_DEQUANT
  return check_launch("dequant_mx4");
}
