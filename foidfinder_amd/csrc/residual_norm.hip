// A block's output into the residual stream, between the block's post-norm and the next block's pre-norm, in one pass:
//   x_out = x + scale gate N_post(y),   h = N_pre(x_out),
// N being RMSNorm v / sqrt(mean(v^2) + eps) gamma, LayerNorm (v - mean) / sqrt(var + eps) gamma + beta, or nothing; gate is a
// row for each run of tokens (one: a layer scale; one a sequence; one a token), or 1. All of it in fp32; x_out and h are rounded
// once each, h from the unrounded x_out.
//
// HBM-bound: 8 bytes a column (x, y read, x_out, h written). LANES lanes hold a row, 16 bytes a lane and chunk; a group of lanes
// keeps to its columns and strides over the rows, so that gammas, betas and a single gate row stay in registers (4 to 20 bytes a
// column; past 8192 columns gammas and betas are read for each row, from the caches). The next row loads under this one's
// arithmetic. Sums: within a wave by DPP; a row of several waves leaves each wave's sum and squares about its own mean in LDS
// and every wave joins them (counts and means known, no cancellation), one barrier a norm.
// Measured: 32 800 x 1024 fp16 with two LayerNorms and a gate row 51.5 us (5.2 TB/s), 9001 x 4096 bf16 with two RMS norms 55.7
// (5.3); a copy of 1 GiB reaches 5.07, of 256 MB 5.42. Gates of their own for each token, loaded in their row and not before
// it, 62 (fp16, 10 bytes a column: 5.4) and 74 (fp32, 12: 5.4), with a post-norm or without; for each of 32 sequences 46, as
// without a gate. 4028 rows of 8192 columns 48 us (5.5 TB/s), 4024 of 8200 77 and 2014 of 16 384 61 (4.4). With the norms
// chosen by branches in the row loop, whose parameters' loads it then waited for: 71. A single row: 2.5 us.
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace ff {

struct ResidualArgs {
  const void *x, *y, *gate;
  void *x_out, *h;
  int64_t xs, ys, os, hs;  // row strides in elements
  const float *post_g, *post_b, *pre_g, *pre_b;
  int rows, width, per_gate, gate_f32;  // per_gate: rows that share a gate row
  float scale, eps;
};

// Sum over groups of LANES <= 64 lanes, in each of them.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
  v = v + dpp<DPP_XOR1>(v);
  v = v + dpp<DPP_XOR3>(v);
  v = v + dpp<DPP_XOR7>(v);
  v = v + dpp<DPP_XOR15>(v);
  if constexpr (LANES > 16) v = v + swz_xor16(v);
  if constexpr (LANES > 32) v = v + xor_shuffle(v, 32);
  return v;
}

// 1 / sqrt(v), about 1 ulp; v_rsq_f32 takes a subnormal number for zero.
__device__ __forceinline__ float inv_root(float v) {
  return v < 0x1p-126f ? __builtin_amdgcn_rsqf(v * 0x1p24f) * 0x1p12f : __builtin_amdgcn_rsqf(v);
}

// sum / n, rounded once; inv: 1 / n, whose own rounding the quotient would keep. Equal elements, whose sum is exact, then have their
// own value as mean: what is left of it would be divided by a variance of nothing.
__device__ __forceinline__ float mean_of(float sum, float n, float inv) {
  const float q = sum * inv;
  return __builtin_fmaf(__builtin_fmaf(-q, n, sum), inv, q);
}

template <typename T, int LANES, int CHUNKS, int POST, int PRE>
__global__ __launch_bounds__(LANES <= 64 ? 256 : LANES) void residual_norm_kernel(const ResidualArgs a) {
  constexpr int THREADS = LANES <= 64 ? 256 : LANES, GROUPS = THREADS / LANES, WIDTH = LANES < 64 ? LANES : 64;
  constexpr int WPR = LANES / WIDTH;  // waves a row
  constexpr bool KEEP = CHUNKS <= 2;  // the parameters stay in registers
  typedef vec8_t<T> T8;
  __shared__ float2 joint[2][THREADS / 64];
  const int lane = threadIdx.x % LANES, wave = threadIdx.x / 64;
  const int step = static_cast<int>(gridDim.x) * GROUPS;
  int row = static_cast<int>(blockIdx.x) * GROUPS + threadIdx.x / LANES;
  if (row >= a.rows) return;  // (a row of several waves is its block's only one)
  int col[CHUNKS];
  bool in[CHUNKS];
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) {
    in[i] = 8 * (i * LANES + lane) < a.width;
    col[i] = in[i] ? 8 * (i * LANES + lane) : 0;  // lanes past the row load its first columns, which the sums leave out
  }
  const float inv_n = 1.f / static_cast<float>(a.width);

  // columns of wave w of the row
  auto columns = [&](int w) __attribute__((always_inline)) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) n += min(max(a.width - 8 * (i * LANES + w * 64), 0), 512);
    return n;
  };
  const int mine = WPR > 1 ? columns(wave) : a.width;
  const float own_n = static_cast<float>(mine), own = mine ? 1.f / own_n : 0.f;

  float post_g[CHUNKS][8], post_b[CHUNKS][8], pre_g[CHUNKS][8], pre_b[CHUNKS][8], factor[CHUNKS][8];
  // The compiler's wait for these loads stands here, before the loop: in it, the same counter holds the next row's loads.
  auto settle = [](float (&k)[CHUNKS][8]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) asm volatile("" : "+v"(k[i][e]));
  };
  auto keep = [&](const float* p, float (&k)[CHUNKS][8]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) k[i][e] = p[col[i] + e];
    settle(k);
  };
  auto gate_at = [&](int64_t r, int i, float (&f)[8]) __attribute__((always_inline)) {
    if (a.gate_f32) {
      const float* g = static_cast<const float*>(a.gate) + r * a.width + col[i];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = g[e];
    } else {
      const T8 g = *reinterpret_cast<const T8*>(static_cast<const T*>(a.gate) + r * a.width + col[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = static_cast<float>(g[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= a.scale;
  };
  const bool gate_moves = a.gate && a.per_gate < a.rows;
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) factor[i][e] = a.scale;
    if (a.gate && !gate_moves) gate_at(0, i, factor[i]);
  }
  settle(factor);
  if constexpr (KEEP && POST != FF_NORM_NONE) keep(a.post_g, post_g);
  if constexpr (KEEP && POST == FF_NORM_LAYER) keep(a.post_b, post_b);
  if constexpr (KEEP && PRE != FF_NORM_NONE) keep(a.pre_g, pre_g);
  if constexpr (KEEP && PRE == FF_NORM_LAYER) keep(a.pre_b, pre_b);

  // Sum over the wave's lanes and chunks of f(chunk's values); chunks past the row count for nothing, whatever they hold.
  auto sum_of = [&](float (&v)[CHUNKS][8], auto f) __attribute__((always_inline)) {
    float all = 0.f;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) s = f(s, v[i][e]);
      all = all + (in[i] ? s : 0.f);
    }
    return lanes_sum<WIDTH>(all);
  };
  int turn = 0;
  // The norm of v in its place.
  auto norm = [&](float (&v)[CHUNKS][8], auto kind, const float* g, const float* b, float (&kg)[CHUNKS][8],
                  float (&kb)[CHUNKS][8]) __attribute__((always_inline)) {
    constexpr bool CENTRED = decltype(kind)::value == FF_NORM_LAYER;
    float sum = 0.f, centre = 0.f;
    if constexpr (CENTRED) {
      sum = sum_of(v, [](float s, float x) { return s + x; });
      centre = mean_of(sum, own_n, own);
    }
    float sq = sum_of(v, [centre](float s, float x) {
      const float d = CENTRED ? x - centre : x;
      return __builtin_fmaf(d, d, s);
    });
    if constexpr (WPR > 1) {
      if (threadIdx.x % 64 == 0) joint[turn][wave] = float2{sum, sq};
      __syncthreads();
      if constexpr (CENTRED) {
        float all = 0.f;
#pragma unroll
        for (int w = 0; w < WPR; ++w) all = all + joint[turn][w].x;
        centre = mean_of(all, static_cast<float>(a.width), inv_n);
      }
      sq = 0.f;
#pragma unroll
      for (int w = 0; w < WPR; ++w) {
        const float2 j = joint[turn][w];
        sq = sq + j.y;
        if constexpr (CENTRED) {
          const float n = static_cast<float>(columns(w));  // 0: of no columns, and j.x is 0
          const float d = __builtin_fmaf(-centre, n, j.x);
          sq = __builtin_fmaf(n > 0.f ? d * __builtin_amdgcn_rcpf(n) : 0.f, d, sq);
        }
      }
      turn ^= 1;  // the next norm writes the other one: its barrier lies between the reads here and the next write
    }
    const float r = inv_root(__builtin_fmaf(sq, inv_n, a.eps));
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float gamma = KEEP ? kg[i][e] : g[col[i] + e];
        if constexpr (CENTRED)
          v[i][e] = __builtin_fmaf((v[i][e] - centre) * r, gamma, KEEP ? kb[i][e] : b[col[i] + e]);
        else
          v[i][e] = v[i][e] * r * gamma;
      }
  };

  const T *x = static_cast<const T*>(a.x), *y = static_cast<const T*>(a.y);
  T *xo = static_cast<T*>(a.x_out), *ho = static_cast<T*>(a.h);
  T8 nx[CHUNKS], ny[CHUNKS];
  auto load = [&](int r) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      nx[i] = *reinterpret_cast<const T8*>(x + r * a.xs + col[i]);
      ny[i] = *reinterpret_cast<const T8*>(y + r * a.ys + col[i]);
    }
  };
  load(row);
  for (;;) {
    float v[CHUNKS][8], s[CHUNKS][8];
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[i][e] = static_cast<float>(ny[i][e]);
        s[i][e] = static_cast<float>(nx[i][e]);
      }
    if (gate_moves)
#pragma unroll
      for (int i = 0; i < CHUNKS; ++i) gate_at(row / a.per_gate, i, factor[i]);
    const int at = row;
    const bool more = row < a.rows - step;
    if (more) {
      row += step;
      load(row);
    }
    if constexpr (POST != FF_NORM_NONE) norm(v, std::integral_constant<int, POST>{}, a.post_g, a.post_b, post_g, post_b);
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      T8 w;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[i][e] = __builtin_fmaf(v[i][e], factor[i][e], s[i][e]);
        w[e] = static_cast<T>(s[i][e]);
      }
      if (in[i])
        __builtin_nontemporal_store(__builtin_bit_cast(int4_t, w), reinterpret_cast<int4_t*>(xo + at * a.os + col[i]));
    }
    if constexpr (PRE != FF_NORM_NONE) {
      norm(s, std::integral_constant<int, PRE>{}, a.pre_g, a.pre_b, pre_g, pre_b);
#pragma unroll
      for (int i = 0; i < CHUNKS; ++i) {
        T8 w;
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = static_cast<T>(s[i][e]);
        if (in[i])
          __builtin_nontemporal_store(__builtin_bit_cast(int4_t, w), reinterpret_cast<int4_t*>(ho + at * a.hs + col[i]));
      }
    }
    if (!more) break;
  }
}

template <typename T, int LANES, int CHUNKS, int POST, int PRE>
static void launch_residual(const ResidualArgs& a, hipStream_t st) {
  constexpr int THREADS = LANES <= 64 ? 256 : LANES, GROUPS = THREADS / LANES;
  int64_t cap = resident_blocks(reinterpret_cast<const void*>(&residual_norm_kernel<T, LANES, CHUNKS, POST, PRE>), THREADS, 0);
  if (cap <= 0) cap = 512;
  const int64_t blocks = std::min<int64_t>((a.rows + GROUPS - 1) / GROUPS, cap);
  residual_norm_kernel<T, LANES, CHUNKS, POST, PRE><<<dim3(static_cast<unsigned>(blocks)), THREADS, 0, st>>>(a);
}

template <typename T, int POST, int PRE>
static void launch_residual_width(const ResidualArgs& a, hipStream_t st) {
  if (a.width <= 128)
    launch_residual<T, 16, 1, POST, PRE>(a, st);
  else if (a.width <= 256)
    launch_residual<T, 16, 2, POST, PRE>(a, st);
  else if (a.width <= 512)
    launch_residual<T, 32, 2, POST, PRE>(a, st);
  else if (a.width <= 1024)
    launch_residual<T, 64, 2, POST, PRE>(a, st);
  else if (a.width <= 2048)
    launch_residual<T, 128, 2, POST, PRE>(a, st);
  else if (a.width <= 4096)
    launch_residual<T, 256, 2, POST, PRE>(a, st);
  else if (a.width <= 8192)
    launch_residual<T, 512, 2, POST, PRE>(a, st);
  else
    launch_residual<T, 512, 4, POST, PRE>(a, st);
}

template <typename T, int POST>
static void launch_residual_pre(const ResidualArgs& a, int pre, hipStream_t st) {
  switch (pre) {
    case FF_NORM_RMS: return launch_residual_width<T, POST, FF_NORM_RMS>(a, st);
    case FF_NORM_LAYER: return launch_residual_width<T, POST, FF_NORM_LAYER>(a, st);
    default: return launch_residual_width<T, POST, FF_NORM_NONE>(a, st);
  }
}

template <typename T>
static void launch_residual_norms(const ResidualArgs& a, int post, int pre, hipStream_t st) {
  switch (post) {
    case FF_NORM_RMS: return launch_residual_pre<T, FF_NORM_RMS>(a, pre, st);
    case FF_NORM_LAYER: return launch_residual_pre<T, FF_NORM_LAYER>(a, pre, st);
    default: return launch_residual_pre<T, FF_NORM_NONE>(a, pre, st);
  }
}

}  // namespace ff

using namespace ff;

extern "C" int ff_residual_norm(const void* x, int64_t x_row, const void* y, int64_t y_row, void* x_out, int64_t xo_row,
                                void* h, int64_t h_row, int dtype, int64_t T, int64_t C, int post, const float* post_gamma,
                                const float* post_beta, int pre, const float* pre_gamma, const float* pre_beta,
                                const void* gate, int64_t gate_rows, int gate_dtype, float scale, float eps, void* stream) {
  clear_error();
  if (dtype != FF_F16 && dtype != FF_BF16) return fail(FF_EINVAL, "residual_norm: x, y and the outputs must be fp16 or bf16");
  if (C <= 0 || C % 8 != 0 || C > 16384)
    return fail(FF_EINVAL, "residual_norm: rows must be a multiple of 8 columns, at most 16384");
  if (T < 0 || T >= (int64_t(1) << 31)) return fail(FF_EINVAL, "residual_norm: need 0 <= T < 2^31");
  for (int n : {post, pre})
    if (n != FF_NORM_NONE && n != FF_NORM_RMS && n != FF_NORM_LAYER) return fail(FF_EINVAL, "residual_norm: unknown norm");
  if ((post_gamma != nullptr) != (post != FF_NORM_NONE) || (pre_gamma != nullptr) != (pre != FF_NORM_NONE))
    return fail(FF_EINVAL, "residual_norm: a gamma goes with its norm");
  if ((post_beta != nullptr) != (post == FF_NORM_LAYER) || (pre_beta != nullptr) != (pre == FF_NORM_LAYER))
    return fail(FF_EINVAL, "residual_norm: a beta goes with its LayerNorm");
  if ((post != FF_NORM_NONE || pre != FF_NORM_NONE) && !(eps > 0.f)) return fail(FF_EINVAL, "residual_norm: eps must be > 0");
  if (gate && gate_dtype != dtype && gate_dtype != FF_F32)
    return fail(FF_EINVAL, "residual_norm: gate must be fp32 or of x's type");
  if (gate && (gate_rows <= 0 || T % gate_rows != 0))
    return fail(FF_EINVAL, "residual_norm: T must be a multiple of the gate's rows");
  if (T == 0) return FF_OK;
  if (!x || !y || !x_out) return fail(FF_EINVAL, "residual_norm: null pointer");
  if ((h != nullptr) != (pre != FF_NORM_NONE)) return fail(FF_EINVAL, "residual_norm: h goes with a pre-norm");
  if (T == 1) x_row = y_row = xo_row = h_row = C;  // a single row's stride says nothing
  if (!h) h_row = C;
  uint64_t low = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(x_out) |
                 reinterpret_cast<uintptr_t>(h) | reinterpret_cast<uintptr_t>(gate);
  for (int64_t s : {x_row, y_row, xo_row, h_row}) {
    if (s < 0) return fail(FF_EINVAL, "residual_norm: strides must not be negative");
    low |= static_cast<uint64_t>(s) * 2;
  }
  if ((low & 15) || ((reinterpret_cast<uintptr_t>(post_gamma) | reinterpret_cast<uintptr_t>(post_beta) |
                      reinterpret_cast<uintptr_t>(pre_gamma) | reinterpret_cast<uintptr_t>(pre_beta)) & 15))
    return fail(FF_EINVAL, "residual_norm: misaligned pointer or stride (multiples of 16 bytes)");
  if (xo_row < C || h_row < C) return fail(FF_EINVAL, "residual_norm: the rows of an output overlap");
  // Rows are read and written by different workgroups, in no order: an output is x or y itself or shares no byte with what is
  // read or with the other output.
  auto rows = [&](const void* p, int64_t stride) {
    return Extent{reinterpret_cast<uintptr_t>(p), {T, 1}, {2 * stride, 0}, 2 * C};
  };
  const Extent in[2] = {rows(x, x_row), rows(y, y_row)}, to[2] = {rows(x_out, xo_row), rows(h, h_row)};
  const Extent read[5] = {range(post_gamma, 4 * C), range(post_beta, 4 * C), range(pre_gamma, 4 * C), range(pre_beta, 4 * C),
                          range(gate, gate_rows * C * (gate_dtype == FF_F32 ? 4 : 2))};
  bool clear = !h || clear_of(to[0], to[1]);
  for (int o = 0; o < (h ? 2 : 1); ++o) {
    for (const Extent& e : in) clear = clear && ((to[o].at == e.at && to[o].pitch[0] == e.pitch[0]) || clear_of(to[o], e));
    for (const Extent& e : read) clear = clear && (e.at == 0 || clear_of(to[o], e));
  }
  if (!clear)
    return fail(FF_EINVAL, "residual_norm: an output overlaps the other one or what is read (x or y, with its stride, may be in "
                           "its place)");
  const ResidualArgs a{x, y, gate, x_out, h, x_row, y_row, xo_row, h_row, post_gamma, post_beta, pre_gamma, pre_beta,
                       static_cast<int>(T), static_cast<int>(C), gate ? static_cast<int>(T / gate_rows) : 1, gate_dtype == FF_F32,
                       scale, eps};
  if (dtype == FF_F16)
    launch_residual_norms<half_t>(a, post, pre, as_stream(stream));
  else
    launch_residual_norms<bf16_t>(a, post, pre, as_stream(stream));
  return check_launch("residual_norm");
}
