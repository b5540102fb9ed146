// The norm of each head's query and key and their rotation by position, in one pass.
//
// Per token t and head, over the head's D columns: RMSNorm x / sqrt(mean(x^2) + eps) gamma, or LayerNorm
// (x - mean) / sqrt(var + eps) gamma + beta, or no norm; then the first R columns are rotated by the angles of table row
// p = positions[t] (or t mod L): the pair (x0, x1) becomes (x0 cos - x1 sin, x0 sin + x1 cos), pairs being neighbours
// (2 i, 2 i + 1) or halves (i, i + R / 2); q is then multiplied by q_scale. All of it in fp32 with one rounding at the store.
//
// HBM-bound: 4 bytes a column (read and written once). A head is VEC columns a lane in a group of 2^k lanes of one wave: its
// sums are lane permutes, its neighbour pairs in-lane and its halves one permute away.
#include <algorithm>

#include "common.h"

namespace ff {

struct QkArgs {
  const void* x[2];       // q, k
  void* out[2];
  int64_t xt[2], xh[2];   // strides in elements: token, head
  int64_t ot[2], oh[2];
  const float* gamma[2];
  const float* beta[2];
  const float* cos;  // [L, R / 2]
  const float* sin;
  const void* pos;   // int32 or int64 [T], or null: t mod L
  int pos64, tokens, heads, kv, D, R, L, norm;
  int lanes;  // lanes a head: the power of two from D / VEC up
  float eps, q_scale;
};

template <typename T, int VEC>
using vec_t = T __attribute__((ext_vector_type(VEC)));

template <typename T, int VEC, bool PAIRS>
__global__ __launch_bounds__(256) void qk_norm_kernel(const QkArgs a) {
  const int lanes = a.lanes, c = threadIdx.x & (lanes - 1);
  const int all = a.heads + a.kv, per = 256 / lanes;
  const bool in = c * VEC < a.D;  // lanes past the head hold zeros and take part in the permutes
  const int half = a.R / 2, hc = half / VEC;
  const uint32_t n = static_cast<uint32_t>(a.tokens) * all;
  for (uint32_t i0 = blockIdx.x * per; i0 < n; i0 += gridDim.x * per) {
    const uint32_t i = i0 + threadIdx.x / lanes;
    const bool live = i < n;
    const uint32_t t = live ? i / all : 0;
    const int h = live ? i - t * all : 0;
    const int which = h >= a.heads, hh = which ? h - a.heads : h;
    float v[VEC] = {};
    if (live && in) {
      const T* p = static_cast<const T*>(a.x[which]) + t * a.xt[which] + hh * a.xh[which] + c * VEC;
      const vec_t<T, VEC> raw = *reinterpret_cast<const vec_t<T, VEC>*>(p);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = static_cast<float>(raw[e]);
    }
    int64_t row = t % a.L;
    if (a.pos && live)
      row = a.pos64 ? static_cast<const int64_t*>(a.pos)[t] : static_cast<const int32_t*>(a.pos)[t];
    const bool known = row >= 0 && row < a.L;
    if (a.norm != FF_NORM_NONE) {
      const float d = static_cast<float>(a.D);
      if (a.norm == FF_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < VEC; ++e) s = s + v[e];
        for (int m = lanes >> 1; m; m >>= 1) s = s + xor_shuffle(s, m);
        const float mean = s / d;
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = in ? v[e] - mean : 0.f;
      }
      float sq = 0.f;
#pragma unroll
      for (int e = 0; e < VEC; ++e) sq = __builtin_fmaf(v[e], v[e], sq);
      for (int m = lanes >> 1; m; m >>= 1) sq = sq + xor_shuffle(sq, m);
      const float rstd = 1.f / sqrtf(sq / d + a.eps);
      const float* g = a.gamma[which];
      const float* b = a.beta[which];
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        v[e] = in ? __builtin_fmaf(v[e] * rstd, g[c * VEC + e], b ? b[c * VEC + e] : 0.f) : 0.f;
    }
    if constexpr (PAIRS) {
      if (known && c * VEC < a.R) {
        const float* co = a.cos + row * half + c * (VEC / 2);
        const float* si = a.sin + row * half + c * (VEC / 2);
#pragma unroll
        for (int e = 0; e < VEC / 2; ++e) {
          const float x0 = v[2 * e], x1 = v[2 * e + 1];
          v[2 * e] = x0 * co[e] - x1 * si[e];
          v[2 * e + 1] = x0 * si[e] + x1 * co[e];
        }
      }
    } else {
      const bool lo = c < hc, turned = c < 2 * hc;
      const int lane = threadIdx.x & 63, from = turned ? (lo ? lane + hc : lane - hc) : lane;
      float w[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) w[e] = __shfl(v[e], from, 64);
      if (known && turned) {
        const float* co = a.cos + row * half + (lo ? c : c - hc) * VEC;
        const float* si = a.sin + row * half + (lo ? c : c - hc) * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = lo ? v[e] * co[e] - w[e] * si[e] : w[e] * si[e] + v[e] * co[e];
      }
    }
    if (live && in) {
      vec_t<T, VEC> o;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float y = which ? v[e] : v[e] * a.q_scale;
        if (!known) y = __builtin_nanf("");  // no such row in the table
        o[e] = static_cast<T>(y);
      }
      T* p = static_cast<T*>(a.out[which]) + t * a.ot[which] + hh * a.oh[which] + c * VEC;
      *reinterpret_cast<vec_t<T, VEC>*>(p) = o;
    }
  }
}

template <typename T, int VEC>
static void launch_qk(const QkArgs& a, bool pairs, hipStream_t st) {
  const int64_t groups = (static_cast<int64_t>(a.tokens) * (a.heads + a.kv) * a.lanes + 255) / 256;
  const void* k = pairs ? reinterpret_cast<const void*>(&qk_norm_kernel<T, VEC, true>)
                        : reinterpret_cast<const void*>(&qk_norm_kernel<T, VEC, false>);
  int64_t cap = resident_blocks(k, 256, 0);
  if (cap <= 0) cap = 1024;
  const dim3 grid(static_cast<unsigned>(std::min(groups, cap)));
  if (pairs)
    qk_norm_kernel<T, VEC, true><<<grid, 256, 0, st>>>(a);
  else
    qk_norm_kernel<T, VEC, false><<<grid, 256, 0, st>>>(a);
}

}  // namespace ff

using namespace ff;

extern "C" int ff_qk_norm_rope(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token,
                               int64_t k_head, void* q_out, int64_t qo_token, int64_t qo_head, void* k_out,
                               int64_t ko_token, int64_t ko_head, int dtype, int64_t T, int64_t heads, int64_t kv_heads,
                               int64_t D, int norm, const float* q_gamma, const float* k_gamma, const float* q_beta,
                               const float* k_beta, float eps, const float* rope_cos, const float* rope_sin,
                               int64_t rope_len, int64_t R, int pairs, const void* positions, int pos64, float q_scale,
                               void* stream) {
  clear_error();
  if (dtype != FF_F16 && dtype != FF_BF16) return fail(FF_EINVAL, "qk_norm_rope: q and k must be fp16 or bf16");
  if (D <= 0 || D % 8 != 0 || D > 256)
    return fail(FF_EINVAL, "qk_norm_rope: heads must be a multiple of 8 columns, at most 256");
  if (R <= 0 || R % 8 != 0 || R > D)
    return fail(FF_EINVAL, "qk_norm_rope: the rotated columns must be a multiple of 8, at most the head's");
  if (heads <= 0 || kv_heads <= 0 || heads > 65535 || kv_heads > 65535)
    return fail(FF_EINVAL, "qk_norm_rope: need 0 < heads, kv_heads <= 65535");
  if (T < 0 || T >= (int64_t(1) << 31) || T * (heads + kv_heads) >= (int64_t(1) << 31))
    return fail(FF_EINVAL, "qk_norm_rope: need 0 <= T and T * (heads + kv_heads) < 2^31");
  if (rope_len <= 0 || rope_len > 0x7fffffff) return fail(FF_EINVAL, "qk_norm_rope: need 0 < rope_len < 2^31");
  if (norm != FF_NORM_NONE && norm != FF_NORM_RMS && norm != FF_NORM_LAYER)
    return fail(FF_EINVAL, "qk_norm_rope: unknown norm");
  const bool normed = norm != FF_NORM_NONE, centred = norm == FF_NORM_LAYER;
  if ((q_gamma != nullptr) != normed || (k_gamma != nullptr) != normed)
    return fail(FF_EINVAL, "qk_norm_rope: q_gamma and k_gamma go with a norm");
  if ((q_beta != nullptr) != centred || (k_beta != nullptr) != centred)
    return fail(FF_EINVAL, "qk_norm_rope: q_beta and k_beta go with the LayerNorm");
  if (normed && !(eps > 0.f)) return fail(FF_EINVAL, "qk_norm_rope: eps must be > 0");
  if (T == 0) return FF_OK;
  if (!q || !k || !q_out || !k_out || !rope_cos || !rope_sin) return fail(FF_EINVAL, "qk_norm_rope: null pointer");
  uint64_t low = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(q_out) |
                 reinterpret_cast<uintptr_t>(k_out);
  for (int64_t s : {q_token, q_head, k_token, k_head, qo_token, qo_head, ko_token, ko_head}) {
    if (s < 0) return fail(FF_EINVAL, "qk_norm_rope: strides must not be negative");
    low |= static_cast<uint64_t>(s) * 2;
  }
  if ((low & 7) || ((reinterpret_cast<uintptr_t>(rope_cos) | reinterpret_cast<uintptr_t>(rope_sin)) & 15) ||
      (reinterpret_cast<uintptr_t>(positions) & (pos64 ? 7 : 3)))
    return fail(FF_EINVAL, "qk_norm_rope: misaligned pointer or stride (q and k: multiples of 8 bytes)");
  // rows of an output must not overlap (a size of one has no stride)
  auto overlaps = [&](int64_t token, int64_t head, int64_t n) {
    if (T > 1 && n > 1) {
      const bool th = token >= head;
      const int64_t small = th ? head : token, big = th ? token : head, count = th ? n : T;
      return small < D || big < small * (count - 1) + D;
    }
    return (T > 1 && token < D) || (n > 1 && head < D);
  };
  if (overlaps(qo_token, qo_head, heads) || overlaps(ko_token, ko_head, kv_heads))
    return fail(FF_EINVAL, "qk_norm_rope: the rows of an output overlap");
  QkArgs a{{q, k}, {q_out, k_out}, {q_token, k_token}, {q_head, k_head}, {qo_token, ko_token}, {qo_head, ko_head},
           {q_gamma, k_gamma}, {q_beta, k_beta}, rope_cos, rope_sin, positions, pos64, static_cast<int>(T),
           static_cast<int>(heads), static_cast<int>(kv_heads), static_cast<int>(D), static_cast<int>(R),
           static_cast<int>(rope_len), norm, 0, eps, q_scale};
  const bool wide = (low & 15) == 0 && (pairs || R % 16 == 0);
  a.lanes = 1;
  while (a.lanes * (wide ? 8 : 4) < D) a.lanes *= 2;
  const hipStream_t st = as_stream(stream);
  if (dtype == FF_F16)
    wide ? launch_qk<half_t, 8>(a, pairs != 0, st) : launch_qk<half_t, 4>(a, pairs != 0, st);
  else
    wide ? launch_qk<bf16_t, 8>(a, pairs != 0, st) : launch_qk<bf16_t, 4>(a, pairs != 0, st);
  return check_launch("qk_norm_rope");
}
