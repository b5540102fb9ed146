// The norm of each head's query and key and their rotation by position, in one pass.
//
// Per token t and head, over the head's D columns: RMSNorm x / sqrt(mean(x^2) + eps) gamma, or LayerNorm
// (x - mean) / sqrt(var + eps) gamma + beta, or no norm; then the first R columns are rotated by the angles of table row
// p = positions[t] (or t mod L): the pair (x0, x1) becomes (x0 cos - x1 sin, x0 sin + x1 cos), pairs being neighbours
// (2 i, 2 i + 1) or halves (i, i + R / 2); q is then multiplied by q_scale. All of it in fp32 with one rounding at the store.
//
// HBM-bound: 4 bytes a column (read and written once). A lane holds 8 columns of a head in two pieces of 4 that rotate in
// the lane: neighbour pairs lie in 8 columns in a row, halves in columns 4 c .. and R / 2 + 4 c .., so the arithmetic has no
// exchange between lanes but the sums' (DPP), and lane c takes the table entries 4 c .. 4 c + 3. Halves still move 16 bytes a lane
// where that is aligned: two lanes load two pieces in a row each and swap one (32 800 tokens x 32 heads of 64, RMS: 54 us,
// 65.6 in 8-byte accesses). A group of 8, 16 or 32 lanes holds a head; it keeps its head and strides over the tokens, so gamma and beta
// stay in registers and nothing is divided in the loop. The next token's columns and entries load under this one's arithmetic,
// its position one token earlier still. Stores stream past L2 (53.5 -> 50.7 us), loads do not (50.0, but the products before
// and after them then run 5 % slower).
//
// Measured: 32 800 tokens x (16 + 16) x 64 fp16 LayerNorm, pairs, 50.7 us, 5.3 TB/s read and written; 9001 x (32 + 8) x 128 bf16
// RMS, halves, 37.5, 5.0 TB/s; one token 8.8, the host's share of a call.
#include <algorithm>

#include "common.h"

namespace ff {

struct QkArgs {
  const void* x[2];  // q, k
  void* out[2];
  int64_t xt[2], xh[2];  // strides in elements: token, head
  int64_t ot[2], oh[2];
  const float* gamma[2];
  const float* beta[2];
  const float* cos;  // [L, R / 2]
  const float* sin;
  const void* pos;  // int32 or int64 [T], or null: t mod L
  int pos64, tokens, heads[2], D, R, L, norm, wide;
  float eps, scale[2];
};

// Sum over groups of LANES lanes, in each of them.
template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
  v = v + dpp<DPP_XOR1>(v);
  v = v + dpp<DPP_XOR3>(v);
  v = v + dpp<DPP_XOR7>(v);
  if constexpr (LANES > 8) v = v + dpp<DPP_XOR15>(v);
  if constexpr (LANES > 16) v = v + swz_xor16(v);
  return v;
}

typedef int int2_t __attribute__((ext_vector_type(2)));

template <int CTRL>
__device__ __forceinline__ int dpp_i32(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, false);
}

template <typename T, int LANES, bool PAIRS, int NORM>
__global__ __launch_bounds__(256) void qk_norm_kernel(const QkArgs a) {
  constexpr int GROUPS = 256 / LANES;
  const int c = threadIdx.x % LANES, half = a.R >> 1;
  const int chunks = a.heads[0] + a.heads[1];
  const int id = static_cast<int>(blockIdx.x) * GROUPS + threadIdx.x / LANES;
  const int stride = static_cast<int>(gridDim.x) * GROUPS / chunks;  // groups that share a head
  int t = id / chunks;
  const int head = id - t * chunks, which = head >= a.heads[0], h = which ? head - a.heads[0] : head;
  if (t >= stride || t >= a.tokens) return;  // the groups left over
  // The lane's pieces: turned ones below R, plain ones from there on; lanes past the head load its first columns as zeros.
  // Both in one aligned 16-byte access where that is allowed (a.wide): halves are then loaded as pieces of two lanes, columns
  // 4 c .. 4 c + 7 by the even one, R / 2 + 4 c .. by the odd one (plain columns 8 c .. by each), and one piece of each is swapped.
  const bool in = 8 * c < a.D, turned = 8 * c < a.R, whole = a.wide, odd = c & 1, cross = !PAIRS && whole;
  int at = 8 * c, pa = 8 * c, pb = 8 * c + 4;  // column of the access, of either piece
  if (!in) {
    at = 0, pa = 0, pb = 4;
  } else if (!PAIRS && turned) {
    pa = 4 * c, pb = half + 4 * c;
    at = whole && odd ? pb - 4 : pa;
  } else if (cross) {
    pa = odd ? 8 * c - 4 : 8 * c, pb = pa + 8;
  }
  float g[8], b[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int col = e < 4 ? pa + e : pb + e - 4;
    if constexpr (NORM != FF_NORM_NONE) g[e] = a.gamma[which][col];
    if constexpr (NORM == FF_NORM_LAYER) b[e] = a.beta[which][col];
  }
  const float q = a.scale[which], inv_d = 1.f / static_cast<float>(a.D);
  const T* x = static_cast<const T*>(a.x[which]) + h * a.xh[which] + t * a.xt[which] + at;
  T* out = static_cast<T*>(a.out[which]) + h * a.oh[which] + t * a.ot[which] + at;
  const int64_t xstep = stride * a.xt[which], ostep = stride * a.ot[which];
  const int apart = pb - pa;
  const float* cos = a.cos + (turned ? 4 * c : 0);
  const float* sin = a.sin + (turned ? 4 * c : 0);

  // The table row of a token, -1 if there is none.
  auto position = [&](int at) __attribute__((always_inline)) {
    if (!a.pos64) {
      const int p = static_cast<const int32_t*>(a.pos)[at];
      return p < a.L ? p : -1;
    }
    const int64_t p = static_cast<const int64_t*>(a.pos)[at];
    return p >= 0 && p < a.L ? static_cast<int>(p) : -1;
  };
  const int wrap = stride % a.L;  // the step of t mod L
  const int last = a.tokens - 1;
  int row = a.pos ? position(t) : t % a.L, after = a.pos ? position(min(t + stride, last)) : 0;
  int4_t nx;
  float4_t nc, ns;
  auto load = [&]() __attribute__((always_inline)) {
    if (whole) {
      nx = *reinterpret_cast<const int4_t*>(x);
    } else {
      const int2_t lo = *reinterpret_cast<const int2_t*>(x), hi = *reinterpret_cast<const int2_t*>(x + apart);
      nx = int4_t{lo[0], lo[1], hi[0], hi[1]};
    }
    const int64_t entry = static_cast<int64_t>(max(row, 0)) * half;
    nc = *reinterpret_cast<const float4_t*>(cos + entry);
    ns = *reinterpret_cast<const float4_t*>(sin + entry);
  };
  // The even lane's second piece for the odd lane's first; its own inverse.
  auto swap = [&](int4_t w) __attribute__((always_inline)) {
    const int r0 = dpp_i32<DPP_XOR1>(odd ? w[0] : w[2]), r1 = dpp_i32<DPP_XOR1>(odd ? w[1] : w[3]);
    return int4_t{odd ? r0 : w[0], odd ? r1 : w[1], odd ? w[2] : r0, odd ? w[3] : r1};
  };
  load();
  for (;;) {
    const vec8_t<T> xs = __builtin_bit_cast(vec8_t<T>, cross ? swap(nx) : nx);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = in ? static_cast<float>(xs[e]) : 0.f;
    const float4_t co = nc, si = ns;
    const float f = row >= 0 ? q : __builtin_nanf("");  // no such row in the table
    const bool more = t < a.tokens - stride;
    if (more) {  // the next token's columns and entries, and the position of the one after it
      t += stride;
      x += xstep;
      if (a.pos) {
        row = after;
        after = position(t < a.tokens - stride ? t + stride : last);
      } else {
        row += wrap;
        row = row >= a.L ? row - a.L : row;
      }
      load();
    }
    if constexpr (NORM == FF_NORM_LAYER) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) s = s + v[e];
      const float mean = group_sum<LANES>(s) * inv_d;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = in ? v[e] - mean : 0.f;
    }
    if constexpr (NORM != FF_NORM_NONE) {
      float sq = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) sq = __builtin_fmaf(v[e], v[e], sq);
      // about 1 ulp; v_rsq_f32 takes a subnormal number for zero, and only a subnormal eps leaves one
      const float ms = __builtin_fmaf(group_sum<LANES>(sq), inv_d, a.eps);
      float r = __builtin_amdgcn_rsqf(ms);
      if (a.eps < 0x1p-126f) r = ms < 0x1p-126f ? __builtin_amdgcn_rsqf(ms * 0x1p24f) * 0x1p12f : r;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        v[e] = NORM == FF_NORM_LAYER ? __builtin_fmaf(v[e] * r, g[e], b[e]) : v[e] * r * g[e];
    }
    if (turned) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float &x0 = v[PAIRS ? 2 * i : i], &x1 = v[PAIRS ? 2 * i + 1 : i + 4];
        const float y0 = __builtin_fmaf(x0, co[i], -(x1 * si[i])), y1 = __builtin_fmaf(x0, si[i], x1 * co[i]);
        x0 = y0;
        x1 = y1;
      }
    }
    vec8_t<T> y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = static_cast<T>(v[e] * f);
    int4_t w = __builtin_bit_cast(int4_t, y);
    if (cross) w = swap(w);
    if (in) {
      if (whole) {
        __builtin_nontemporal_store(w, reinterpret_cast<int4_t*>(out));
      } else {
        __builtin_nontemporal_store(int2_t{w[0], w[1]}, reinterpret_cast<int2_t*>(out));
        __builtin_nontemporal_store(int2_t{w[2], w[3]}, reinterpret_cast<int2_t*>(out + apart));
      }
    }
    if (!more) break;
    out += ostep;
  }
}

template <typename T, int LANES, bool PAIRS, int NORM>
static void launch_qk(const QkArgs& a, hipStream_t st) {
  constexpr int GROUPS = 256 / LANES;
  const int64_t chunks = a.heads[0] + a.heads[1];
  int64_t cap = resident_blocks(reinterpret_cast<const void*>(&qk_norm_kernel<T, LANES, PAIRS, NORM>), 256, 0);
  if (cap <= 0) cap = 1024;
  const int64_t need = (a.tokens * chunks + GROUPS - 1) / GROUPS;
  const int64_t grid = std::max(std::min(need, cap), (chunks + GROUPS - 1) / GROUPS);  // at least a group a head
  qk_norm_kernel<T, LANES, PAIRS, NORM><<<dim3(static_cast<unsigned>(grid)), 256, 0, st>>>(a);
}

template <typename T, int LANES, bool PAIRS>
static void launch_qk_norm(const QkArgs& a, hipStream_t st) {
  switch (a.norm) {
    case FF_NORM_RMS: return launch_qk<T, LANES, PAIRS, FF_NORM_RMS>(a, st);
    case FF_NORM_LAYER: return launch_qk<T, LANES, PAIRS, FF_NORM_LAYER>(a, st);
    default: return launch_qk<T, LANES, PAIRS, FF_NORM_NONE>(a, st);
  }
}

template <typename T>
static void launch_qk_shape(const QkArgs& a, bool pairs, hipStream_t st) {
  if (a.D <= 64)
    pairs ? launch_qk_norm<T, 8, true>(a, st) : launch_qk_norm<T, 8, false>(a, st);
  else if (a.D <= 128)
    pairs ? launch_qk_norm<T, 16, true>(a, st) : launch_qk_norm<T, 16, false>(a, st);
  else
    pairs ? launch_qk_norm<T, 32, true>(a, st) : launch_qk_norm<T, 32, false>(a, st);
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
  if (rope_len <= 0 || rope_len >= (1 << 30)) return fail(FF_EINVAL, "qk_norm_rope: need 0 < rope_len < 2^30");
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
  if (q_out == k_out || q_out == k || k_out == q)
    return fail(FF_EINVAL, "qk_norm_rope: q_out and k_out must be two, each apart from the other's input");
  // Rows are read and written by different workgroups, in no order: an output is its input itself or shares no byte with what
  // is read or with the other output.
  auto rows = [&](const void* p, int64_t token, int64_t head, int64_t n) {
    return Extent{reinterpret_cast<uintptr_t>(p), {T, n}, {2 * token, 2 * head}, 2 * D};
  };
  const Extent in[2] = {rows(q, q_token, q_head, heads), rows(k, k_token, k_head, kv_heads)};
  const Extent to[2] = {rows(q_out, qo_token, qo_head, heads), rows(k_out, ko_token, ko_head, kv_heads)};
  auto in_place = [](const Extent& a, const Extent& b) {
    return a.at == b.at && (a.n[0] <= 1 || a.pitch[0] == b.pitch[0]) && (a.n[1] <= 1 || a.pitch[1] == b.pitch[1]);
  };
  const Extent read[7] = {range(rope_cos, rope_len * R * 2), range(rope_sin, rope_len * R * 2), range(q_gamma, 4 * D),
                          range(k_gamma, 4 * D), range(q_beta, 4 * D), range(k_beta, 4 * D),
                          range(positions, T * (pos64 ? 8 : 4))};
  bool clear = clear_of(to[0], to[1]);
  for (int i = 0; i < 2; ++i) {
    clear = clear && (in_place(to[i], in[i]) || clear_of(to[i], in[i])) && clear_of(to[i], in[1 - i]);
    for (const Extent& e : read) clear = clear && (e.at == 0 || clear_of(to[i], e));
  }
  if (!clear)
    return fail(FF_EINVAL, "qk_norm_rope: an output overlaps the other one or what is read (its own input, with its strides, "
                           "may be in its place)");
  // 16-byte accesses: halves need pairs of lanes that swap pieces, which pays where columns fill three quarters of a head's
  // lanes (32 800 tokens x 32 heads of 48 47.4 us, 55.3 without; 16 400 x 24 of 96 37.0 and 42.4, of 80 29.0 and 28.2)
  const int64_t lanes = D <= 64 ? 8 : D <= 128 ? 16 : 32;
  const bool wide = (low & 15) == 0 && (pairs || (D % 16 == 0 && R % 16 == 0 && D >= 6 * lanes));
  const QkArgs a{{q, k}, {q_out, k_out}, {q_token, k_token}, {q_head, k_head}, {qo_token, ko_token}, {qo_head, ko_head},
                 {q_gamma, k_gamma}, {q_beta, k_beta}, rope_cos, rope_sin, positions, pos64, static_cast<int>(T),
                 {static_cast<int>(heads), static_cast<int>(kv_heads)}, static_cast<int>(D), static_cast<int>(R),
                 static_cast<int>(rope_len), norm, wide, eps, {q_scale, 1.f}};
  if (dtype == FF_F16)
    launch_qk_shape<half_t>(a, pairs != 0, as_stream(stream));
  else
    launch_qk_shape<bf16_t>(a, pairs != 0, as_stream(stream));
  return check_launch("qk_norm_rope");
}
