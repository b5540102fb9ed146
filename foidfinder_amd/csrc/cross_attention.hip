// Attention of queries to keys and values of another length (cross_attention), and of a batch whose sequences share a prefix
// (prefix_attention), on the fp16 and bf16 matrix cores of gfx950.
//
// o = sum_j p_j v_j / sum_j p_j with p_j = 2^(c q.k_j - m), c = scale log2(e), over the keys that a query sees; m is a reference
// near the largest c q.k_j, raised as larger ones come, and drops out of the quotient. q is used as given: c multiplies the
// products in fp32 (folded into q it would round q once more). Sums, p's sum, m and O are fp32; p is rounded to the values' type
// for the second product, half a step each, which is what the matrix cores take. fp16 has 2^-14 as its least normal number, so its p
// reach 2^LIFT where m is set, and those below 2^-22 of the largest are rounded to steps of 2^-32 of it: n keys lose n 2^-33 of
// the weight at most.
//
// Rows: the G = heads / kv_heads query heads of a key head read the same keys, so a key head's rows are (sequence, token, head
// of the group), 32 of them a unit.
// Tiles (cross_kernel): four waves and up to 128 rows, K and V in tiles of 64 keys through two LDS slots that all waves read. Four
// units: a wave each. Two: two waves a unit, each over one half of every tile. One is streamed.
// Streams (stream_kernel; up to 32 rows a sequence and key head): four or eight waves share a unit, each with keys of its own, 32
// at a time through LDS of its own, without a barrier until the waves' O, m and l are joined.
// Keys: a workgroup runs over all keys of its rows, or over one of several runs of them where there are few rows, or where a last
// round of workgroups would leave much of the chip idle (Plan). The runs' O, m and l go to the workspace in fp32 and join_kernel
// joins them in a fixed order.
// Shared prefix: its keys have no sequence, so the rows of all sequences together read it; the same launch's other workgroups
// take each sequence's own keys, and join_kernel joins the parts. Streams of one sequence, or behind a short prefix, read both.
// Masks: a workgroup lists the keys that the mask leaves in LDS, a chunk of the mask at a time, and its tiles hold only those;
// streams leave out masked keys' loads.
//
// Causal: a key that only later tokens see is in the tile all the same, with p = 0 for the earlier ones. Where its value is not
// finite that product would not be 0: such values are found, added to the rows that see them (add_unbounded), and cleared in LDS.
//
// Loads go straight into LDS. Rows that no query of the workgroup may see (past the length, or masked) and columns past D are
// out of the descriptor's range: they read as zeros and cost no traffic, and what the memory there holds never reaches a product.
// Per wave, S^T = K Q^T by 32x32x16 products leaves a lane with one query and 16 of 32 keys; P^T then is the column operand of
// O^T = V^T P^T, V read with the transposing ds_read_b64_tr_b16. Both tiles are row-major, their 16-byte chunks XOR-swizzled
// against bank conflicts (counted: none).
//
// What bounds it, measured: with long keys the softmax between the products (8 x 1025 queries, 5184 keys, 16 heads x 64, fp16, in
// 220 us or 790 TF/s: matrix cores busy 41 % of the cycles, vector units 63 %, both at once 22 %, at 1.8 GHz) and the card's power
// (random values take a fifth more time than zeros); at 96 columns 830, at 128 860 to 920 TF/s. With few rows memory: 64 single tokens
// against up to 1025 keys of 8 heads x 128 in 45 us, 4.5 TB/s of the keys read.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attention_common.h"
#include "gemm_common.h"

namespace ff {

constexpr int QW = 32;     // rows of a unit
constexpr int WAVES = 4;   // waves a workgroup
constexpr int BKV = 64;    // keys a tile
constexpr float SUM_LIMIT = 32768.f;  // a lane's sum of 16 p above which m is raised (fp16 holds p up to it)
constexpr float CAP = 12.f;          // exponent of the largest p after m was raised
// m below the largest c S, where it is set. SUM_LIMIT is passed by a p of 2^11 at least, so that a raise moves m. Less room above
// means more raises: us for 0, 6, 8, 10 of it 220, 222, 222, 226 (8 x 1025 queries, 5184 keys, 16 heads x 64), 12.8, 12.8, 13.2, 14.9
// (2 x 256, 512, 8 x 64). bf16 has the exponents of fp32.
template <typename T>
constexpr float LIFT = std::is_same_v<T, half_t> ? 8.f : 0.f;
constexpr float LOWEST = -3.402823466e38f;
// m of a row, or of a part of it, that saw no key. One that saw keys of -inf alone keeps LOWEST: its sum is 0 too, and its softmax
// not a number.
constexpr float NONE = -__builtin_inff();
// 1 / l, 0 without keys.
__device__ __forceinline__ float inverse(float m, float l) {
  return l != 0.f ? 1.f / l : m == NONE ? 0.f : __builtin_nanf("");
}

struct KeySource {
  const void *k, *v;
  int64_t kb, kt, kh, vb, vt, vh;  // strides in elements: sequence, token, head
  int keys;                        // tokens of a sequence
};

struct CrossArgs {
  const void* q;
  void* out;
  int64_t qb, qt, qh, ob, ot, oh;
  KeySource own, prefix;
  const int32_t* lens;
  const uint8_t* mask;
  int64_t mask_b;
  float* work;    // parts' O [slots, D], then their (m, l) [slots, 2]; a slot for each part and row; null: one part a row
  int64_t slots;
  int batch, tokens, kv, group, dim, causal;
  int rows;  // batch * tokens * group: of a key head
  int block_rows, own_tiles, own_splits, prefix_tiles, prefix_splits;
  int tail, tail_splits;  // the last row tiles of the grid, whose keys are cut (no prefix, own_splits 1)
  float c;
};

// Physical 16-byte chunk of chunk c in row r of a tile (its own inverse). K is read 16 rows of a chunk at a time, V 4 rows of
// 64 bytes: both spread over the 64 banks whatever the row's length.
template <int DP>
__device__ __forceinline__ int k_slot(int r, int c) {
  return DP == 64 ? c ^ ((r >> 1) & 7) : DP == 96 ? c ^ ((r >> 2) & 3) : c ^ (r & 15);
}
template <int DP>
__device__ __forceinline__ int v_slot(int r, int c) {
  return DP == 64 ? c ^ ((r & 2) << 1) : DP == 96 ? c : c ^ ((r & 3) << 2);
}

__device__ __forceinline__ float16_t mfma(vec8_t<half_t> a, vec8_t<half_t> b, float16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float16_t mfma(vec8_t<bf16_t> a, vec8_t<bf16_t> b, float16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

typedef bf16_t bf16x2_t __attribute__((ext_vector_type(2)));
// a + b + c in fp32, subnormal a and b included.
__device__ __forceinline__ float add_pair(half_t a, half_t b, float c) {
  return __builtin_amdgcn_fdot2(half2_t{a, b}, half2_t{half_t(1.f), half_t(1.f)}, c, false);
}
__device__ __forceinline__ float add_pair(bf16_t a, bf16_t b, float c) {
  return __builtin_amdgcn_fdot2_f32_bf16(bf16x2_t{a, b}, bf16x2_t{bf16_t(1.f), bf16_t(1.f)}, c, false);
}

// Keys that rows see: all up to a length; those of them that a mask leaves; fewer for earlier tokens.
enum class Keys { ALL, LISTED, CAUSAL };

typedef unsigned short ushort8_t __attribute__((ext_vector_type(8)));
// Magnitude of an infinity as bits; those above are not numbers.
template <typename T>
constexpr unsigned short INFINITE = std::is_same_v<T, half_t> ? 0x7c00 : 0x7f80;
template <typename T>
__device__ __forceinline__ bool finite(T v) {
  return (__builtin_bit_cast(unsigned short, v) & 0x7fff) < INFINITE<T>;
}
// Whether N KB of LDS hold finite values alone.
template <int N, typename T>
__device__ __forceinline__ bool all_finite(const T* p, int lane) {
  ushort8_t top = {};
#pragma unroll
  for (int i = 0; i < N; ++i)
    top = __builtin_elementwise_max(top, *reinterpret_cast<const ushort8_t*>(p + i * 512 + lane * 8) & ushort8_t(0x7fff));
  int most = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) most = max(most, static_cast<int>(top[e]));
  return !__any(most >= INFINITE<T>);
}

// Clears the others, N times 16 bytes of each of `threads` threads.
template <int N, typename T>
__device__ __forceinline__ void keep_finite(T* p, int thread, int threads) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    vec8_t<T>& x = *reinterpret_cast<vec8_t<T>*>(p + (i * threads + thread) * 8);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = finite(x[e]) ? x[e] : static_cast<T>(0.f);
  }
}

// What a workgroup works on; the same in all its lanes.
struct Piece {
  int seq;           // -1: the shared prefix, rows of all sequences
  int head;          // key head
  int row0, row_end;
  int keys, len;     // keys that some row sees; the sequence's length
  int front;         // slices of 32 prefix keys before the sequence's own (streams only)
  int t0, t1;        // tiles, or slices of 32 keys
  int64_t slot;      // of row0 in the workspace; -1: rows go to out
};

// Where a lane's row lies, and how many of the sequence's own keys it sees.
struct Place {
  int seq, token, head, limit;
};
__device__ __forceinline__ Place place_of(const CrossArgs& a, const Piece& w, int row) {
  const int real = min(row, w.row_end - 1), per = a.tokens * a.group;
  Place p;
  p.seq = w.seq < 0 ? real / per : w.seq;
  const int rest = real - p.seq * per;
  p.token = rest / a.group;
  p.head = w.head * a.group + rest - p.token * a.group;
  p.limit = a.causal && w.seq >= 0 ? min(max(w.len - a.tokens + 1 + p.token, 0), w.keys) : w.keys;
  return p;
}

// 32 rows in a wave: q, O, m and the lane's part of l. Lane: row fr = lane % 32, half fh = lane / 32.
template <typename T, int DP>
struct Unit {
  static constexpr int KS = DP / 16, DT = DP / 32, VSTEP = DT == 4 ? 2 : 1;
  typedef vec8_t<T> T8;
  typedef vec4_t<T> T4;
  T8 qf[KS];       // column operand of S^T: the row's columns 16 s + 8 fh + 0..7
  float16_t o[DT]; // O^T: columns 32 dt + 8 (r / 4) + 4 fh + r % 4
  float m = LOWEST, l = 0.f, c;
  // LDS offsets (elements) of the first fragments within 32 keys. The others' follow from the swizzle: an exclusive or with the
  // fragment's place in the row, or for rows of 96 columns a step, from the second one where the fragment is odd.
  int koff, koff_odd, voff;
  static __device__ __forceinline__ int kfrag(int ka, int ka_odd, int s) {
    return DP == 96 ? (s & 1 ? ka_odd : ka) + (s >> 1) * 32 : ka ^ (16 * s);
  }
  static __device__ __forceinline__ int vfrag(int va, int dt) { return DP == 96 ? va + 32 * dt : va ^ (32 * dt); }

  __device__ __forceinline__ void start(const CrossArgs& a, const Place& p, int lane) {
    const int fr = lane & 31, fh = lane >> 5;
    const T* q = static_cast<const T*>(a.q) + p.seq * a.qb + p.token * a.qt + p.head * a.qh;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      qf[s] = T8{};
      if (16 * s + 8 * fh < a.dim) qf[s] = *reinterpret_cast<const T8*>(q + 16 * s + 8 * fh);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
    c = a.c;
    // K fragment s: row fr, chunk 2 s + fh. V^T fragment (dt, tt), part j: lane l of 16 addresses row 16 tt + 8 j + 4 fh + l / 4,
    // columns 32 dt + 16 (group) + 4 (l % 4), and receives four keys in a row of column 32 dt + fr: the keys of P^T's slots.
    koff = fr * DP + k_slot<DP>(fr, fh) * 8;
    if constexpr (DP == 96) koff_odd = fr * DP + k_slot<DP>(fr, 2 + fh) * 8;
    const int r = 4 * fh + ((lane & 15) >> 2), col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    voff = r * DP + v_slot<DP>(r, col >> 3) * 8 + (col & 7);
  }
  // q consumed, so that the compiler's wait for its loads stands here, before the loop and after the first keys' loads, not in it.
  __device__ __forceinline__ void settle() {
#pragma unroll
    for (int s = 0; s < KS; ++s) asm volatile("" ::"v"(qf[s]));
  }
  // x = S^T of the 32 keys at k (+ ka): keys 8 (r / 4) + 4 fh + r % 4.
  __device__ __forceinline__ void score(float16_t& x, const T* k, int ka, int ka_odd) {
    T8 kf[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) kf[s] = *reinterpret_cast<const T8*>(k + kfrag(ka, ka_odd, s));
    const float16_t zero = {};
#pragma unroll
    for (int s = 0; s < KS; ++s) x = mfma(kf[s], qf[s], s == 0 ? zero : x);
  }
  // p of the scores, at most 2^cap each, and the lane's sum of it: of the rounded p, which the second product takes, so that a key
  // with most of the weight is divided by itself.
  __device__ __forceinline__ float weights(const float16_t& xs, T8 (&pf)[2], float cap) {
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float x = __builtin_fmaf(xs[r], c, -m);
      if (!__builtin_isinf(cap)) x = x > cap ? cap : x;  // not a number stays so
      pf[r >> 3][r & 7] = static_cast<T>(__builtin_amdgcn_exp2f(x));
    }
#pragma unroll
    for (int r = 0; r < 16; r += 2) sum[(r >> 1) & 1] = add_pair(pf[r >> 3][r & 7], pf[r >> 3][(r & 7) + 1], sum[(r >> 1) & 1]);
    return sum[0] + sum[1];
  }
  // Scores of keys that the lane's row does not see (bits: those that it sees).
  __device__ __forceinline__ void hide(float16_t& xs, uint32_t bits, int fh) {
    if (__any(bits != ~0u)) {
      bits >>= 4 * fh;
#pragma unroll
      for (int r = 0; r < 16; ++r) xs[r] = (bits >> (8 * (r >> 2) + (r & 3))) & 1 ? xs[r] : -__builtin_inff();
    }
  }
  // p of the scores; bits: the keys that the lane's row sees; first: m is not set yet, which the first pass would only find out.
  __device__ __forceinline__ void weigh(float16_t& xs, T8 (&pf)[2], uint32_t bits, int fh, bool first) {
    hide(xs, bits, fh);
    float sum = 0.f;
    if (!first) sum = weights(xs, pf, __builtin_inff());
    if (first || __any(sum > SUM_LIMIT))
      raise(xs, pf);
    else
      l += sum;
  }
  // The keys' p passed the limit, or m is not set: m becomes LIFT less than the largest c S, or just below, and O and l follow. Scores
  // from 2^30 up are too coarse for the multiply-add: what it leaves of the largest can be of any size then, and is capped.
  // An infinite c S makes m infinite, and l not a number from then on (m - m): inf - inf, as the row's softmax has it. The joints
  // of m and l keep it so.
  __device__ __forceinline__ void raise(const float16_t& xs, T8 (&pf)[2]) {
    float top = xs[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, xs[r]);
    top = fmaxf(top, xor_shuffle(top, 32)) * c;
    const float m_old = m;
    m = fmaxf(m, top * (top > 0.f ? 1.f - 0x1p-23f : 1.f + 0x1p-23f) - LIFT<T>);
    const float corr = m_old == LOWEST ? 1.f : __builtin_amdgcn_exp2f(m_old - m);  // O held nothing, or infinities to be kept
    l = __builtin_fmaf(l, corr, m - m);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[dt][r] *= corr;
    l += weights(xs, pf, CAP);
  }
  // O^T += V^T P^T, the 32 values at LDS byte v + OFF (+ va).
  template <int OFF>
  __device__ __forceinline__ void mix(uint32_t v, int va, const T8 (&pf)[2]) {
#pragma unroll
    for (int dt = 0; dt < DT; dt += VSTEP) {
      T4 x[VSTEP][4];  // [][2 tt + j]
      const uint32_t at = v + 2u * static_cast<uint32_t>(vfrag(va, dt));
      if constexpr (VSTEP == 2)
        tr_read4<OFF, 8 * DP * 2>(x[0], at, x[1], v + 2u * static_cast<uint32_t>(vfrag(va, dt + 1)));
      else
        tr_read4<OFF, 8 * DP * 2>(x[0], at);
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int i = 0; i < VSTEP; ++i)
          o[dt + i] = mfma(__builtin_shufflevector(x[i][2 * tt], x[i][2 * tt + 1], 0, 1, 2, 3, 4, 5, 6, 7), pf[tt], o[dt + i]);
    }
  }
  // Adds the values that are not finite among those of N keys at `rows` to the rows that see them: the first `left` keys.
  template <int N>
  __device__ __forceinline__ void add_unbounded(const T* rows, int left, int fh) {
#pragma unroll 1
    for (int j = 0; j < N; ++j) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const T4 x = *reinterpret_cast<const T4*>(rows + j * DP + v_slot<DP>(j, 4 * dt + g) * 8 + 4 * fh);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[dt][4 * g + e] += j < left && !finite(x[e]) ? static_cast<float>(x[e]) : 0.f;
        }
    }
  }
};

// Four columns of a row's O to the workspace, or its quotient to out; (m, l) with the first.
template <typename T>
__device__ __forceinline__ void store4(const CrossArgs& a, const Piece& w, const Place& p, int row, int col, float4_t o, float m,
                                       float l) {
  if (col >= a.dim) return;
  if (w.slot >= 0) {
    const int64_t n = w.slot + row - w.row0;
    *reinterpret_cast<float4_t*>(a.work + n * a.dim + col) = o;
    if (col == 0) *reinterpret_cast<float2*>(a.work + a.slots * a.dim + 2 * n) = float2{m, l};
    return;
  }
  const float inv = inverse(m, l);
  vec4_t<T> v;
#pragma unroll
  for (int u = 0; u < 4; ++u) v[u] = static_cast<T>(o[u] * inv);
  *reinterpret_cast<vec4_t<T>*>(static_cast<T*>(a.out) + p.seq * a.ob + p.token * a.ot + p.head * a.oh + col) = v;
}

// LDS of streams and of tiles, and of the joints that follow in the same place.
constexpr int stream_bytes(int dp, int waves) {
  const int slices = waves * 2 * 32 * dp * 2, joint = waves * (dp / 2 + 2) * 256;
  return slices > joint ? slices : joint;
}
constexpr int tile_bytes(int dp) { return 4 * BKV * dp * 2 > stream_bytes(dp, WAVES) ? 4 * BKV * dp * 2 : stream_bytes(dp, WAVES); }
// Keys of a mask that are listed at a time: what the LDS leaves room for beside a CU's workgroups.
constexpr int list_chunk(int dp) { return dp == 64 ? 1024 : dp == 96 ? 512 : 2048; }

// Tiles of 64 keys for four waves: a wave a unit (SHARE 1), or two (SHARE 2), each with one half of every tile. LISTED: tiles hold
// keys that the mask leaves, and no others. Us for half the keys masked at random, a third at the end, none, where a tile's mask
// word left out loads and empty tiles, and by list: 15.1 -> 16.1, 14.7 -> 16.1, 14.6 -> 15.7 (2 x 256 queries, 512 keys, 8 heads x
// 64); 26.8 -> 18.4, 20.5 -> 20.4, 24.3 -> 25.8 (4 x 512, 1024, 16 x 64); 62 -> 36, 46 -> 44, 56 -> 58 (2 x 512, 2048, 32 / 8 x
// 128); 330 -> 172, 226 -> 217, 289 -> 291 (4 x 1024, 4096, 32 / 8 x 128). A list in memory, by a kernel of its own: 182, 228, 300.
template <typename T, int DP, int SHARE, Keys KEYS>
__device__ __forceinline__ void tile_block(const CrossArgs& a, const Piece& w, T* smem) {
  typedef vec8_t<T> T8;
  constexpr bool LIST = KEYS == Keys::LISTED, CAUSAL = KEYS == Keys::CAUSAL;
  constexpr int CH = DP / 8, TILE = BKV * DP, LPW = CH / 4, KS = DP / 16, DT = DP / 32;
  const uint32_t smem_lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void*)smem));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int fr = lane & 31, fh = lane >> 5, unit = wave / SHARE, half_sel = SHARE == 2 ? wave & 1 : 0;
  const bool active = w.row0 + unit * QW < w.row_end;  // other waves only load
  int row = w.row0 + unit * QW + fr, limit;
  const int lowest = CAUSAL ? place_of(a, w, w.row0).limit : 0;  // of the workgroup's first row
  Unit<T, DP> u;
  {
    const Place p = place_of(a, w, row);
    u.start(a, p, lane);
    limit = p.limit;
  }

  const KeySource& src = w.seq < 0 ? a.prefix : a.own;
  const int64_t at = max(w.seq, 0);
  const T* kbase = static_cast<const T*>(src.k) + at * src.kb + w.head * src.kh;
  const T* vbase = static_cast<const T*>(src.v) + at * src.vb + w.head * src.vh;
  const bool guard = src.kt < a.dim || src.vt < a.dim;  // rows left out that the descriptor's range does not leave out

  // Tile loads: wave w fills the 1 KB blocks LPW w .. of either tile, lane l the chunk l of a block; it fetches what the swizzle
  // puts there.
  uint32_t voff_k[LPW], voff_v[LPW];
#pragma unroll
  for (int i = 0; i < LPW; ++i) {
    const int n = (LPW * wave + i) * 64 + lane, r = n / CH, slot = n % CH;
    const int ck = k_slot<DP>(r, slot), cv = v_slot<DP>(r, slot);
    const int kr = LIST ? 0 : r * static_cast<int>(src.kt), vr = LIST ? 0 : r * static_cast<int>(src.vt);
    voff_k[i] = 8 * ck < a.dim ? static_cast<uint32_t>((kr + ck * 8) * 2) : OOB_OFFSET;
    voff_v[i] = 8 * cv < a.dim ? static_cast<uint32_t>((vr + cv * 8) * 2) : OOB_OFFSET;
  }
  // The list: keys that the mask leaves, in order; [pos, have) have not been loaded yet.
  constexpr int CHUNK = list_chunk(DP), EACH = CHUNK / (64 * WAVES);
  int32_t *list = reinterpret_cast<int32_t*>(smem + tile_bytes(DP) / 2), *counts = list + CHUNK + BKV;
  const uint8_t* bytes = LIST ? a.mask + at * a.mask_b : nullptr;
  const int end = LIST ? min(w.t1 * BKV, w.keys) : 0;
  int pos = 0, have = 0, raw = w.t0 * BKV;
  // Moves them to the front and lists the next chunks' keys behind them until there are a tile's, or all.
  auto refill = [&]() __attribute__((always_inline)) {
    const int tid = threadIdx.x, left = have - pos, carried = tid < left ? list[pos + tid] : 0;
    __syncthreads();
    if (tid < left) list[tid] = carried;
    pos = 0, have = left;
    while (have < BKV && raw < end) {
      uint32_t bits = 0;
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int n = EACH * tid + e;
        const uint8_t byte = bytes[raw + min(n, end - raw - 1)];
        bits |= byte != 0 && n < end - raw ? 1u << e : 0u;
      }
      const int mine = __popc(bits);
      int before = mine;  // in the wave, this thread's with them
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int other = __shfl_up(before, d, 64);
        before += lane >= d ? other : 0;
      }
      if (lane == 63) counts[wave] = before;
      __syncthreads();
      int to = have + before - mine, all = 0;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) {
        const int n = counts[i];
        to += i < wave ? n : 0;
        all += n;
      }
#pragma unroll
      for (int e = 0; e < EACH; ++e)
        if (bits >> e & 1) list[to++] = raw + EACH * tid + e;
      __syncthreads();
      have += __builtin_amdgcn_readfirstlane(all);
      raw = end - raw > CHUNK ? raw + CHUNK : end;
    }
  };
  auto issue = [&](int tile, uint64_t word) __attribute__((always_inline)) {
    const int st = (tile - w.t0) & 1, rows = min(BKV, w.keys - tile * BKV);
    const int64_t first = static_cast<int64_t>(tile) * BKV;
    const int nk = ((rows - 1) * static_cast<int>(src.kt) + a.dim) * 2, nv = ((rows - 1) * static_cast<int>(src.vt) + a.dim) * 2;
    const T *k = kbase + first * src.kt, *v = vbase + first * src.vt;
#pragma unroll
    for (int i = 0; i < LPW; ++i) {
      const bool in = !guard || ((word >> (((LPW * wave + i) * 64 + lane) / CH)) & 1);
      buffer_to_lds(k, nk, reinterpret_cast<uint8_t*>(smem + st * TILE + (LPW * wave + i) * 512), in ? voff_k[i] : OOB_OFFSET);
      buffer_to_lds(v, nv, reinterpret_cast<uint8_t*>(smem + (2 + st) * TILE + (LPW * wave + i) * 512),
                    in ? voff_v[i] : OOB_OFFSET);
    }
  };
  // The keys of a tile that may be seen, as bits.
  auto valid = [&](int n) __attribute__((always_inline)) { return n >= 64 ? ~uint64_t(0) : (uint64_t(1) << n) - 1; };
  auto bits_of = [&](int tile, uint64_t word, int half) __attribute__((always_inline)) {
    if constexpr (LIST) return static_cast<uint32_t>(word >> (32 * half));
    const int left = limit - (tile * BKV + 32 * half);
    return static_cast<uint32_t>(word >> (32 * half)) & (left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1);
  };
  auto half_tile = [&](int tile, uint64_t word, int half, int ka, int ka_odd, int va) __attribute__((always_inline)) {
    float16_t x;
    vec8_t<T> pf[2];
    u.score(x, smem, ka, ka_odd);
    u.weigh(x, pf, bits_of(tile, word, half), fh, tile == w.t0 && half == 0);
    u.template mix<0>(smem_lds, va, pf);
  };
  // Both halves of a tile: either product of one runs under the softmax of the other. Returns the half from which on it is not
  // done, because p passed the limit (2: it is done): half_tile does these, and raises m.
  auto whole_tile = [&](int tile, uint64_t word, int ka, int ka_odd, int va) __attribute__((always_inline)) {
    vec8_t<T> pf[2][2];
    float16_t x[2];
    u.score(x[0], smem, ka, ka_odd);
    u.hide(x[0], bits_of(tile, word, 0), fh);
    u.score(x[1], smem + 32 * DP, ka, ka_odd);
    float sum = u.weights(x[0], pf[0], __builtin_inff());
    if (__any(sum > SUM_LIMIT)) return 0;
    u.l += sum;
    u.hide(x[1], bits_of(tile, word, 1), fh);
    u.template mix<0>(smem_lds, va, pf[0]);
    sum = u.weights(x[1], pf[1], __builtin_inff());
    if (__any(sum > SUM_LIMIT)) return 1;
    u.l += sum;
    u.template mix<32 * DP * 2>(smem_lds, va, pf[1]);
    return 2;
  };

  // The list's rows: those of the keys up to `usable` lie within 2^31 bytes from that of key `base` on.
  const int kt = static_cast<int>(src.kt), vt = static_cast<int>(src.vt), reach = ((1 << 30) - 2 * DP) / max(max(kt, vt), 1);
  int usable = 0, base = 0;
  // Takes the next tile's keys from the list and loads their rows into a slot: how many.
  auto issue_listed = [&](int st) __attribute__((always_inline)) {
    if (usable - pos < BKV) {
      if (have - pos < BKV && raw < end) refill();
      if (have == pos) return 0;
      base = __builtin_amdgcn_readfirstlane(list[pos]), usable = have;
      if (__builtin_amdgcn_readfirstlane(list[have - 1]) - base > reach)
        usable = pos + __popcll(__ballot(lane < have - pos && list[min(pos + lane, have - 1)] - base <= reach));
    }
    const int n = min(BKV, usable - pos), span = min(reach, w.keys - 1 - base);
    const int nk = (span * kt + a.dim) * 2, nv = (span * vt + a.dim) * 2;
    const T *k = kbase + base * src.kt, *v = vbase + base * src.vt;
    int on[LPW];
#pragma unroll
    for (int i = 0; i < LPW; ++i) on[i] = list[pos + min(((LPW * wave + i) * 64 + lane) / CH, n - 1)] - base;
#pragma unroll
    for (int i = 0; i < LPW; ++i) {
      const bool in = ((LPW * wave + i) * 64 + lane) / CH < n;
      const uint32_t ko = voff_k[i] + static_cast<uint32_t>(on[i] * kt) * 2, vo = voff_v[i] + static_cast<uint32_t>(on[i] * vt) * 2;
      buffer_to_lds(k, nk, reinterpret_cast<uint8_t*>(smem + st * TILE + (LPW * wave + i) * 512), in ? ko : OOB_OFFSET);
      buffer_to_lds(v, nv, reinterpret_cast<uint8_t*>(smem + (2 + st) * TILE + (LPW * wave + i) * 512), in ? vo : OOB_OFFSET);
    }
    pos += n;
    return n;
  };

  bool listed = false;  // any key
  if (w.t0 < w.t1) {
    uint64_t word, next = 0;  // of a list, 0 behind the last tile
    if constexpr (LIST) {
      word = valid(issue_listed(0));
      listed = word != 0;
    } else {
      word = valid(w.keys - w.t0 * BKV);
      issue(w.t0, word);
    }
    u.settle();
    for (int tile = w.t0; LIST ? word != 0 : tile < w.t1; ++tile) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();  // no fence: the wait covers this thread's LDS writes
      const int st = (tile - w.t0) & 1;  // the other slot was last read for tile - 1, which every wave has finished
      if constexpr (LIST) {
        next = valid(issue_listed(st ^ 1));
      } else if (tile + 1 < w.t1) {
        next = valid(w.keys - (tile + 1) * BKV);
        issue(tile + 1, next);
      }
      if constexpr (CAUSAL) {
        T* values = smem + (2 + st) * TILE;
        if (min((tile + 1) * BKV, w.keys) > lowest && !all_finite<TILE * 2 / 1024>(values, lane)) {  // the same in all waves
          if (active) u.template add_unbounded<BKV / SHARE>(values + half_sel * 32 * DP, limit - tile * BKV - 32 * half_sel, fh);
          __syncthreads();
          keep_finite<LPW>(values, threadIdx.x, 64 * WAVES);
          __syncthreads();
        }
      }
      if (active) {
        // read bases, opaque to the compiler so that the fragment offsets fold into the reads' immediate offsets
        int ka = st * TILE + half_sel * 32 * DP + u.koff, ka_odd = 0, va = (2 + st) * TILE + half_sel * 32 * DP + u.voff;
        asm volatile("" : "+v"(ka), "+v"(va));
        if constexpr (DP == 96) {
          ka_odd = st * TILE + half_sel * 32 * DP + u.koff_odd;
          asm volatile("" : "+v"(ka_odd));
        }
        if constexpr (SHARE == 2) {
          half_tile(tile, word, half_sel, ka, ka_odd, va);
        } else {
#pragma unroll 1
          for (int half = whole_tile(tile, word, ka, ka_odd, va); half < 2; ++half)
            half_tile(tile, word, half, ka + half * 32 * DP, ka_odd + half * 32 * DP, va + half * 32 * DP);
        }
      }
      word = next;
    }
  }

  // A row that saw keys saw the first of the first tile, or of the list.
  if (!(w.t0 < w.t1 && (LIST ? listed : limit > w.t0 * BKV))) u.m = NONE;
  if constexpr (SHARE == 2) {  // the second wave of a unit leaves O, m and l in LDS; the first joins them
    constexpr int WORDS = 16 * DT + 2;
    static_assert(2 * WORDS * 64 * 4 <= 4 * TILE * 2, "the joint exceeds the ring");
    float* joint = reinterpret_cast<float*>(smem) + unit * WORDS * 64 + lane;
    __syncthreads();
    if (active && half_sel) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) joint[(dt * 16 + r) * 64] = u.o[dt][r];
      joint[(WORDS - 2) * 64] = u.m;
      joint[(WORDS - 1) * 64] = u.l;
    }
    __syncthreads();
    if (!active || half_sel) return;
    const float m1 = joint[(WORDS - 2) * 64], top = fmaxf(fmaxf(u.m, m1), LOWEST);
    const float c0 = __builtin_amdgcn_exp2f(u.m - top), c1 = __builtin_amdgcn_exp2f(m1 - top);
    u.m = fmaxf(u.m, m1);
    u.l = __builtin_fmaf(joint[(WORDS - 1) * 64], c1, u.l * c0);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) u.o[dt][r] = __builtin_fmaf(joint[(dt * 16 + r) * 64], c1, u.o[dt][r] * c0);
  } else {
    if (!active) return;
  }
  const float l = u.l + xor_shuffle(u.l, 32);
  if (row >= w.row_end) return;
  asm volatile("" : "+v"(row));  // its place is found again here: kept through the loop it would hold registers
  const Place p = place_of(a, w, row);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      store4<T>(a, w, p, row, dt * 32 + 8 * g + 4 * fh,
                float4_t{u.o[dt][4 * g], u.o[dt][4 * g + 1], u.o[dt][4 * g + 2], u.o[dt][4 * g + 3]}, u.m, l);
}

// One unit of rows and NW waves, each with slices of 32 keys of its own (slice t0 + wave, + NW, ...) in LDS of its own, so no
// barrier stands between load and use: a wave asks for the next slice's K once it has read this one's, and for its V likewise, so
// that half a slice or more (8 KB at 128 columns) is on its way to each wave at any time. The slices are those of the prefix
// (w.front), then the sequence's own. The waves' O, m and l are joined through LDS, four columns a wave and turn.
template <typename T, int DP, int NW, bool CAUSAL>
__device__ __forceinline__ void stream_block(const CrossArgs& a, const Piece& w, T* smem) {
  typedef vec8_t<T> T8;
  constexpr int CH = DP / 8, SLICE = 32 * DP, LP = CH / 2, DT = DP / 32, WORDS = 16 * DT + 2;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fr = lane & 31, fh = lane >> 5;
  T* kbuf = smem + wave * 2 * SLICE;
  const uint32_t vbuf = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void*)(kbuf + SLICE)));
  const int row = w.row0 + fr;
  const Place p = place_of(a, w, row);
  Unit<T, DP> u;
  u.start(a, p, lane);

  const int64_t seq = max(w.seq, 0);
  const uint8_t* mask = a.mask && w.seq >= 0 ? a.mask + seq * a.mask_b : nullptr;
  // Loads of a slice: 1 KB each, lane l the chunk l.
  int lrow[LP];
  uint32_t coff_k[LP], coff_v[LP];
#pragma unroll
  for (int i = 0; i < LP; ++i) {
    const int n = i * 64 + lane, r = n / CH, slot = n % CH, ck = k_slot<DP>(r, slot), cv = v_slot<DP>(r, slot);
    lrow[i] = r;
    coff_k[i] = 8 * ck < a.dim ? 16 * ck : OOB_OFFSET;
    coff_v[i] = 8 * cv < a.dim ? 16 * cv : OOB_OFFSET;
  }
  // own: of the sequence (the prefix's otherwise)
  struct Slice {
    bool own;
    int first, rows;
    uint32_t word;
  };
  auto mask_byte = [&](int n) __attribute__((always_inline)) {
    const int key = (n - w.front) * 32 + fr;
    return mask && n < w.t1 && key < w.keys ? mask[key] : uint8_t(0);
  };
  auto slice = [&](int n, uint8_t byte) __attribute__((always_inline)) {
    Slice s;
    s.own = w.seq >= 0 && n >= w.front;
    s.first = (s.own ? n - w.front : n) * 32;
    s.rows = min(32, (s.own ? w.keys : a.prefix.keys) - s.first);
    s.word = s.rows >= 32 ? ~0u : (1u << s.rows) - 1;
    if (mask) s.word = static_cast<uint32_t>(__ballot(byte != 0));
    return s;
  };
  auto load = [&](const Slice& s, bool values) __attribute__((always_inline)) {
    const KeySource& src = s.own ? a.own : a.prefix;
    const int64_t step = values ? src.vt : src.kt, at = s.own ? seq : 0;
    const T* base = static_cast<const T*>(values ? src.v : src.k) + at * (values ? src.vb : src.kb) +
                    w.head * (values ? src.vh : src.kh) + s.first * step;
    const int bytes = ((s.rows - 1) * static_cast<int>(step) + a.dim) * 2;
#pragma unroll
    for (int i = 0; i < LP; ++i) {
      const uint32_t chunk = values ? coff_v[i] : coff_k[i];
      const bool in = (s.word >> lrow[i]) & 1;
      buffer_to_lds(base, bytes, reinterpret_cast<uint8_t*>(kbuf + (values ? SLICE : 0) + i * 512),
                    in ? chunk + static_cast<uint32_t>(lrow[i] * static_cast<int>(step)) * 2 : OOB_OFFSET);
    }
  };

  int n = w.t0 + wave;
  uint32_t seen = 0;  // of any slice
  if (n < w.t1) {
    Slice now = slice(n, mask_byte(n));
    uint8_t byte = mask_byte(n + NW);
    load(now, false);
    load(now, true);
    u.settle();
    for (;;) {
      const bool more = n + NW < w.t1;
      Slice next = now;
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LP) : "memory");  // all but V
      float16_t x;
      T8 pf[2];
      u.score(x, kbuf, u.koff, u.koff_odd);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (more) {
        next = slice(n + NW, byte);
        byte = mask_byte(n + 2 * NW);
        load(next, false);
      }
      const int left = now.own ? p.limit - now.first : 32;
      const uint32_t bits = now.word & (left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1);
      seen |= bits;
      u.weigh(x, pf, bits, fh, n == w.t0 + wave);
      if (more)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LP) : "memory");  // all but the next K
      else
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (CAUSAL && __any(bits != now.word) && !all_finite<LP>(kbuf + SLICE, lane)) {
        u.template add_unbounded<32>(kbuf + SLICE, left, fh);
        keep_finite<LP>(kbuf + SLICE, lane, 64);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      u.template mix<0>(vbuf, u.voff, pf);
      if (!more) break;
      load(next, true);
      now = next;
      n += NW;
    }
  }

  __syncthreads();  // the slices' memory becomes the joint's
  float* joint = reinterpret_cast<float*>(smem) + lane;
  const float l_own = u.l + xor_shuffle(u.l, 32);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) joint[(wave * WORDS + dt * 16 + r) * 64] = u.o[dt][r];
  joint[(wave * WORDS + WORDS - 2) * 64] = seen ? u.m : NONE;
  joint[(wave * WORDS + WORDS - 1) * 64] = l_own;
  __syncthreads();
  if (row >= w.row_end) return;
  float m = NONE;
#pragma unroll
  for (int k = 0; k < NW; ++k) m = fmaxf(m, joint[(k * WORDS + WORDS - 2) * 64]);
  const float top = fmaxf(m, LOWEST);
  for (int g = wave; g < 4 * DT; g += NW) {  // words 4 g .. 4 g + 3: columns 32 (g / 4) + 8 (g % 4) + 4 fh + 0..3
    float4_t o = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
#pragma unroll 4
    for (int k = 0; k < NW; ++k) {
      const float* part = joint + k * WORDS * 64;
      const float f = __builtin_amdgcn_exp2f(part[(WORDS - 2) * 64] - top);
      l = __builtin_fmaf(part[(WORDS - 1) * 64], f, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(part[(4 * g + e) * 64], f, o[e]);
    }
    store4<T>(a, w, p, row, (g >> 2) * 32 + (g & 3) * 8 + 4 * fh, o, m, l);
  }
}

// The arguments' cache lines asked for at once, at the start: each costs a trip of its own where it is first used.
__device__ __forceinline__ void touch(const CrossArgs& a) {
  asm volatile("" ::"s"(a.qb), "s"(a.own.k), "s"(a.own.vt), "s"(a.prefix.kt), "s"(a.lens), "s"(a.batch), "s"(a.c));
}

// Waves a SIMD: what the LDS leaves room for (34, 50 and 66 KB a workgroup).
template <typename T, int DP, Keys KEYS>
__global__ __launch_bounds__(64 * WAVES, DP == 64 ? 4 : DP == 96 ? 3 : 2) void cross_kernel(const CrossArgs a) {
  constexpr bool LIST = KEYS == Keys::LISTED;
  // K slots, then V slots; the list and its counts
  __shared__ __attribute__((aligned(1024))) T smem[tile_bytes(DP) / 2 + (LIST ? 2 * (list_chunk(DP) + BKV + WAVES) : 0)];
  touch(a);
  const int per = a.tokens * a.group, prefix_items = a.prefix_splits * a.kv * a.prefix_tiles;
  int item = static_cast<int>(blockIdx.x);
  Piece w;
  int split = 0, splits = 1, tile, x;
  // Row tiles of one run of keys are neighbours, and neighbours share an XCD's L2 (the prefix's pieces by themselves, as they
  // differ from the others in length). Runs are counted by sequences first, so that every XCD has long and short ones: 8 x 1024
  // queries of 16 heads x 64 to 4096 / 8 .. 4096 keys 146 -> 123 us, 4 x 1000 of 32 / 8 x 128 265 -> 192. A run's last tile, where
  // it has fewer rows and takes less time, comes after all whole ones and fills the end of the grid; before it come the tail's
  // pieces.
  auto place = [&](int n, int tiles, int rows, int tail, int tail_splits) __attribute__((always_inline)) {
    const int whole = rows / a.block_rows, runs = n / tiles, all = runs * whole;
    if (item < all - tail) {
      item = xcd_remap(item, all - tail);
    } else if (item < all - tail + tail * tail_splits) {
      const int cut = xcd_remap(item - (all - tail), tail * tail_splits);
      split = cut / tail, splits = tail_splits, item = all - tail + cut - split * tail;
    } else {
      x = xcd_remap(item - (all - tail + tail * tail_splits), runs), tile = whole;
      return;
    }
    x = item / whole, tile = item - x * whole;
  };
  if (item < prefix_items) {
    place(prefix_items, a.prefix_tiles, a.rows, 0, 1);
    split = x % a.prefix_splits, splits = a.prefix_splits;
    w.seq = -1, w.head = x / a.prefix_splits;
    w.row0 = tile * a.block_rows, w.row_end = a.rows;
    w.slot = (static_cast<int64_t>(split) * a.kv + w.head) * a.rows + w.row0;
    w.len = w.keys = a.prefix.keys;
  } else {
    item -= prefix_items;
    place(a.batch * a.kv * a.own_splits * a.own_tiles, a.own_tiles, per, a.tail, a.tail_splits);
    const int y = x / a.own_splits;
    w.head = y / a.batch, w.seq = y - w.head * a.batch;
    w.row0 = w.seq * per + tile * a.block_rows, w.row_end = (w.seq + 1) * per;
    w.slot = -1;
    if (splits > 1) {  // of the tail
      w.slot = (static_cast<int64_t>(split) * a.tail + item - (a.batch * a.kv * (per / a.block_rows) - a.tail)) * a.block_rows;
    } else if (a.tail == 0 && a.work) {
      split = x - y * a.own_splits, splits = a.own_splits;
      w.slot = (static_cast<int64_t>(a.prefix_splits + split) * a.kv + w.head) * a.rows + w.row0;
    }
    w.len = w.keys = a.lens ? min(max(a.lens[w.seq], 0), a.own.keys) : a.own.keys;
    if (a.causal) {
      const int last = (min(w.row0 + a.block_rows, w.row_end) - 1 - w.seq * per) / a.group;
      w.keys = min(max(w.len - a.tokens + 1 + last, 0), a.own.keys);
    }
  }
  const int units = (min(a.block_rows, w.row_end - w.row0) + QW - 1) / QW, step = units == 1 ? 32 : BKV;
  const int steps = (w.keys + step - 1) / step;
  w.t0 = static_cast<int>(static_cast<int64_t>(steps) * split / splits);
  w.t1 = static_cast<int>(static_cast<int64_t>(steps) * (split + 1) / splits);
  w.front = w.seq < 0 ? w.t1 : 0;
  if (units == 1)
    stream_block<T, DP, WAVES, KEYS == Keys::CAUSAL>(a, w, smem);
  else if (units == 2)
    tile_block<T, DP, 2, KEYS>(a, w, smem);
  else
    tile_block<T, DP, 1, KEYS>(a, w, smem);
}

// Up to 32 rows a sequence and key head: workgroups of NW waves that all read the same rows' keys, the prefix's among them. Where
// there are few (NW 8, one a CU), a single launch does as long as the keys are few enough. Sequences of a head are neighbours: they
// share the prefix.
template <typename T, int DP, int NW, bool CAUSAL>
__global__ __launch_bounds__(64 * NW, NW == 8 ? 2 : DP == 64 ? 4 : DP == 96 ? 3 : 2) void stream_kernel(const CrossArgs a) {
  __shared__ __attribute__((aligned(1024))) T smem[stream_bytes(DP, NW) / 2];
  touch(a);
  const int split = static_cast<int>(blockIdx.z), per = a.tokens * a.group;
  Piece w;
  w.seq = static_cast<int>(blockIdx.x), w.head = static_cast<int>(blockIdx.y);
  w.row0 = w.seq * per, w.row_end = w.row0 + per;
  w.slot = a.work ? (static_cast<int64_t>(split) * a.kv + w.head) * a.rows + w.row0 : -1;
  w.len = w.keys = a.lens ? min(max(a.lens[w.seq], 0), a.own.keys) : a.own.keys;
  w.front = (a.prefix.keys + 31) / 32;
  const int64_t slices = w.front + (w.keys + 31) / 32;
  w.t0 = static_cast<int>(slices * split / a.own_splits);
  w.t1 = static_cast<int>(slices * (split + 1) / a.own_splits);
  stream_block<T, DP, NW, CAUSAL>(a, w, smem);
}

// Joins the parts of a row: CH lanes for its columns (8 each), LANES times over for as many parts at a time, joined at the end.
template <typename T, int CH, int LANES>
__global__ __launch_bounds__(256) void join_kernel(const CrossArgs a) {
  const int lane = threadIdx.x & 63, c = lane % CH, first = lane / CH % LANES, of = lane / (CH * LANES);
  const int parts = a.tail ? a.tail_splits : a.prefix_splits + a.own_splits;
  const int64_t all = a.tail ? static_cast<int64_t>(a.tail) * a.block_rows : static_cast<int64_t>(a.kv) * a.rows;
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6)) * (64 / (CH * LANES)) + of;
  if (at >= all) return;
  const float2* ml = reinterpret_cast<const float2*>(a.work + a.slots * a.dim) + at;
  float m = NONE;
  for (int p = lane % (CH * LANES); p < parts; p += CH * LANES) m = fmaxf(m, ml[p * all].x);
#pragma unroll
  for (int d = 1; d < CH * LANES; d <<= 1) m = fmaxf(m, xor_shuffle(m, d));
  const float top = fmaxf(m, LOWEST);
  const int col = 8 * c < a.dim ? 8 * c : 0;  // lanes past the columns join the first again
  const float* from = a.work + at * a.dim + col;
  const int64_t step = all * a.dim;
  float l = 0.f, o[8] = {};
#pragma unroll 4
  for (int p = first; p < parts; p += LANES) {
    const float2 x = ml[p * all];
    const float4_t u = *reinterpret_cast<const float4_t*>(from + p * step);
    const float4_t v = *reinterpret_cast<const float4_t*>(from + p * step + 4);
    const float f = __builtin_amdgcn_exp2f(x.x - top);
    l = __builtin_fmaf(x.y, f, l);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] = __builtin_fmaf(u[e], f, o[e]);
      o[e + 4] = __builtin_fmaf(v[e], f, o[e + 4]);
    }
  }
#pragma unroll
  for (int d = CH; d < CH * LANES; d <<= 1) {
    l = l + xor_shuffle(l, d);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = o[e] + xor_shuffle(o[e], d);
  }
  if (first != 0 || 8 * c >= a.dim) return;
  const float inv = inverse(m, l);
  vec8_t<T> y;
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = static_cast<T>(o[e] * inv);
  const int per = a.tokens * a.group;
  int head, seq, rest;
  if (a.tail) {
    const int whole = per / a.block_rows, item = a.batch * a.kv * whole - a.tail + static_cast<int>(at / a.block_rows);
    const int run = item / whole;
    head = run / a.batch, seq = run - head * a.batch;
    rest = (item - run * whole) * a.block_rows + static_cast<int>(at % a.block_rows);
  } else {
    head = static_cast<int>(at / a.rows);
    const int row = static_cast<int>(at - static_cast<int64_t>(head) * a.rows);
    seq = row / per, rest = row - seq * per;
  }
  const int token = rest / a.group;
  T* to = static_cast<T*>(a.out) + seq * a.ob + token * a.ot + (head * a.group + rest - token * a.group) * a.oh + col;
  *reinterpret_cast<vec4_t<T>*>(to) = vec4_t<T>{y[0], y[1], y[2], y[3]};
  *reinterpret_cast<vec4_t<T>*>(to + 4) = vec4_t<T>{y[4], y[5], y[6], y[7]};
}

template <typename T, int DP>
static void launch_cross(const CrossArgs& a, int64_t blocks, int stream, hipStream_t st) {
  const dim3 runs(a.batch, a.kv, a.own_splits);
  const dim3 all(static_cast<unsigned>(blocks));
  if (stream == 8)
    a.causal ? stream_kernel<T, DP, 8, true><<<runs, 64 * 8, 0, st>>>(a) : stream_kernel<T, DP, 8, false><<<runs, 64 * 8, 0, st>>>(a);
  else if (stream == 4)
    a.causal ? stream_kernel<T, DP, 4, true><<<runs, 64 * 4, 0, st>>>(a) : stream_kernel<T, DP, 4, false><<<runs, 64 * 4, 0, st>>>(a);
  else if (a.mask)
    cross_kernel<T, DP, Keys::LISTED><<<all, 64 * WAVES, 0, st>>>(a);
  else if (a.causal)
    cross_kernel<T, DP, Keys::CAUSAL><<<all, 64 * WAVES, 0, st>>>(a);
  else
    cross_kernel<T, DP, Keys::ALL><<<all, 64 * WAVES, 0, st>>>(a);
  if (!a.work) return;
  constexpr int CH = DP == 64 ? 8 : 16;
  const int parts = a.tail ? a.tail_splits : a.prefix_splits + a.own_splits;
  const int64_t rows = a.slots / parts;
  // a row's parts in several lanes at once where rows are few (16 rows of 32 parts, 64 columns: 17 us in one, 4.6 in 8; 24 576
  // rows of 2 parts: 6.0 in one, 14.7 in 8)
  if (rows * CH < 65536)
    join_kernel<T, CH, 64 / CH><<<dim3(static_cast<unsigned>((rows + 3) / 4)), 256, 0, st>>>(a);
  else
    join_kernel<T, CH, 1><<<dim3(static_cast<unsigned>((rows + 4 * (64 / CH) - 1) / (4 * (64 / CH)))), 256, 0, st>>>(a);
}

// Kernels of 64, 96 and 128 columns; between them the rest is zeros, which take products and LDS but no memory: 32, 48, 64
// columns in 156, 165, 178 us, 72, 80, 88, 96 in 242 to 253, 104 and 128 in 319 and 322 (8 x 1024 queries, 4096 keys, 16 heads,
// fp16); 32, 64, 72, 96, 128 in 15, 25, 33, 43, 59 (64 single tokens, 1025 keys, 32 / 8 heads).
template <typename T>
static void launch_cross_dim(const CrossArgs& a, int64_t blocks, int stream, hipStream_t st) {
  if (a.dim <= 64)
    launch_cross<T, 64>(a, blocks, stream, st);
  else if (a.dim <= 96)
    launch_cross<T, 96>(a, blocks, stream, st);
  else
    launch_cross<T, 128>(a, blocks, stream, st);
}

// How rows and keys are cut, from the sizes alone (the workspace's size follows from it).
struct Plan {
  int stream;  // waves of stream_kernel's workgroups, 0: cross_kernel
  int64_t block_rows, own_tiles, own_splits, prefix_tiles, prefix_splits, tail, tail_splits, slots, blocks;
};

constexpr int64_t CUS = 256;
// Bytes of keys and values up to which one workgroup reads a sequence's and head's: 8.6 us, where two launches take 9 and more.
constexpr int64_t ONE_GO = int64_t(5) << 16;
// Bytes of a prefix that a CU's streams may read, once for each of theirs, in place of pieces of its own and a join: 12.6 -> 6.5 us
// at 32 KB (64 x 4 tokens, 64 + 64 keys, 8 heads x 64), 22.6 -> 18.9 at 250 (300 x 1, 100 + 50, 16 / 4 x 128), 17.4 -> 16.1 at 500
// (64 x 1, 500 + 100, 32 / 8 x 128), 19.0 -> 19.6 at 600, 17.6 -> 22.9 at 1000.
constexpr double AGAIN = 512 << 10;

// Times in us on this card: a tile of 64 keys takes a workgroup of four units `alone` at least, and a CU `cu` for each workgroup in
// it.
struct Rates {
  double alone, cu;
  int64_t resident;  // workgroups a CU holds
};
static Rates rates_of(int64_t D) {
  if (D <= 64) return {1.0, 0.55, 4};
  if (D <= 96) return {1.1, 0.80, 3};
  return {1.2, 0.95, 2};
}

// Cuts of the keys of `blocks` workgroups that have `tiles` tiles each, beside `others` workgroups of `theirs`: the cut that ends
// first. A CU's load is taken halfway between the mean and the fullest CU's, and rounds halfway between their number and the next
// whole one; the two kinds share the chip by their tiles. Parts of a row are written and read again, half of it within the caches,
// and joined by a second launch. From two workgroups a CU on keys are not cut: what that loses is small (640 of 66 tiles: 124 us
// uncut, 118 in two, 127 in four), and a cut may lose more (720 of 32: 65, 78, 91). Over the 32 shapes timed with 1 .. 48 cuts (1
// to 128 sequences of 1 to 1025 tokens, 512 to 16384 keys, 9 of them with a prefix) its choice takes 2 % more than the fastest
// cut on average and 14 % at worst.
static int64_t split_keys(int64_t blocks, int64_t tiles, int64_t others, int64_t theirs, int64_t rows, int64_t D, bool joined) {
  if (blocks <= 0 || tiles <= 1 || (!joined && blocks >= 2 * CUS)) return 1;
  const Rates r = rates_of(D);
  const double mine = static_cast<double>(blocks) * static_cast<double>(tiles);
  const double share = mine / (mine + static_cast<double>(others) * static_cast<double>(theirs));
  const double slots = static_cast<double>(CUS * r.resident) * share;
  int64_t best = 1;
  double least = 0;
  for (int64_t s = 1; s <= std::min<int64_t>(64, (tiles + 1) / 2); ++s) {
    const double all = static_cast<double>(blocks * s), rounds = std::max(1.0, all / slots);
    const double together = std::min(0.5 * (all / CUS + std::ceil(all / CUS)), static_cast<double>(r.resident));
    const double turns = static_cast<double>((tiles + s - 1) / s) * 0.5 * (rounds + std::ceil(rounds));
    const double t = turns * std::max(r.alone, r.cu * together) +
                     (s > 1 || joined ? 6.0 + static_cast<double>(s * rows * (D + 2)) * 8.0 / 9e6 : 0.0);
    if (s == 1 || t < least) least = t, best = s;
  }
  return best;
}

// prefix < 0: none
static Plan plan_of(int64_t batch, int64_t tokens, int64_t keys, int64_t prefix, int64_t kv, int64_t group, int64_t D) {
  Plan p{};
  const int64_t per = tokens * group, rows = batch * per, runs = batch * kv, all = keys + std::max<int64_t>(prefix, 0);
  const bool cut = all * D * 4 > ONE_GO;
  p.own_splits = p.tail_splits = 1;
  const double again = static_cast<double>((runs + CUS - 1) / CUS) * static_cast<double>(prefix) * static_cast<double>(D * 4);
  if (per <= QW && (prefix <= 0 || (runs <= CUS ? batch == 1 || !cut : again <= AGAIN))) {
    p.stream = runs <= CUS ? 8 : 4;
    p.block_rows = QW;
    p.own_tiles = 1;
    if (cut) p.own_splits = std::max<int64_t>(1, std::min(CUS / std::max<int64_t>(runs, 1), all / 256));
    p.slots = p.own_splits > 1 ? p.own_splits * rows * kv : 0;
    p.blocks = runs * p.own_splits;
    return p;
  }
  const int64_t most = prefix > 0 ? rows : per;
  p.block_rows = most <= QW ? QW : most <= 2 * QW ? 2 * QW : 4 * QW;
  p.own_tiles = (per + p.block_rows - 1) / p.block_rows;
  const int64_t own = p.own_tiles * runs, tiles = (keys + BKV - 1) / BKV;
  if (prefix == 0) {  // nothing to join: 12.5 -> 7.6 us for 4 x 128 tokens of 16 heads x 64
    p.own_splits = split_keys(own, tiles, 0, 0, rows * kv, D, false);
    p.slots = p.own_splits > 1 ? p.own_splits * rows * kv : 0;
  } else if (prefix > 0) {
    p.prefix_tiles = (rows + p.block_rows - 1) / p.block_rows;
    const int64_t shared = p.prefix_tiles * kv, front = (prefix + BKV - 1) / BKV;
    p.own_splits = split_keys(own, tiles, shared, front, rows * kv, D, true);
    p.prefix_splits = split_keys(shared, front, own, tiles, rows * kv, D, true);
    p.slots = (p.own_splits + p.prefix_splits) * rows * kv;
  } else {
    const Rates r = rates_of(D);
    const int64_t slots = CUS * r.resident, whole = per / p.block_rows * runs, last = whole % slots;
    p.own_splits = split_keys(own, tiles, 0, 0, rows * kv, D, false);
    if (p.own_splits == 1 && whole > slots && last > 0) {
      // The last round's workgroups, cut so that they fill the chip too, if that saves more than the join costs: 120 -> 99 us (2 x
      // 1029 queries, 2100 keys, 32 / 1 heads x 128), 246 -> 231 (9 x 1024, 5184, 16 x 64), 122 -> 122 (9 x 1024, 2100)
      const int64_t cuts = std::min<int64_t>(slots / last, tiles / 8);
      const double now = static_cast<double>(tiles) * std::max(r.alone, r.cu * static_cast<double>(last) / CUS);
      const double then = static_cast<double>(tiles) / static_cast<double>(std::max<int64_t>(cuts, 1)) *
                              std::max(r.alone, r.cu * static_cast<double>(last * cuts) / CUS) +
                          5.0 + static_cast<double>(cuts * last * p.block_rows * (D + 2)) * 8.0 / 4.5e6;
      if (cuts > 1 && then < now) p.tail = last, p.tail_splits = cuts;
    }
    p.slots = p.tail ? p.tail_splits * p.tail * p.block_rows : p.own_splits > 1 ? p.own_splits * rows * kv : 0;
  }
  p.blocks = own * p.own_splits + p.tail * (p.tail_splits - 1) + p.prefix_tiles * kv * p.prefix_splits;
  return p;
}

}  // namespace ff

using namespace ff;

namespace {

// Rows of D 16-bit values: [batch, tokens, heads] by strides in elements.
struct Rows {
  const void* p;
  int64_t n[3], stride[3];
};

// A dimension of one row has no stride.
Rows plain(Rows r) {
  for (int d = 0; d < 3; ++d) r.stride[d] = r.n[d] > 1 ? r.stride[d] : 0;
  return r;
}

// Sorts the dimensions that have several rows at a pitch, in bytes, from the smallest up.
int pitches(const Rows& r, int64_t (&n)[3], int64_t (&pitch)[3]) {
  int dims = 0;
  for (int d = 0; d < 3; ++d) {
    if (r.n[d] <= 1 || r.stride[d] == 0) continue;
    int at = dims++;
    for (; at > 0 && pitch[at - 1] > 2 * r.stride[d]; --at) n[at] = n[at - 1], pitch[at] = pitch[at - 1];
    n[at] = r.n[d], pitch[at] = 2 * r.stride[d];
  }
  return dims;
}

// The bytes of such rows: rows that touch or overlap as one run, and the closest dimension as its whole extent where three stay.
Extent extent_of(const Rows& r, int64_t D) {
  Extent e = range(r.p, 2 * D);
  if (r.n[0] == 0 || r.n[1] == 0 || r.n[2] == 0) return range(r.p, 0);
  int64_t n[3], pitch[3];
  const int dims = pitches(r, n, pitch);
  int d = 0;
  while (d < dims && (pitch[d] <= e.len || dims - d > 2)) e.len += (n[d] - 1) * pitch[d], ++d;
  for (int i = 0; d < dims; ++d, ++i) e.n[i] = n[d], e.pitch[i] = pitch[d];
  return e;
}

bool overlaps_itself(const Rows& r, int64_t D) {
  for (int d = 0; d < 3; ++d)
    if (r.n[d] > 1 && r.stride[d] == 0) return true;
  int64_t n[3], pitch[3], len = 2 * D;
  const int dims = pitches(r, n, pitch);
  for (int d = 0; d < dims; ++d) {
    if (pitch[d] < len) return true;
    len += (n[d] - 1) * pitch[d];
  }
  return false;
}

bool misaligned(const Rows& r, uint64_t bytes) {
  uint64_t low = reinterpret_cast<uintptr_t>(r.p);
  for (int d = 0; d < 3; ++d) low |= r.n[d] > 1 ? static_cast<uint64_t>(r.stride[d]) * 2 : 0;
  return (low & (bytes - 1)) != 0;
}

bool negative(const Rows& r) { return r.stride[0] < 0 || r.stride[1] < 0 || r.stride[2] < 0; }

// Sizes that both entries share: null and the plan if they are taken.
const char* bad_sizes(int64_t batch, int64_t tokens, int64_t keys, int64_t prefix, int64_t heads, int64_t kv, int64_t D,
                      Plan& p) {
  if (D <= 0 || D % 8 != 0 || D > 128) return "heads must be a multiple of 8 columns, at most 128";
  if (heads <= 0 || kv <= 0 || heads > 65535 || heads % kv != 0)
    return "need 0 < heads <= 65535, a multiple of kv_heads > 0";
  if (batch < 0 || tokens < 0 || keys < 0 || prefix < -1 || batch > 0x7fffffff || tokens > 0x7fffffff)
    return "sizes must not be negative, nor reach 2^31";
  if (keys > 0x7fffff00 || prefix > 0x7fffff00) return "need fewer than 2^31 - 255 keys";
  if (batch != 0 && tokens != 0 && (tokens > 0x7fffffff / batch || batch * tokens > 0x7fffffff / heads))
    return "need batch * tokens * heads < 2^31";
  p = plan_of(batch, tokens, keys, prefix, kv, heads / kv, D);
  const int64_t joined = p.tail ? p.tail * p.block_rows : p.slots > 0 ? batch * tokens * heads : 0;
  if (p.blocks >= (int64_t(1) << 24) || joined > (1 << 26) - 4) return "too many rows for one launch";
  return nullptr;
}

int attend(const char* name, const Rows& q, const Rows& k, const Rows& v, const Rows* pk, const Rows* pv, const Rows& out,
           int dtype, int64_t D, float scale, const int32_t* lens, const uint8_t* mask, int64_t mask_batch, float* work,
           int64_t work_size, void* stream) {
  auto bad = [&](const char* msg) { return fail(FF_EINVAL, std::string(name) + ": " + msg); };
  const int64_t batch = q.n[0], tokens = q.n[1], heads = q.n[2], keys = k.n[1], kv = k.n[2], prefix = pk ? pk->n[1] : -1;
  if (dtype != FF_F16 && dtype != FF_BF16) return bad("q, k, v and out must be fp16 or bf16");
  Plan p;
  if (const char* msg = bad_sizes(batch, tokens, keys, prefix, heads, kv, D, p)) return bad(msg);
  const float c = scale * 1.4426950408889634f;  // log2(e)
  if (!(scale > 0.f) || !std::isfinite(c)) return bad("scale must be > 0, and finite times log2(e)");
  if (batch == 0 || tokens == 0) return FF_OK;
  const Rows* given[6] = {&q, &k, &v, pk, pv, &out};
  for (const Rows* r : given) {
    if (!r) continue;
    if (!r->p && r->n[1] != 0) return bad("null pointer");
    if (negative(*r)) return bad("strides must not be negative");
    if (misaligned(*r, r == &out ? 8 : 16))
      return bad("misaligned pointer or stride (q, k, v: multiples of 16 bytes; out: of 8)");
  }
  for (const Rows* r : {&k, &v, pk, pv})
    if (r && r->n[1] > 1 && r->stride[1] >= (1 << 24)) return bad("tokens of k and v must be fewer than 2^24 elements apart");
  if (mask_batch < 0) return bad("strides must not be negative");  // a batch of one: index 0 alone
  const int64_t need = p.slots * (D + 2);
  if (need > 0 && (!work || work_size < need)) return bad("the workspace is too small");
  if ((reinterpret_cast<uintptr_t>(work) & 15) || (reinterpret_cast<uintptr_t>(lens) & 3)) return bad("misaligned pointer");
  if (overlaps_itself(out, D)) return bad("the rows of out overlap");
  // Rows are read and written by different workgroups, in no order.
  const Extent to = extent_of(out, D), scratch = range(work, need * 4);
  const Extent read[7] = {extent_of(q, D), extent_of(k, D), extent_of(v, D), pk ? extent_of(*pk, D) : range(nullptr, 0),
                          pv ? extent_of(*pv, D) : range(nullptr, 0), range(lens, lens ? batch * 4 : 0),
                          Extent{reinterpret_cast<uintptr_t>(mask), {batch, 1}, {mask_batch, 0}, mask ? keys : 0}};
  const bool used = scratch.len > 0;
  if (used && !clear_of(to, scratch)) return bad("out overlaps the workspace");
  for (const Extent& e : read) {
    if (e.len == 0) continue;
    if (!clear_of(to, e)) return bad("out overlaps what is read");
    if (used && !clear_of(scratch, e)) return bad("the workspace overlaps what is read");
  }
  CrossArgs a{};
  a.q = q.p, a.out = const_cast<void*>(out.p);
  a.qb = q.stride[0], a.qt = q.stride[1], a.qh = q.stride[2];
  a.ob = out.stride[0], a.ot = out.stride[1], a.oh = out.stride[2];
  auto source = [](const Rows& x, const Rows& y) {
    return KeySource{x.p, y.p, x.stride[0], x.stride[1], x.stride[2], y.stride[0], y.stride[1], y.stride[2],
                     static_cast<int>(x.n[1])};
  };
  a.own = source(k, v);
  if (pk) a.prefix = source(*pk, *pv);
  a.lens = lens, a.mask = mask, a.mask_b = mask_batch, a.work = p.slots > 0 ? work : nullptr, a.slots = p.slots;
  a.batch = static_cast<int>(batch), a.tokens = static_cast<int>(tokens), a.kv = static_cast<int>(kv);
  a.group = static_cast<int>(heads / kv), a.dim = static_cast<int>(D), a.causal = pk && tokens > 1;  // a single token sees all
  a.rows = static_cast<int>(batch * tokens) * a.group;
  a.block_rows = static_cast<int>(p.block_rows), a.own_tiles = static_cast<int>(p.own_tiles);
  a.own_splits = static_cast<int>(p.own_splits), a.prefix_tiles = static_cast<int>(p.prefix_tiles);
  a.prefix_splits = static_cast<int>(p.prefix_splits);
  a.tail = static_cast<int>(p.tail), a.tail_splits = static_cast<int>(p.tail_splits);
  a.c = c;
  if (dtype == FF_F16)
    launch_cross_dim<half_t>(a, p.blocks, p.stream, as_stream(stream));
  else
    launch_cross_dim<bf16_t>(a, p.blocks, p.stream, as_stream(stream));
  return check_launch(name);
}

}  // namespace

extern "C" int64_t ff_cross_attention_work(int64_t B, int64_t L, int64_t S, int64_t heads, int64_t kv_heads, int64_t D) {
  Plan p;
  return bad_sizes(B, L, S, -1, heads, kv_heads, D, p) ? 0 : p.slots * (D + 2);
}

extern "C" int64_t ff_prefix_attention_work(int64_t B, int64_t L, int64_t P, int64_t S, int64_t heads, int64_t kv_heads,
                                            int64_t D) {
  Plan p;
  return P < 0 || bad_sizes(B, L, S, P, heads, kv_heads, D, p) ? 0 : p.slots * (D + 2);
}

extern "C" int ff_cross_attention(const void* q, int64_t q_batch, int64_t q_token, int64_t q_head, const void* k,
                                  int64_t k_batch, int64_t k_token, int64_t k_head, const void* v, int64_t v_batch,
                                  int64_t v_token, int64_t v_head, void* out, int64_t o_batch, int64_t o_token,
                                  int64_t o_head, int dtype, int64_t B, int64_t L, int64_t S, int64_t heads,
                                  int64_t kv_heads, int64_t D, float scale, const int32_t* lens, const uint8_t* mask,
                                  int64_t mask_batch, float* work, int64_t work_size, void* stream) {
  clear_error();
  return attend("cross_attention", plain({q, {B, L, heads}, {q_batch, q_token, q_head}}),
                plain({k, {B, S, kv_heads}, {k_batch, k_token, k_head}}),
                plain({v, {B, S, kv_heads}, {v_batch, v_token, v_head}}), nullptr, nullptr,
                plain({out, {B, L, heads}, {o_batch, o_token, o_head}}), dtype, D, scale, lens, mask, mask_batch, work,
                work_size, stream);
}

extern "C" int ff_prefix_attention(const void* q, int64_t q_batch, int64_t q_token, int64_t q_head, const void* prefix_k,
                                   int64_t pk_token, int64_t pk_head, const void* prefix_v, int64_t pv_token,
                                   int64_t pv_head, const void* k, int64_t k_batch, int64_t k_token, int64_t k_head,
                                   const void* v, int64_t v_batch, int64_t v_token, int64_t v_head, void* out,
                                   int64_t o_batch, int64_t o_token, int64_t o_head, int dtype, int64_t B, int64_t L,
                                   int64_t P, int64_t S, int64_t heads, int64_t kv_heads, int64_t D, float scale,
                                   const int32_t* lens, float* work, int64_t work_size, void* stream) {
  clear_error();
  if (P < 0) return fail(FF_EINVAL, "prefix_attention: sizes must not be negative, nor reach 2^31");
  const Rows pk = plain({prefix_k, {1, P, kv_heads}, {0, pk_token, pk_head}});
  const Rows pv = plain({prefix_v, {1, P, kv_heads}, {0, pv_token, pv_head}});
  return attend("prefix_attention", plain({q, {B, L, heads}, {q_batch, q_token, q_head}}),
                plain({k, {B, S, kv_heads}, {k_batch, k_token, k_head}}),
                plain({v, {B, S, kv_heads}, {v_batch, v_token, v_head}}), &pk, &pv,
                plain({out, {B, L, heads}, {o_batch, o_token, o_head}}), dtype, D, scale, lens, nullptr, 0, work, work_size,
                stream);
}
