// Attention of queries to keys and values of another length (cross_attention), and of a batch whose sequences share a prefix
// (prefix_attention), on the fp16 and bf16 matrix cores of gfx950.
//
// o = sum_j p_j v_j / sum_j p_j with p_j = 2^(c q.k_j - m), c = scale log2(e), over the keys that a query sees; m is a reference
// near the largest c q.k_j, raised as larger ones come, and drops out of the quotient. q is used as given: c multiplies the
// products in fp32 (folded into q it would round q once more). Sums, p's sum, m and O are fp32; p is rounded to the values' type
// for the second product, half a step each, which is what the matrix cores take.
//
// Rows: the G = heads / kv_heads query heads of a key head read the same keys, so a key head's rows are (sequence, token, head
// of the group). A workgroup has four waves and 32, 64 or 128 rows; 32 rows are a unit. Four units: a wave each, over all
// keys. Two: two waves a unit, each over one half of every 64-key tile. One (single tokens): all four share it, by halves and by
// tiles of either parity. Waves that share a unit are joined through LDS.
// Keys: a workgroup runs over all keys of its rows, or, where rows are few, over one of several runs of tiles; the runs' O, m
// and l then go to the workspace in fp32 and join_kernel joins them in a fixed order.
// Shared prefix: its keys have no sequence, so the rows of all sequences together read it; the same launch's other workgroups
// take each sequence's own keys, and join_kernel joins the parts.
//
// K and V stream through two LDS slots of 64 keys (buffer loads straight into LDS). Rows that no query of the workgroup may see
// (past the length, or masked) and columns past D are loads out of the descriptor's range: they read as zeros and cost no
// traffic, and what the memory there holds never reaches a product. Per wave, S^T = K Q^T by 32x32x16 products leaves a lane
// with one query and 16 of 32 keys; P^T then is the column operand of O^T = V^T P^T, V read with the transposing
// ds_read_b64_tr_b16. Both tiles are row-major, their 16-byte chunks XOR-swizzled against bank conflicts.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attention_common.h"
#include "gemm_common.h"

namespace ff {

constexpr int QW = 32;     // rows of a unit
constexpr int WAVES = 4;   // waves a workgroup
constexpr int BKV = 64;    // keys a tile
constexpr float SUM_LIMIT = 8192.f;  // a lane's sum of p over a half tile above which m is raised (fp16 holds p up to it)
constexpr float LOWEST = -3.402823466e38f;

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
  float* work;  // parts' O [part, kv, rows, D], then their (m, l) [part, kv, rows, 2]; null: one part, written to out
  int batch, tokens, kv, group, dim, causal;
  int rows;  // batch * tokens * group: of a key head
  int block_rows, own_tiles, own_splits, prefix_tiles, prefix_splits;
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

// What a workgroup works on; the same in all its lanes.
struct Piece {
  int seq;          // -1: the shared prefix, rows of all sequences
  int head;         // key head
  int row0, row_end;
  int keys, len;    // keys that some row sees; the sequence's length
  int t0, t1;       // tiles
  int part;
};

template <typename T, int DP, int SPLIT>
__device__ __forceinline__ void cross_block(const CrossArgs& a, const Piece& w, T* smem) {
  constexpr int CH = DP / 8, TILE = BKV * DP, LPW = CH / 4, KS = DP / 16, DT = DP / 32;
  typedef vec8_t<T> T8;
  typedef vec4_t<T> T4;
  const uint32_t smem_lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void*)smem));
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 31, fh = lane >> 5;
  const int unit = SPLIT == 2 ? 0 : (SPLIT ? wave >> 1 : wave);
  const int half_sel = SPLIT ? wave & 1 : 0, parity = SPLIT == 2 ? wave >> 1 : 0;
  const bool active = w.row0 + unit * QW < w.row_end;  // other waves only load

  // The lane's row: sequence, token, head
  const int row = w.row0 + unit * QW + fr, real = min(row, w.row_end - 1), per = a.tokens * a.group;
  const int seq = w.seq < 0 ? real / per : w.seq, rest = real - seq * per, token = rest / a.group;
  const int head = w.head * a.group + rest - token * a.group;
  const int limit = a.causal && w.seq >= 0 ? min(max(w.len - a.tokens + 1 + token, 0), w.keys) : w.keys;

  T8 qf[KS];  // column operand of S^T: the lane's row, columns 16 s + 8 fh + 0..7
  {
    const T* q = static_cast<const T*>(a.q) + seq * a.qb + token * a.qt + head * a.qh;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      qf[s] = T8{};
      if (16 * s + 8 * fh < a.dim) qf[s] = *reinterpret_cast<const T8*>(q + 16 * s + 8 * fh);
    }
    // consumed here, so that the compiler's wait for these loads stands before the loop and not in it
#pragma unroll
    for (int s = 0; s < KS; ++s) asm volatile("" ::"v"(qf[s]));
  }

  const KeySource& src = w.seq < 0 ? a.prefix : a.own;
  const int64_t at = max(w.seq, 0);
  const T* kbase = static_cast<const T*>(src.k) + at * src.kb + w.head * src.kh;
  const T* vbase = static_cast<const T*>(src.v) + at * src.vb + w.head * src.vh;
  const uint8_t* mask = a.mask && w.seq >= 0 ? a.mask + at * a.mask_b : nullptr;

  // Tile loads: wave w fills the 1 KB blocks LPW w .. of either tile, lane l the chunk l of a block; it fetches what the swizzle
  // puts there.
  uint32_t voff_k[LPW], voff_v[LPW];
  int lrow[LPW];
#pragma unroll
  for (int p = 0; p < LPW; ++p) {
    const int n = (LPW * wave + p) * 64 + lane, r = n / CH, slot = n % CH;
    const int ck = k_slot<DP>(r, slot), cv = v_slot<DP>(r, slot);
    lrow[p] = r;
    voff_k[p] = 8 * ck < a.dim ? static_cast<uint32_t>((r * static_cast<int>(src.kt) + ck * 8) * 2) : OOB_OFFSET;
    voff_v[p] = 8 * cv < a.dim ? static_cast<uint32_t>((r * static_cast<int>(src.vt) + cv * 8) * 2) : OOB_OFFSET;
  }
  auto issue = [&](int tile, uint64_t word) __attribute__((always_inline)) {
    const int st = (tile - w.t0) & 1, rows = min(BKV, w.keys - tile * BKV);
    const int64_t first = static_cast<int64_t>(tile) * BKV;
    const int nk = ((rows - 1) * static_cast<int>(src.kt) + a.dim) * 2, nv = ((rows - 1) * static_cast<int>(src.vt) + a.dim) * 2;
    const T *k = kbase + first * src.kt, *v = vbase + first * src.vt;
#pragma unroll
    for (int p = 0; p < LPW; ++p) {
      const bool in = !mask || ((word >> lrow[p]) & 1);
      buffer_to_lds(k, nk, reinterpret_cast<uint8_t*>(smem + st * TILE + (LPW * wave + p) * 512), in ? voff_k[p] : OOB_OFFSET);
      buffer_to_lds(v, nv, reinterpret_cast<uint8_t*>(smem + (2 + st) * TILE + (LPW * wave + p) * 512),
                    in ? voff_v[p] : OOB_OFFSET);
    }
  };
  // The keys of a tile that may be seen, as bits.
  auto mask_byte = [&](int tile) __attribute__((always_inline)) {
    const int key = tile * BKV + lane;
    return mask && tile < w.t1 && key < w.keys ? mask[key] : uint8_t(0);
  };
  auto valid = [&](int tile, uint8_t byte) __attribute__((always_inline)) {
    if (mask) return static_cast<uint64_t>(__ballot(byte != 0));
    const int n = w.keys - tile * BKV;
    return n >= 64 ? ~uint64_t(0) : (uint64_t(1) << n) - 1;
  };

  // LDS read offsets within a tile. K fragment (half, s): row 32 half + fr, chunk 2 s + fh. V^T fragment (dt, half, tt), part j:
  // lane l of 16 addresses row 32 half + 16 tt + 8 j + 4 fh + l / 4, columns 32 dt + 16 (group) + 4 (l % 4), and receives four
  // keys in a row of column 32 dt + fr: the keys of P^T's slots.
  int koff[KS], voff[DT];
#pragma unroll
  for (int s = 0; s < KS; ++s) koff[s] = (fr + 32 * half_sel) * DP + k_slot<DP>(fr, 2 * s + fh) * 8;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    const int r = 4 * fh + ((lane & 15) >> 2), col = dt * 32 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    voff[dt] = (r + 32 * half_sel) * DP + v_slot<DP>(r, col >> 3) * 8 + (col & 7);
  }

  float16_t o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
  float m = LOWEST, l_run = 0.f, hs[2] = {0.f, 0.f};
  float16_t xs;  // S^T of a half: keys 8 (r / 4) + 4 fh + r % 4
  T8 pf[2];
  int ka[KS], va[DT];

  auto qk = [&](int half) __attribute__((always_inline)) {
    const float16_t zero = {};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const T8 kf = *reinterpret_cast<const T8*>(smem + ka[s] + half * 32 * DP);
      xs = mfma(kf, qf[s], s == 0 ? zero : xs);
    }
  };
  auto soft = [&](int half) __attribute__((always_inline)) {
    float e[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      e[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(xs[r], a.c, -m));
      pf[r >> 3][r & 7] = static_cast<T>(e[r]);
    }
#pragma unroll
    for (int n = 8; n >= 1; n >>= 1)
#pragma unroll
      for (int r = 0; r < n; ++r) e[r] = e[r] + e[r + n];
    hs[half] = e[0];
  };
  // A half whose p passed the limit: m becomes the largest c S of the half, O and l follow.
  auto raise = [&](int half) __attribute__((always_inline)) {
    float top = xs[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, xs[r]);
    top = fmaxf(top, xor_shuffle(top, 32)) * a.c;
    const float m_old = m;
    m = fmaxf(m, top);
    const float corr = __builtin_amdgcn_exp2f(m_old - m);
    l_run *= corr;
    if (half == 1) hs[0] *= corr;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[dt][r] *= corr;
    soft(half);
  };
  auto pv = [&](auto halfc) __attribute__((always_inline)) {
    constexpr int half = decltype(halfc)::value;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      T4 v[4];  // [2 tt + j]
      const uint32_t base = smem_lds + 2u * static_cast<uint32_t>(va[dt]);
      tr_read<(half * 32 + 0) * DP * 2>(v[0], base);
      tr_read<(half * 32 + 8) * DP * 2>(v[1], base);
      tr_read<(half * 32 + 16) * DP * 2>(v[2], base);
      tr_read<(half * 32 + 24) * DP * 2>(v[3], base);
      asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]));
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
        o[dt] = mfma(__builtin_shufflevector(v[2 * tt], v[2 * tt + 1], 0, 1, 2, 3, 4, 5, 6, 7), pf[tt], o[dt]);
    }
  };
  auto half_tile = [&](int tile, uint64_t word, auto halfc) __attribute__((always_inline)) {
    constexpr int half = decltype(halfc)::value;
    const int h = SPLIT ? half_sel : half;  // of the tile
    qk(half);
    const int left = limit - (tile * BKV + 32 * h);
    uint32_t bits = static_cast<uint32_t>(word >> (32 * h));
    bits &= left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1;
    if (__any(bits != ~0u)) {
      bits >>= 4 * fh;
#pragma unroll
      for (int r = 0; r < 16; ++r) xs[r] = (bits >> (8 * (r >> 2) + (r & 3))) & 1 ? xs[r] : -__builtin_inff();
    }
    soft(half);
    if (__any(hs[half] > SUM_LIMIT)) raise(half);
    pv(halfc);
  };

  if (w.t0 < w.t1) {
    uint64_t word = valid(w.t0, mask_byte(w.t0)), next = 0;
    uint8_t byte = mask_byte(w.t0 + 1);
    issue(w.t0, word);
    for (int tile = w.t0; tile < w.t1; ++tile) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();  // no fence: the wait covers this thread's LDS writes
      if (tile + 1 < w.t1) {         // its slot was last read for tile - 1, which every wave has finished
        next = valid(tile + 1, byte);
        issue(tile + 1, next);
        byte = mask_byte(tile + 2);
      }
      const int st = (tile - w.t0) & 1;
      if (active && (SPLIT != 2 || ((tile - w.t0) & 1) == parity) && word != 0) {
        // read bases, opaque to the compiler so that the fragment offsets fold into the reads' immediate offsets
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          ka[s] = st * TILE + koff[s];
          asm volatile("" : "+v"(ka[s]));
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          va[dt] = (2 + st) * TILE + voff[dt];
          asm volatile("" : "+v"(va[dt]));
        }
        hs[1] = 0.f;
        half_tile(tile, word, std::integral_constant<int, 0>{});
        if constexpr (!SPLIT) half_tile(tile, word, std::integral_constant<int, 1>{});
        l_run += hs[0] + hs[1];
      }
      word = next;
    }
  }

  if constexpr (SPLIT) {  // the waves of a unit leave O, m and l in LDS; the first joins them
    constexpr int SHARE = SPLIT == 2 ? WAVES : 2, WORDS = 16 * DT + 2;
    static_assert((WAVES - 1) * WORDS * 64 * 4 <= 4 * TILE * 2, "the joint exceeds the ring");
    const int me = SPLIT == 2 ? wave : half_sel;
    float* joint = reinterpret_cast<float*>(smem) + unit * (SHARE - 1) * WORDS * 64 + lane;
    __syncthreads();
    if (active && me != 0) {
      float* mine = joint + (me - 1) * WORDS * 64;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) mine[(dt * 16 + r) * 64] = o[dt][r];
      mine[(WORDS - 2) * 64] = m;
      mine[(WORDS - 1) * 64] = l_run;
    }
    __syncthreads();
    if (!active || me != 0) return;
    float top = m;
#pragma unroll
    for (int k = 0; k < SHARE - 1; ++k) top = fmaxf(top, joint[(k * WORDS + WORDS - 2) * 64]);
    const float c0 = __builtin_amdgcn_exp2f(m - top);
    m = top;
    l_run *= c0;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[dt][r] *= c0;
#pragma unroll
    for (int k = 0; k < SHARE - 1; ++k) {
      const float* theirs = joint + k * WORDS * 64;
      const float ck = __builtin_amdgcn_exp2f(theirs[(WORDS - 2) * 64] - top);
      l_run = __builtin_fmaf(theirs[(WORDS - 1) * 64], ck, l_run);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] = __builtin_fmaf(theirs[(dt * 16 + r) * 64], ck, o[dt][r]);
    }
  } else {
    if (!active) return;
  }

  const float l = l_run + xor_shuffle(l_run, 32);
  if (row >= w.row_end) return;
  if (a.work) {
    const int64_t n = (static_cast<int64_t>(w.part) * a.kv + w.head) * a.rows + row;
    float* to = a.work + n * a.dim;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if (dt * 32 + 8 * g + 4 * fh < a.dim)
          *reinterpret_cast<float4_t*>(to + dt * 32 + 8 * g + 4 * fh) =
              float4_t{o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]};
    if (fh == 0) {
      const int64_t parts = a.prefix_splits + a.own_splits;
      float* ml = a.work + parts * a.kv * a.rows * a.dim + 2 * n;
      ml[0] = m;
      ml[1] = l;
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // no keys: zeros
  T* to = static_cast<T*>(a.out) + seq * a.ob + token * a.ot + head * a.oh;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      T4 v;
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = static_cast<T>(o[dt][4 * g + u] * inv);
      if (dt * 32 + 8 * g + 4 * fh < a.dim) *reinterpret_cast<T4*>(to + dt * 32 + 8 * g + 4 * fh) = v;
    }
}

// Waves a SIMD: what the LDS ring leaves room for (32, 48 and 64 KB).
template <typename T, int DP>
__global__ __launch_bounds__(64 * WAVES, DP == 64 ? 4 : DP == 96 ? 3 : 2) void cross_kernel(const CrossArgs a) {
  __shared__ __attribute__((aligned(1024))) T smem[4 * BKV * DP];  // K slots, then V slots
  const int per = a.tokens * a.group, prefix_items = a.prefix_splits * a.kv * a.prefix_tiles;
  int item = static_cast<int>(blockIdx.x);
  Piece w;
  int split, splits;
  // Row tiles of one run of keys are neighbours, and neighbours share an XCD's L2; the prefix's pieces are spread over the XCDs
  // by themselves, as they differ from the others in length.
  if (item < prefix_items) {
    item = xcd_remap(item, prefix_items);
    const int x = item / a.prefix_tiles;
    split = x % a.prefix_splits, splits = a.prefix_splits;
    w.seq = -1, w.head = x / a.prefix_splits, w.part = split;
    w.row0 = (item - x * a.prefix_tiles) * a.block_rows, w.row_end = a.rows;
    w.len = w.keys = a.prefix.keys;
  } else {
    item = xcd_remap(item - prefix_items, static_cast<int>(gridDim.x) - prefix_items);
    const int x = item / a.own_tiles, y = x / a.own_splits;
    split = x - y * a.own_splits, splits = a.own_splits;
    w.seq = y / a.kv, w.head = y - w.seq * a.kv, w.part = a.prefix_splits + split;
    w.row0 = w.seq * per + (item - x * a.own_tiles) * a.block_rows, w.row_end = (w.seq + 1) * per;
    w.len = w.keys = a.lens ? min(max(a.lens[w.seq], 0), a.own.keys) : a.own.keys;
    if (a.causal) {
      const int last = (min(w.row0 + a.block_rows, w.row_end) - 1 - w.seq * per) / a.group;
      w.keys = min(max(w.len - a.tokens + 1 + last, 0), a.own.keys);
    }
  }
  const int tiles = (w.keys + BKV - 1) / BKV;
  w.t0 = static_cast<int>(static_cast<int64_t>(tiles) * split / splits);
  w.t1 = static_cast<int>(static_cast<int64_t>(tiles) * (split + 1) / splits);
  const int units = (min(a.block_rows, w.row_end - w.row0) + QW - 1) / QW;
  if (units == 1)
    cross_block<T, DP, 2>(a, w, smem);
  else if (units == 2)
    cross_block<T, DP, 1>(a, w, smem);
  else
    cross_block<T, DP, 0>(a, w, smem);
}

// Joins the parts of a row: a thread has 8 columns.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const CrossArgs a) {
  const int parts = a.prefix_splits + a.own_splits, chunks = a.dim / 8;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, all = static_cast<int64_t>(a.kv) * a.rows;
  const int64_t at = n / chunks;
  const int col = static_cast<int>(n - at * chunks) * 8;
  if (at >= all) return;
  const float2* ml = reinterpret_cast<const float2*>(a.work + parts * all * a.dim);
  float top = LOWEST;
  for (int p = 0; p < parts; ++p) top = fmaxf(top, ml[p * all + at].x);
  float l = 0.f, o[8] = {};
  for (int p = 0; p < parts; ++p) {
    const float2 x = ml[p * all + at];
    const float f = __builtin_amdgcn_exp2f(x.x - top);
    const float4_t* from = reinterpret_cast<const float4_t*>(a.work + (p * all + at) * a.dim + col);
    const float4_t u = from[0], v = from[1];
    l = __builtin_fmaf(x.y, f, l);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] = __builtin_fmaf(u[e], f, o[e]);
      o[e + 4] = __builtin_fmaf(v[e], f, o[e + 4]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  vec8_t<T> y;
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = static_cast<T>(o[e] * inv);
  const int head = static_cast<int>(at / a.rows), row = static_cast<int>(at - static_cast<int64_t>(head) * a.rows);
  const int per = a.tokens * a.group, seq = row / per, rest = row - seq * per, token = rest / a.group;
  T* to = static_cast<T*>(a.out) + seq * a.ob + token * a.ot + (head * a.group + rest - token * a.group) * a.oh + col;
  *reinterpret_cast<vec4_t<T>*>(to) = vec4_t<T>{y[0], y[1], y[2], y[3]};
  *reinterpret_cast<vec4_t<T>*>(to + 4) = vec4_t<T>{y[4], y[5], y[6], y[7]};
}

template <typename T, int DP>
static void launch_cross(const CrossArgs& a, int64_t blocks, hipStream_t st) {
  cross_kernel<T, DP><<<dim3(static_cast<unsigned>(blocks)), 64 * WAVES, 0, st>>>(a);
  if (!a.work) return;
  const int64_t threads = static_cast<int64_t>(a.kv) * a.rows * (a.dim / 8);
  join_kernel<T><<<dim3(static_cast<unsigned>((threads + 255) / 256)), 256, 0, st>>>(a);
}

template <typename T>
static void launch_cross_dim(const CrossArgs& a, int64_t blocks, hipStream_t st) {
  if (a.dim <= 64)
    launch_cross<T, 64>(a, blocks, st);
  else if (a.dim <= 96)
    launch_cross<T, 96>(a, blocks, st);
  else
    launch_cross<T, 128>(a, blocks, st);
}

// How rows and keys are cut, from the sizes alone (the workspace's size follows from it).
struct Plan {
  int64_t block_rows, own_tiles, own_splits, prefix_tiles, prefix_splits, parts, blocks;
};

constexpr int64_t WANT = 512;  // workgroups that fill the 256 CUs

static int64_t split_keys(int64_t blocks, int64_t keys) {
  const int64_t tiles = (keys + BKV - 1) / BKV;
  return std::max<int64_t>(1, std::min(WANT / std::max<int64_t>(blocks, 1), tiles / 2));
}

// prefix < 0: none
static Plan plan_of(int64_t batch, int64_t tokens, int64_t keys, int64_t prefix, int64_t kv, int64_t group) {
  Plan p{};
  const int64_t per = tokens * group, rows = batch * per, most = prefix >= 0 ? rows : per;
  p.block_rows = most <= QW ? QW : most <= 2 * QW ? 2 * QW : 4 * QW;
  p.own_tiles = (per + p.block_rows - 1) / p.block_rows;
  p.own_splits = split_keys(p.own_tiles * batch * kv, keys);
  if (prefix >= 0) {
    p.prefix_tiles = (rows + p.block_rows - 1) / p.block_rows;
    p.prefix_splits = split_keys(p.prefix_tiles * kv, prefix);
  }
  p.parts = p.own_splits + p.prefix_splits;
  p.blocks = p.own_tiles * batch * kv * p.own_splits + p.prefix_tiles * kv * p.prefix_splits;
  return p;
}

static int64_t work_of(const Plan& p, int64_t batch, int64_t tokens, int64_t heads, int64_t dim) {
  return p.parts > 1 ? p.parts * batch * tokens * heads * (dim + 2) : 0;
}

}  // namespace ff

using namespace ff;

namespace {

// Rows of D 16-bit values: [batch, tokens, heads] by strides in elements.
struct Rows {
  const void* p;
  int64_t n[3], stride[3];
};

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

// Sizes that both entries share; null if they are taken.
const char* bad_sizes(int64_t batch, int64_t tokens, int64_t keys, int64_t prefix, int64_t heads, int64_t kv, int64_t D) {
  if (D <= 0 || D % 8 != 0 || D > 128) return "heads must be a multiple of 8 columns, at most 128";
  if (heads <= 0 || kv <= 0 || heads > 65535 || heads % kv != 0)
    return "need 0 < heads <= 65535, a multiple of kv_heads > 0";
  if (batch < 0 || tokens < 0 || keys < 0 || prefix < -1 || batch > 0x7fffffff || tokens > 0x7fffffff)
    return "sizes must not be negative, nor reach 2^31";
  if (keys > 0x7fffff00 || prefix > 0x7fffff00) return "need fewer than 2^31 - 255 keys";
  if (batch != 0 && tokens != 0 && (tokens > 0x7fffffff / batch || batch * tokens > 0x7fffffff / heads))
    return "need batch * tokens * heads < 2^31";
  const Plan p = plan_of(batch, tokens, keys, prefix, kv, heads / kv);
  if (p.blocks >= (int64_t(1) << 24) || (p.parts > 1 && batch * tokens * heads * (D / 8) > 0xffffff00LL))
    return "too many rows for one launch";
  return nullptr;
}

int attend(const std::string& name, const Rows& q, const Rows& k, const Rows& v, const Rows* pk, const Rows* pv, const Rows& out,
           int dtype, int64_t D, float scale, const int32_t* lens, const uint8_t* mask, int64_t mask_batch, float* work,
           int64_t work_size, void* stream) {
  auto bad = [&](const char* msg) { return fail(FF_EINVAL, name + ": " + msg); };
  const int64_t batch = q.n[0], tokens = q.n[1], heads = q.n[2], keys = k.n[1], kv = k.n[2], prefix = pk ? pk->n[1] : -1;
  if (dtype != FF_F16 && dtype != FF_BF16) return bad("q, k, v and out must be fp16 or bf16");
  if (const char* msg = bad_sizes(batch, tokens, keys, prefix, heads, kv, D)) return bad(msg);
  if (!(scale > 0.f) || !std::isfinite(scale)) return bad("scale must be finite and > 0");
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
  if (mask_batch < 0) return bad("strides must not be negative");
  const Plan p = plan_of(batch, tokens, keys, prefix, kv, heads / kv);
  const int64_t need = work_of(p, batch, tokens, heads, D);
  if (need > 0 && (!work || work_size < need)) return bad("the workspace is too small");
  if ((reinterpret_cast<uintptr_t>(work) & 15) || (reinterpret_cast<uintptr_t>(lens) & 3)) return bad("misaligned pointer");
  if (overlaps_itself(out, D)) return bad("the rows of out overlap");
  // Rows are read and written by different workgroups, in no order.
  const Extent to = extent_of(out, D), scratch = range(work, need * 4);
  const Extent read[7] = {extent_of(q, D), extent_of(k, D), extent_of(v, D), pk ? extent_of(*pk, D) : range(nullptr, 0),
                          pv ? extent_of(*pv, D) : range(nullptr, 0), range(lens, lens ? batch * 4 : 0),
                          Extent{reinterpret_cast<uintptr_t>(mask), {batch, 1}, {mask_batch, 0}, mask ? keys : 0}};
  if (!clear_of(to, scratch)) return bad("out overlaps the workspace");
  for (const Extent& e : read) {
    if (e.len == 0) continue;
    if (!clear_of(to, e)) return bad("out overlaps what is read");
    if (need > 0 && !clear_of(scratch, e)) return bad("the workspace overlaps what is read");
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
  a.lens = lens, a.mask = mask, a.mask_b = mask_batch, a.work = need > 0 ? work : nullptr;
  a.batch = static_cast<int>(batch), a.tokens = static_cast<int>(tokens), a.kv = static_cast<int>(kv);
  a.group = static_cast<int>(heads / kv), a.dim = static_cast<int>(D), a.causal = pk != nullptr;
  a.rows = static_cast<int>(batch * tokens) * a.group;
  a.block_rows = static_cast<int>(p.block_rows), a.own_tiles = static_cast<int>(p.own_tiles);
  a.own_splits = static_cast<int>(p.own_splits), a.prefix_tiles = static_cast<int>(p.prefix_tiles);
  a.prefix_splits = static_cast<int>(p.prefix_splits);
  a.c = scale * 1.4426950408889634f;
  if (dtype == FF_F16)
    launch_cross_dim<half_t>(a, p.blocks, as_stream(stream));
  else
    launch_cross_dim<bf16_t>(a, p.blocks, as_stream(stream));
  return check_launch(name.c_str());
}

}  // namespace

extern "C" int64_t ff_cross_attention_work(int64_t B, int64_t L, int64_t S, int64_t heads, int64_t kv_heads, int64_t D) {
  if (bad_sizes(B, L, S, -1, heads, kv_heads, D)) return 0;
  return work_of(plan_of(B, L, S, -1, kv_heads, heads / kv_heads), B, L, heads, D);
}

extern "C" int64_t ff_prefix_attention_work(int64_t B, int64_t L, int64_t P, int64_t S, int64_t heads, int64_t kv_heads,
                                            int64_t D) {
  if (P < 0 || bad_sizes(B, L, S, P, heads, kv_heads, D)) return 0;
  return work_of(plan_of(B, L, S, P, kv_heads, heads / kv_heads), B, L, heads, D);
}

extern "C" int ff_cross_attention(const void* q, int64_t q_batch, int64_t q_token, int64_t q_head, const void* k,
                                  int64_t k_batch, int64_t k_token, int64_t k_head, const void* v, int64_t v_batch,
                                  int64_t v_token, int64_t v_head, void* out, int64_t o_batch, int64_t o_token,
                                  int64_t o_head, int dtype, int64_t B, int64_t L, int64_t S, int64_t heads,
                                  int64_t kv_heads, int64_t D, float scale, const int32_t* lens, const uint8_t* mask,
                                  int64_t mask_batch, float* work, int64_t work_size, void* stream) {
  clear_error();
  return attend("cross_attention", {q, {B, L, heads}, {q_batch, q_token, q_head}},
                {k, {B, S, kv_heads}, {k_batch, k_token, k_head}}, {v, {B, S, kv_heads}, {v_batch, v_token, v_head}}, nullptr,
                nullptr, {out, {B, L, heads}, {o_batch, o_token, o_head}}, dtype, D, scale, lens, mask, mask_batch, work,
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
  const Rows pk{prefix_k, {1, P, kv_heads}, {0, pk_token, pk_head}}, pv{prefix_v, {1, P, kv_heads}, {0, pv_token, pv_head}};
  return attend("prefix_attention", {q, {B, L, heads}, {q_batch, q_token, q_head}},
                {k, {B, S, kv_heads}, {k_batch, k_token, k_head}}, {v, {B, S, kv_heads}, {v_batch, v_token, v_head}}, &pk,
                &pv, {out, {B, L, heads}, {o_batch, o_token, o_head}}, dtype, D, scale, lens, nullptr, 0, work, work_size,
                stream);
}
