// Attention of the drafted tokens of a tree over the cached keys and over each other: the verification step of speculative
// decoding.  (No counterpart in the reference, whose decode step takes one token a sequence.)
//
// A KV head's T * G query rows (T drafted tokens, G query heads) share its keys, so K and V (2 * 128 elements a key) are read once for
// all of them: up to some 64 rows the bytes bound it, beyond 256 the instructions of the softmax and the matrix products.  Rows go to the
// matrix cores 16 at a time; the key axis is split over waves and workgroups, whose partial results a second launch joins.
//   scores   S^T[key][row] = K[key][dim] . Q^T[dim][row]: lane (n, j) receives the scores of row n for four keys 4j .. 4j+3 of a
//            tile of 16 ...
//   output   O[row][dim] += P[row][key] . V[key][dim]: ... which is where this product wants the weights: nothing is moved.
// bf16: v_mfma_f32_16x16x32_bf16, 32 keys a step; the weights are rounded to bf16 for the second product (half a step of 2^-8 each) and
//       the normaliser is the sum of the same rounded weights, from one more product with ones.
// fp32: v_mfma_f32_16x16x4_f32, 16 keys a step; no rounding.
// Softmax over all keys a row sees in one pass with a running base and sum, fp32.
#include "pkv_attn.h"

#pragma clang fp contract(fast)

namespace {

constexpr int kTreeWaves = 4, kWideWaves = 8, kTreeMaxSplits = 64, kTreeWorkgroups = 256;

struct TreeCall {
  const void *q;
  int64_t q_stride_b, q_stride_t;  // elements
  int n_kv_heads, group, n_draft;
  uint32_t total;                  // cached keys
  const int32_t *row_keys;
  const char *dk, *dv;
  int64_t dk_b, dk_h, dk_t, dv_b, dv_h, dv_t;  // bytes
  const uint8_t *mask;
  int64_t mask_b, mask_t;
  float scale_log2e;
  float *ws_o, *ws_ml;  // [row of (b, h)][split][query row][128], [..][2]
  void *out;
  int n_splits, row_tiles, n_pairs;  // (b, h) times splits
  int n_bh, by_keys;                 // by_keys: splits in proportion to the rows' keys, 1 + log2 of the keys of a turn; else 0
};

// A workgroup's part: a split of the keys of one (b, h), and a tile of its query rows.  Workgroups go to the eight dies in turn, and the tiles of
// one split read the same keys: they are eight numbers apart, so that a die's L2 reads the keys once for all.
struct TreePart {
  int bh, split, tile, n_splits, first;  // first: the partial result of the row's split 0
  bool any;
};

// Key counts that differ: the splits' slots go to the (at most 64) rows in proportion to their turns of keys, at least one each, so that all
// workgroups have about as much to do.  Lane l finds the slots [first, end) of row l, of which it uses n: at most a turn each, at most
// kTreeMaxSplits.  All lanes active.  3 x 4 x 9001 fp32 of which the rows see from none to all, 49 rows: 33 us; 46 with as many splits for every row.  (8 x 8 x 20000 bf16, 20 rows: 70, 79.)
struct TreeShare {
  int first, end, n;
};
__device__ __forceinline__ TreeShare tree_share(const int32_t *row_keys, uint32_t total, int n_bh, int slots, int by_keys) {
  const int lane = pkv_lane(), rk = lane < n_bh ? row_keys[lane] : 0;
  const uint32_t keys = rk <= 0 ? 0u : (uint32_t)rk < total ? (uint32_t)rk : total;
  const int turns = keys == 0 ? 1 : (int)((keys - 1) >> (by_keys - 1)) + 1, mine = lane < n_bh ? turns : 0;
  const int upto = pkv_wave_incl_scan(mine);
  const float each = (float)(slots - n_bh) / (float)__builtin_amdgcn_readlane(upto, 63);
  TreeShare t;
  t.first = lane + (int)((float)(upto - mine) * each), t.end = lane + 1 + (int)((float)upto * each);
  const int most = turns < kTreeMaxSplits ? turns : kTreeMaxSplits;
  t.n = t.end - t.first < most ? t.end - t.first : most;
  return t;
}

// SHARES: by_keys is set (of its own kernels: looked up at run time it costs every call 0.5 us).
template <bool SHARES>
__device__ __forceinline__ TreePart tree_part(const TreeCall &a) {
  const int pair = (int)blockIdx.y * 8 + (blockIdx.x & 7), tile = (int)blockIdx.x >> 3;
  if constexpr (SHARES) {
    const TreeShare t = tree_share(a.row_keys, a.total, a.n_bh, a.n_pairs, a.by_keys);
    const int bh = __builtin_popcountll(__ballot(pkv_lane() < a.n_bh && t.first <= pair)) - 1;
    const int first = __builtin_amdgcn_readlane(t.first, bh), n = __builtin_amdgcn_readlane(t.n, bh);
    return {bh, pair - first, tile, n, first, pair - first < n};
  }
  if constexpr (!SHARES) {
    const int bh = (unsigned)pair / (unsigned)a.n_splits;
    return {bh, pair - bh * a.n_splits, tile, a.n_splits, bh * a.n_splits, pair < a.n_pairs};
  }
}
static dim3 tree_grid(const TreeCall &a) { return dim3(8u * a.row_tiles, (unsigned)((a.n_pairs + 7) / 8)); }

template <bool BF16, int NT>
struct TreeWave {
  static constexpr int kQ = BF16 ? 4 : 8;   // 16-byte vectors of a query row in a lane
  static constexpr int kE = BF16 ? 8 : 4;   // keys of a step in a lane
  static constexpr int kKeys = BF16 ? 32 : 16;
  static constexpr uint32_t kRow = BF16 ? 256 : 512;
  pkv_u32x4 q[NT][kQ];
  // Weights are 2^(score - use): use is the largest score of some step, not of all.  It moves (and the sums with it) when a score is above
  // it by more than lim = 8, so that most steps neither look for the row's maximum across lanes nor touch the sums: exact all the same, as
  // a weight of 2^8 has the precision of one below 1.  lim = -inf: the row has seen nothing yet.
  float use[NT], lim[NT];
  pkv_f32x4 l[NT];     // sums: of rows 4j + i (bf16); of row n, this lane's keys, in the first element (fp32)
  pkv_f32x4 o[NT][8];  // o[m][i]: row 4j + i, dim tree_dim(n, m)
};

__device__ __forceinline__ pkv_f32x4 mfma_f32(float a, float b, pkv_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// Two numbers as bf16 in one instruction.
__device__ __forceinline__ uint32_t tree_pack(float lo, float hi) {
  const pkv_f32x2 v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, pkv_bf16x2));
}

// Key of the step that element e of lane (., j) belongs to.
__device__ __forceinline__ int tree_key(int e, int j) { return 16 * (e >> 2) + 4 * j + (e & 3); }

// Dim of column n of the m-th product with V, chosen so that rows of V are read whole: 16 bytes a lane, or (TURNED) as the transposing
// LDS read delivers them.
template <bool BF16, bool TURNED>
__device__ __forceinline__ int tree_dim(int n, int m) {
  return !BF16 ? 4 * n + (m & 3) + 64 * (m >> 2) : TURNED ? 16 * m + n : 8 * n + m;
}

// The scores of tile t.
template <bool BF16, int NT>
__device__ __forceinline__ void tree_scores(const TreeWave<BF16, NT> &w, const pkv_u32x4 (&k)[8], int t, float (&s)[TreeWave<BF16, NT>::kE]) {
  pkv_f32x4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = {0.f, 0.f, 0.f, 0.f};
  if constexpr (BF16) {
#pragma unroll
    for (int c = 0; c < 4; ++c) s0 = mfma_bf16(k[c], w.q[t][c], s0), s1 = mfma_bf16(k[4 + c], w.q[t][c], s1);
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = e < 4 ? s0[e & 3] : s1[e & 3];
  } else {
#pragma unroll
    for (int c = 0; c < 8; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) s0 = mfma_f32(__uint_as_float(k[c][i]), __uint_as_float(w.q[t][c][i]), s0);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = s0[e];
  }
}

// The larger of both halves each.
__device__ __forceinline__ uint32_t tree_max_u16(uint32_t a, uint32_t b) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}

// Scores into weights 2^(scale s - use) of the keys in `bits` (MASKED; else of all), as the operand of the second product; the sum and
// the base of the sums kept.
template <bool MASKED, bool BF16, int NT>
__device__ __forceinline__ pkv_u32x4 tree_weights(TreeWave<BF16, NT> &w, int t, const float (&s)[TreeWave<BF16, NT>::kE], uint32_t bits,
                                                  float scale_log2e) {
  constexpr int kE = TreeWave<BF16, NT>::kE;
  const int j = pkv_lane() >> 4;
  float p[kE], top = -INFINITY;
#pragma unroll
  for (int e = 0; e < kE; ++e) p[e] = fmaf(s[e], scale_log2e, -w.use[t]);
  if (MASKED) {
#pragma unroll
    for (int e = 0; e < kE; ++e) p[e] = (bits >> e) & 1u ? p[e] : -INFINITY;
  }
#pragma unroll
  for (int e = 0; e < kE; ++e) top = fmaxf(top, p[e]);
  if (__any(top > w.lim[t])) {
    // From here the scores as rounded numbers: the largest is the base itself, and its weight 1, however large they are.
    float x[kE];
    top = -INFINITY;
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      x[e] = att_scaled(s[e], scale_log2e);
      if (MASKED) x[e] = (bits >> e) & 1u ? x[e] : -INFINITY;
      top = fmaxf(top, x[e]);
    }
    top = pkv_pair_max<32>(pkv_pair_max<16>(top));
    const bool fresh = w.lim[t] < 0.f, moves = top > -INFINITY && (fresh || top > w.use[t]);
    const float next = moves ? top : w.use[t], corr = fresh ? 0.f : __builtin_amdgcn_exp2f(w.use[t] - next);
    w.use[t] = next, w.lim[t] = moves ? 8.f : w.lim[t];
    float cr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) cr[i] = __shfl(corr, 4 * j + i, PKV_WAVE);
#pragma unroll
    for (int m = 0; m < 8; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) w.o[t][m][i] *= cr[i];
    if constexpr (BF16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w.l[t][i] *= cr[i];
    } else {
      w.l[t][0] *= corr;
    }
#pragma unroll
    for (int e = 0; e < kE; ++e) p[e] = x[e] - next;
  }
#pragma unroll
  for (int e = 0; e < kE; ++e) p[e] = __builtin_amdgcn_exp2f(p[e]);
  if constexpr (BF16) {
    const pkv_u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
    const pkv_u32x4 a = {tree_pack(p[0], p[1]), tree_pack(p[2], p[3]), tree_pack(p[4], p[5]), tree_pack(p[6], p[7])};
    w.l[t] = mfma_bf16(a, ones, w.l[t]);
    return a;
  } else {
    w.l[t][0] += (p[0] + p[1]) + (p[2] + p[3]);
    return pkv_u32x4{__float_as_uint(p[0]), __float_as_uint(p[1]), __float_as_uint(p[2]), __float_as_uint(p[3])};
  }
}

// O += P V.  v_of(m): the operand of the m-th product, rows of V for the lane's keys: element e in half e % 2 of word e / 2 (bf16), or in word e.
template <bool BF16, int NT, typename Of>
__device__ __forceinline__ void tree_output(TreeWave<BF16, NT> &w, const pkv_u32x4 (&p)[NT], Of v_of) {
#pragma unroll
  for (int m = 0; m < 8; ++m) {
    const pkv_u32x4 v = v_of(m);
    if constexpr (BF16) {
#pragma unroll
      for (int t = 0; t < NT; ++t) w.o[t][m] = mfma_bf16(p[t], v, w.o[t][m]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int t = 0; t < NT; ++t) w.o[t][m] = mfma_f32(__uint_as_float(p[t][e]), __uint_as_float(v[e]), w.o[t][m]);
    }
  }
}

// The m-th operand out of rows of V as loaded, 16 bytes a key (bf16) or twice 16 (fp32).
template <bool BF16>
__device__ __forceinline__ pkv_u32x4 tree_turn(const pkv_u32x4 (&v)[8], int m) {
  pkv_u32x4 b;
  if constexpr (BF16) {
    const uint32_t sel = (m & 1) ? 0x07060302u : 0x05040100u;  // element m of each of the eight rows
#pragma unroll
    for (int d = 0; d < 4; ++d) b[d] = __builtin_amdgcn_perm(v[2 * d + 1][m >> 1], v[2 * d][m >> 1], sel);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = v[2 * e + (m >> 2)][m & 3];
  }
  return b;
}

// A step with keys that the rows do not all see: its first `here` keys are there; drafted ones (dv not null: the drafted V rows of this
// (b, h)), the tokens from u0 on, only for the rows whose token sees them.  v_of as in tree_output; weight: room of this wave's own.
template <bool BF16, bool TURNED, int NT, typename Of>
__device__ __forceinline__ void tree_masked_step(TreeWave<BF16, NT> &w, const TreeCall &a, int b, const char *dv, int u0, int here,
                                                 const int (&token)[NT], float (*weight)[33], const pkv_u32x4 (&k)[8], Of v_of) {
  using W = TreeWave<BF16, NT>;
  const int lane = pkv_lane(), n = lane & 15, j = lane >> 4;
  const bool draft = dv != nullptr;
  uint32_t there = 0, bits[NT];
#pragma unroll
  for (int e = 0; e < W::kE; ++e) there |= tree_key(e, j) < here ? 1u << e : 0u;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    bits[t] = there;
    if (draft && a.mask) {
      const uint8_t *const row = a.mask + (int64_t)b * a.mask_b + (int64_t)token[t] * a.mask_t + u0;
      uint32_t x = 0;
#pragma unroll
      for (int e = 0; e < W::kE; ++e) {
        const int key = tree_key(e, j);
        x |= (row[key < here ? key : here - 1] != 0 ? 1u : 0u) << e;
      }
      bits[t] &= x;
    } else if (draft) {
      uint32_t x = 0;
#pragma unroll
      for (int e = 0; e < W::kE; ++e) x |= (u0 + tree_key(e, j) <= token[t] ? 1u : 0u) << e;
      bits[t] &= x;
    }
  }
  pkv_u32x4 p[NT], keep;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    float s[W::kE];
    tree_scores(w, k, t, s);
    p[t] = tree_weights<true>(w, t, s, bits[t], a.scale_log2e);
  }
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    if constexpr (BF16) keep[d] = ((there >> (2 * d)) & 1u ? 0xffffu : 0u) | ((there >> (2 * d + 1)) & 1u ? 0xffff0000u : 0u);
    else keep[d] = (there >> d) & 1u ? 0xffffffffu : 0u;
  }
  // Keys that are not there were read again: zeros, so that nothing of them reaches the sums.  A drafted value that is not finite is for the
  // rows that see it and for no other, but in the product it would be 0 * inf for all: zero there, and added below.
  bool odd = false;
  if (draft) {
    uint32_t most = 0;
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      const pkv_u32x4 v = v_of(m);
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        if constexpr (BF16) most = tree_max_u16(most, v[d] & 0x7fff7fffu);
        else most = most > (v[d] & 0x7fffffffu) ? most : v[d] & 0x7fffffffu;
      }
    }
    odd = __any(BF16 ? (most & 0xffffu) >= 0x7f80u || most >= 0x7f800000u : most >= 0x7f800000u);
  }
  if (!odd) {
    tree_output(w, p, [&](int m) {
      pkv_u32x4 v = v_of(m);
#pragma unroll
      for (int d = 0; d < 4; ++d) v[d] &= keep[d];
      return v;
    });
    return;
  }
  tree_output(w, p, [&](int m) {
    pkv_u32x4 v = v_of(m);
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      uint32_t x = v[d] & keep[d], bad;
      if constexpr (BF16) bad = ((x & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((x & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
      else bad = (x & 0x7f800000u) == 0x7f800000u ? 0xffffffffu : 0u;
      v[d] = x & ~bad;
    }
    return v;
  });
  // the whole wave: one key at a time
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int e = 0; e < W::kE; ++e) {
      const uint32_t d = BF16 ? p[t][e >> 1] : p[t][e & 3];
      weight[n][tree_key(e, j)] = __uint_as_float(!BF16 ? d : e & 1 ? d & 0xffff0000u : d << 16);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    for (int key = 0; key < here; ++key) {
      const char *vp = dv + (int64_t)(u0 + key) * a.dv_t;
      float f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = weight[4 * j + i][key];
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        const int d = tree_dim<BF16, TURNED>(n, m);
        float x;
        if constexpr (BF16) x = pkv_bf16_bits_to_f32(((const uint16_t *)vp)[d]);
        else x = ((const float *)vp)[d];
#pragma unroll
        for (int i = 0; i < 4; ++i) w.o[t][m][i] += f[i] != 0.f && !(fabsf(x) < INFINITY) ? f[i] * x : 0.f;
      }
    }
  }
}

// The waves that took keys of the same rows meet, a tile of 16 rows at a time, and leave their result, or the split's part of it.
template <bool BF16, bool TURNED, int NT, int RW, int WAVES>
__device__ __forceinline__ void tree_finish(const TreeWave<BF16, NT> &w, const TreeCall &a, const TreePart &part, float (&s_m)[WAVES][16],
                                            float (&s_l)[WAVES][16], float (&s_o)[WAVES][16][132]) {
  constexpr int KW = WAVES / RW;
  const int tid = threadIdx.x, lane = pkv_lane(), wave = tid / PKV_WAVE, n = lane & 15, j = lane >> 4;
  const int bh = part.bh, rows = a.n_draft * a.group, b = (unsigned)bh / (unsigned)a.n_kv_heads, h = bh - b * a.n_kv_heads;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    __syncthreads();
    if (j == 0) s_m[wave][n] = w.lim[t] < 0.f ? -INFINITY : w.use[t];
    if constexpr (BF16) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n == 0) s_l[wave][4 * j + i] = w.l[t][i];
    } else {
      const float l = pkv_pair_add<32>(pkv_pair_add<16>(w.l[t][0]));
      if (j == 0) s_l[wave][n] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float *const row = s_o[wave][4 * j + i];
      if constexpr (BF16 && TURNED) {
#pragma unroll
        for (int m = 0; m < 8; ++m) row[tree_dim<BF16, TURNED>(n, m)] = w.o[t][m][i];
      } else {
        *(float4 *)(row + tree_dim<BF16, TURNED>(n, 0)) = float4{w.o[t][0][i], w.o[t][1][i], w.o[t][2][i], w.o[t][3][i]};
        *(float4 *)(row + tree_dim<BF16, TURNED>(n, 4)) = float4{w.o[t][4][i], w.o[t][5][i], w.o[t][6][i], w.o[t][7][i]};
      }
    }
    __syncthreads();
#pragma unroll
    for (int e0 = 0; e0 < RW * 16 * 32; e0 += WAVES * PKV_WAVE) {  // four dims at a time
      const int e = e0 + tid, rw = e >> 9, r = (e >> 5) & 15, d = 4 * (e & 31), row = (part.tile * RW + rw) * 16 * NT + 16 * t + r;
      if (row >= rows) continue;
      float mx = s_m[rw][r];
#pragma unroll
      for (int i = 1; i < KW; ++i) mx = fmaxf(mx, s_m[rw + i * RW][r]);
      const float base = mx == -INFINITY ? 0.f : mx;
      float ls = 0.f;
      pkv_f32x4 os = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KW; ++i) {
        const float c = __builtin_amdgcn_exp2f(s_m[rw + i * RW][r] - base);
        const pkv_f32x4 x = *(const pkv_f32x4 *)&s_o[rw + i * RW][r][d];
        ls = fmaf(s_l[rw + i * RW][r], c, ls);
#pragma unroll
        for (int u = 0; u < 4; ++u) os[u] = fmaf(x[u], c, os[u]);
      }
      if (a.n_splits == 1) {
        const int u = (unsigned)row / (unsigned)a.group;
        const int64_t to = (((int64_t)b * a.n_draft + u) * a.n_kv_heads * a.group + h * a.group + (row - u * a.group)) * 128 + d;
        const float share = ls == 0.f ? 0.f : 1.0f / ls;  // 0: nothing seen
#pragma unroll
        for (int i = 0; i < 4; ++i) os[i] *= share;
        if constexpr (BF16) *(pkv_u32x2 *)((uint16_t *)a.out + to) = pkv_u32x2{tree_pack(os[0], os[1]), tree_pack(os[2], os[3])};
        else *(pkv_f32x4 *)((float *)a.out + to) = os;
      } else {
        const int64_t at = ((int64_t)part.first + part.split) * rows + row;
        *(pkv_f32x4 *)(a.ws_o + at * 128 + d) = os;
        if (d == 0) *(float2 *)(a.ws_ml + at * 2) = float2{mx, ls};
      }
    }
  }
}

// Query rows r0 .. of this wave (those past the last repeat it and are not stored), and sums of nothing.
template <bool BF16, int NT>
__device__ __forceinline__ void tree_begin(TreeWave<BF16, NT> &w, const TreeCall &a, int b, int h, int r0, int (&token)[NT]) {
  const int lane = pkv_lane(), n = lane & 15, j = lane >> 4, rows = a.n_draft * a.group;
  constexpr int es = BF16 ? 2 : 4;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = r0 + 16 * t + n, rr = r < rows ? r : rows - 1;
    token[t] = (unsigned)rr / (unsigned)a.group;
    const char *qp = (const char *)a.q + ((int64_t)b * a.q_stride_b + (int64_t)token[t] * a.q_stride_t +
                                          (int64_t)(h * a.group + rr - token[t] * a.group) * 128) * es + 16 * j;
#pragma unroll
    for (int c = 0; c < TreeWave<BF16, NT>::kQ; ++c) w.q[t][c] = *(const pkv_u32x4 *)(qp + 64 * c);
    w.use[t] = 0.f, w.lim[t] = -INFINITY, w.l[t] = pkv_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int m = 0; m < 8; ++m) w.o[t][m] = pkv_f32x4{0.f, 0.f, 0.f, 0.f};
  }
}

// Cached keys of row bh.
__device__ __forceinline__ uint32_t tree_total(const TreeCall &a, int bh) {
  if (!a.row_keys) return a.total;
  const int rk = a.row_keys[bh];
  return rk <= 0 ? 0u : (uint32_t)rk < a.total ? (uint32_t)rk : a.total;
}

typedef const __attribute__((address_space(1))) char *tree_global;
__device__ __forceinline__ pkv_u32x4 tree_read(const char *p) { return *(const pkv_u32x4 *)p; }
__device__ __forceinline__ pkv_u32x4 tree_read(tree_global p) { return *(const __attribute__((address_space(1))) pkv_u32x4 *)p; }

// Places of cached keys of one (b, h), found in two steps: find() asks for the row's number where the keys are selected, place() waits for it.  (In
// one, with a branch round the load, every search waited for all rows under way: 8 x 8 x 1617 selected keys, 256 rows 46 us, dense ones 37.)
// Fields of segments are held in registers and added up: a field picked by a lane would be loaded from memory, and the wait for it would be for
// all keys under way too.
//
// Segments in any tensors: of each the addresses that key 0 would have if the segment were all there is.  Such addresses are plain numbers to
// the compiler, which reads them with instructions that may go to LDS and are waited for with it, unless told that they are global.
// us, two tensors, like this / with every field picked on its own and unmarked addresses: 2 x 8 x 20000 keys, 32 rows 40 / 68, fp32 81 / 148.
template <bool BF16, bool INDEXED, typename SEGS>
struct TreePlaces {
  static constexpr uint32_t kRow = BF16 ? 256 : 512;
  static_assert(PKV_ATTN_MAX_SEGMENTS == 4, "segments one by one");
  uint32_t end0, end1, end2;
  uint64_t k0, k1, k2, k3, v0, v1, v2, v3, i0, i1, i2, i3;  // differences from the one before, after the first
  uint32_t l0, l1, l2, l3;
  struct Found {
    uint32_t at, limit;  // limit: rows of a selected key's segment, 0 where it is not selected
    int64_t x;
  };
  static __device__ __forceinline__ uint32_t end_of(const SEGS &s, int t) { return t < s.n ? (uint32_t)att_field(s.end[t]) : 0xffffffffu; }
  static __device__ __forceinline__ void field(const SEGS &s, int t, int bh, int b, int h, uint64_t &k, uint64_t &v, uint64_t &i, uint32_t &l) {
    const int64_t first = t > 0 ? att_field(s.end[t > 0 ? t - 1 : 0]) : 0;
    const uint64_t ip = (uint64_t)att_field(s.idx[t]);
    const bool selected = INDEXED && ip != 0;
    const int64_t row0 = att_field(s.row0[t]) - (selected ? 0 : first);
    const int64_t off = ((int64_t)b * att_field(s.stride_b[t]) + (int64_t)h * att_field(s.stride_h[t])) * (kRow / 128) + row0 * kRow;
    k = (uint64_t)att_field(s.k[t]) + off, v = (uint64_t)att_field(s.v[t]) + off;
    i = selected ? ip + ((int64_t)bh * att_field(s.idx_stride[t]) - first) * 8 : 0;
    l = selected ? (uint32_t)att_field(s.idx_limit[t]) : 0;
  }
  __device__ __forceinline__ TreePlaces(const SEGS &s, int bh, int b, int h) {
    end0 = end_of(s, 0), end1 = end_of(s, 1), end2 = end_of(s, 2);
    field(s, 0, bh, b, h, k0, v0, i0, l0);
    field(s, 1, bh, b, h, k1, v1, i1, l1);
    field(s, 2, bh, b, h, k2, v2, i2, l2);
    field(s, 3, bh, b, h, k3, v3, i3, l3);
    k3 -= k2, v3 -= v2, i3 -= i2, l3 -= l2;
    k2 -= k1, v2 -= v1, i2 -= i1, l2 -= l1;
    k1 -= k0, v1 -= v0, i1 -= i0, l1 -= l0;
  }
  template <typename T>
  __device__ __forceinline__ T pick(uint32_t at, T a, T b, T c, T d) const {
    return a + (at >= end0 ? b : 0) + (at >= end1 ? c : 0) + (at >= end2 ? d : 0);
  }
  __device__ __forceinline__ Found find(uint32_t at) const {
    Found f = {at, 0u, 0};
    if constexpr (INDEXED) {
      f.limit = pick(at, l0, l1, l2, l3);
      if (f.limit) f.x = *(const __attribute__((address_space(1))) int64_t *)(pick(at, i0, i1, i2, i3) + (uint64_t)at * 8);
    }
    return f;
  }
  __device__ __forceinline__ AttPlace<false> place(const Found &f) const {
    uint32_t r = f.at;
    if constexpr (INDEXED) r = f.limit ? (uint32_t)(f.x < 0 ? 0 : (f.x >= (int64_t)f.limit ? f.limit - 1 : f.x)) : r;
    const uint64_t off = (uint64_t)r * kRow;
    return {pick(f.at, k0, k1, k2, k3) + off, pick(f.at, v0, v1, v2, v3) + off};
  }
};
// Segments in one tensor: byte offsets in it.
template <bool BF16, bool INDEXED>
struct TreePlaces<BF16, INDEXED, AttOne> {
  static constexpr uint32_t kRow = BF16 ? 256 : 512;
  static_assert(PKV_ATTN_MAX_SEGMENTS == 4, "segments one by one");
  const char *k, *v;
  uint32_t end0, end1, end2;
  uint32_t delta0, more1, more2, more3;
  const int64_t *idx;
  int64_t limit;
  uint32_t lo, hi, row0;
  __device__ __forceinline__ TreePlaces(const AttOne &s, int bh, int b, int h) {
    const int64_t slab = (int64_t)b * s.stride_b + (int64_t)h * s.stride_h;
    k = s.k + slab, v = s.v + slab;
    end0 = att_field(s.end[0]), end1 = att_field(s.end[1]), end2 = att_field(s.end[2]);
    const uint32_t d0 = (uint32_t)att_field(s.delta[0]), d1 = (uint32_t)att_field(s.delta[1]), d2 = (uint32_t)att_field(s.delta[2]);
    delta0 = d0, more1 = d1 - d0, more2 = d2 - d1, more3 = (uint32_t)att_field(s.delta[3]) - d2;
    if (INDEXED) idx = s.idx + (int64_t)bh * s.idx_stride, limit = s.idx_limit, lo = s.idx_lo, hi = s.idx_hi, row0 = s.idx_row0;
  }
  struct Found {
    uint32_t off;  // of a row that is not selected, else kSelected
    int64_t x;
  };
  static constexpr uint32_t kSelected = 0xffffffffu;
  __device__ __forceinline__ Found find(uint32_t at) const {
    Found f;
    f.off = (at + delta0 + (at >= end0 ? more1 : 0u) + (at >= end1 ? more2 : 0u) + (at >= end2 ? more3 : 0u)) * kRow;
    if constexpr (INDEXED) {
      const bool in = at >= lo && at < hi;
      f.x = idx[in ? at - lo : 0u];
      f.off = in ? kSelected : f.off;
    }
    return f;
  }
  __device__ __forceinline__ AttPlace<true> place(const Found &f) const {
    if constexpr (INDEXED) {
      const uint32_t r = row0 + (uint32_t)(f.x < 0 ? 0 : (f.x >= limit ? limit - 1 : f.x));
      return {f.off == kSelected ? r * kRow : f.off};
    }
    return {f.off};
  }
};

// Lane `key`'s place, key = a constant plus what the lane adds: the constant goes into the instruction.
__device__ __forceinline__ AttPlace<true> tree_from(const AttPlace<true> &p, int base4, int key) {
  return {(uint32_t)__builtin_amdgcn_ds_bpermute(base4 + 4 * key, (int)p.off)};
}

// at(what the lane adds, constant part): address of that key's row.
template <bool BF16, typename At>
__device__ __forceinline__ void tree_load_k(pkv_u32x4 (&k)[8], At at) {
  const int lane = pkv_lane(), n = lane & 15, j = lane >> 4;
  constexpr int kTiles = BF16 ? 2 : 1, kVecs = BF16 ? 4 : 8;
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    const auto kp = at(n, 16 * t);
#pragma unroll
    for (int c = 0; c < kVecs; ++c) k[kVecs * t + c] = tree_read(kp + 64 * c + 16 * j);
  }
}
template <bool BF16, typename At>
__device__ __forceinline__ void tree_load_v(pkv_u32x4 (&v)[8], At at) {
  const int lane = pkv_lane(), n = lane & 15, j = lane >> 4;
  constexpr int kE = BF16 ? 8 : 4, kVecs = BF16 ? 1 : 2;
#pragma unroll
  for (int e = 0; e < kE; ++e) {
    const auto vp = at(4 * j, tree_key(e, 0));
#pragma unroll
    for (int c = 0; c < kVecs; ++c) v[kVecs * e + c] = tree_read(vp + 16 * n + 256 * c);
  }
}

// Workgroups of a launch: one to a compute unit (kTreeWorkgroups).  us, 128 / 256 / 512 / 1024 workgroups: 4 x 8 heads x 65536 keys, 16 rows
// a head 226 / 191 / 195 / 212, 64 rows 260 / 178 / 189 / 222; 1 x 8 x 32768, 32 rows 39.5 / 35.4 / 46.2 / 46.3; 3 x 4 x 9001 fp32, 49 rows 78 / 50 / 59 / 67.
//
// Up to 16 query rows.  The four waves of a workgroup take steps of keys in turns, straight from memory into the operands' registers.
// Full steps go round the waves of all splits, so that what the chip reads at one time lies side by side; the steps that not all rows see in
// full, the cached keys behind the last full step and the drafted tokens, are dealt out behind them.
template <bool BF16, bool INDEXED, typename SEGS, bool SHARES>
__global__ __launch_bounds__(kTreeWaves * PKV_WAVE, 2) void pkv_tree_partial_kernel(TreeCall a, SEGS segs) {
  using W = TreeWave<BF16, 1>;
  constexpr bool ONE = __is_same(SEGS, AttOne);
  const TreePart part = tree_part<SHARES>(a);
  if (!part.any) return;  // the whole workgroup
  const int split = part.split, n_splits = part.n_splits, bh = part.bh;
  const int b = (unsigned)bh / (unsigned)a.n_kv_heads, h = bh - b * a.n_kv_heads;
  const int lane = pkv_lane(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / PKV_WAVE);

  const uint32_t total = tree_total(a, bh);
  const int turns = kTreeWaves * n_splits, turn0 = split * kTreeWaves + wave;
  const int all_full = (int)(total / W::kKeys), rest = (int)(total % W::kKeys);
  const int n_full = turn0 < all_full ? (all_full - 1 - turn0) / turns + 1 : 0;

  // Where the keys of a step lie: lane l knows key l's place.  Found two steps ahead, since a selected row's number is read from memory.
  const TreePlaces<BF16, INDEXED, SEGS> places(segs, bh, b, h);
  auto find = [&](int first, int keys) {
    const int key = lane & (W::kKeys - 1);
    return places.find((uint32_t)(first + (key < keys ? key : keys - 1)));
  };
  auto k_at = [&](const AttPlace<ONE> &place) {
    return [&](int base, int key) {
      if constexpr (ONE) return places.k + (uint64_t)tree_from(place, 4 * base, key).off;
      else return (tree_global)place.pull(place.k, base + key);
    };
  };
  auto v_at = [&](const AttPlace<ONE> &place) {
    return [&](int base, int key) {
      if constexpr (ONE) return places.v + (uint64_t)tree_from(place, 4 * base, key).off;
      else return (tree_global)place.pull(place.v, base + key);
    };
  };

  W w;
  pkv_u32x4 k[8], v[8];
  int token[1];
  tree_begin<BF16, 1>(w, a, b, h, 0, token);
  // In the order of the loop, so that a wait there is for what it needs alone: K, the place of the next step, V.
  AttPlace<ONE> mine;
  typename TreePlaces<BF16, INDEXED, SEGS>::Found next;
  if (n_full > 0) {
    mine = places.place(find(turn0 * W::kKeys, W::kKeys));
    tree_load_k<BF16>(k, k_at(mine));
    next = find((n_full > 1 ? turn0 + turns : turn0) * W::kKeys, W::kKeys);
    tree_load_v<BF16>(v, v_at(mine));
  }
  // Keys and values of the next step are requested where the registers of this one's are free again.
  for (int i = 0; i < n_full; ++i) {
    float s[W::kE];
    tree_scores(w, k, 0, s);
    mine = places.place(next);
    if (i + 1 < n_full) tree_load_k<BF16>(k, k_at(mine));
    if (i + 2 < n_full) next = find((turn0 + (i + 2) * turns) * W::kKeys, W::kKeys);
    const pkv_u32x4 p[1] = {tree_weights<false>(w, 0, s, 0u, a.scale_log2e)};
    tree_output(w, p, [&](int m) { return tree_turn<BF16>(v, m); });
    if (i + 1 < n_full) tree_load_v<BF16>(v, v_at(mine));
  }

  __shared__ float s_m[kTreeWaves][16], s_l[kTreeWaves][16];
  __shared__ alignas(16) float s_o[kTreeWaves][16][128 + 4];
  const char *const dk = a.dk + (int64_t)b * a.dk_b + (int64_t)h * a.dk_h, *const dv = a.dv + (int64_t)b * a.dv_b + (int64_t)h * a.dv_h;
  const int n_tail = rest > 0 ? 1 : 0, n_more = n_tail + (a.n_draft - 1) / W::kKeys + 1;
  for (int i = (turn0 - all_full % turns + turns) % turns; i < n_more; i += turns) {
    const bool draft = i >= n_tail;
    const int u0 = (i - n_tail) * W::kKeys, left = draft ? a.n_draft - u0 : rest, here = left < W::kKeys ? left : W::kKeys;
    if (draft) {
      tree_load_k<BF16>(k, [&](int base, int key) { return dk + (int64_t)(u0 + (base + key < here ? base + key : here - 1)) * a.dk_t; });
      tree_load_v<BF16>(v, [&](int base, int key) { return dv + (int64_t)(u0 + (base + key < here ? base + key : here - 1)) * a.dv_t; });
    } else {
      mine = places.place(find(all_full * W::kKeys, rest));
      tree_load_k<BF16>(k, k_at(mine));
      tree_load_v<BF16>(v, v_at(mine));
    }
    tree_masked_step<BF16, false, 1>(w, a, b, draft ? dv : nullptr, u0, here, token, (float(*)[33]) & s_o[wave][0][0], k,
                                     [&](int m) { return tree_turn<BF16>(v, m); });
  }
  tree_finish<BF16, false, 1, 1, kTreeWaves>(w, a, part, s_m, s_l, s_o);
}

// Registers: 256 a lane, for two waves a SIMD.  What does not fit into them (bytes of scratch a lane; without / with key counts of the rows): bf16
// above, selected rows 8 / 8, in several tensors 20 / 20; below, 17 to 32 query rows with selected ones in several tensors 72 / 24 (fp32 108 / 24); two
// row tiles a wave 36 / 36, several tensors 96 / 24, selected rows in them 244 / 100: two turns of rows under way and the sums of two tiles are more
// than there is room for.  The other forms spill nothing.
typedef short tree_s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) tree_s16x4 tree_lds_s16x4;

// More than 16 query rows: the waves of a workgroup share the keys, which go through LDS once for all of them.
// RW of the eight waves take 16 NT rows each; the 8 / RW groups of such waves take neighbouring steps of keys, a turn of them at a time.  Rows of K and V
// are requested two turns ahead into registers, written to one of two LDS buffers a turn ahead, and read from there as operands; one
// barrier a turn.  us, straight from memory with each wave's own loads (two tiles a wave) / through LDS: 4 x 8 x 65536 keys, 64 rows 240 / 170;
// 8 x 8 x 1617 selected keys, 256 rows 54 / 46.  A 16-byte vector c of a row r lies at c ^ (r mod 16), so that the 16 rows of an operand of K are on different banks.
template <bool BF16, int NT, int RW, bool INDEXED, typename SEGS, bool SHARES>
__global__ __launch_bounds__(kWideWaves * PKV_WAVE, 2) void pkv_tree_wide_kernel(TreeCall a, SEGS segs) {
  using W = TreeWave<BF16, NT>;
  constexpr bool ONE = __is_same(SEGS, AttOne);
  constexpr int KW = kWideWaves / RW, kTurnKeys = KW * W::kKeys, kRow = W::kRow, kVecs = kRow / 16;
  constexpr int kRowsAt = kWideWaves * PKV_WAVE / kVecs, kLoads = kTurnKeys / kRowsAt;  // rows a load of the workgroup covers; loads a turn
  constexpr int kTensor = kTurnKeys * kRow;
  const TreePart part = tree_part<SHARES>(a);
  if (!part.any) return;  // the whole workgroup
  const int split = part.split, n_splits = part.n_splits, bh = part.bh;
  const int b = (unsigned)bh / (unsigned)a.n_kv_heads, h = bh - b * a.n_kv_heads;
  const int tid = threadIdx.x, lane = pkv_lane(), wave = __builtin_amdgcn_readfirstlane(tid / PKV_WAVE), n = lane & 15, j = lane >> 4;
  const int row_wave = wave % RW, key_wave = wave / RW, r0 = (part.tile * RW + row_wave) * 16 * NT;
  constexpr int kEnd = kWideWaves * (16 * 132 + 32) * 4, kLds = 4 * kTensor > kEnd ? 4 * kTensor : kEnd;
  static_assert(2 * kTensor + kWideWaves * 16 * 33 * 4 <= kLds, "room for the weights of drafted tokens behind a turn");
  __shared__ alignas(16) char lds[kLds];

  const uint32_t total = tree_total(a, bh);
  const int all_full = (int)(total / kTurnKeys), rest = (int)(total % kTurnKeys);
  const int n_mine = split < all_full ? (all_full - 1 - split) / n_splits + 1 : 0, n_full = n_mine > 1 ? n_mine : 0;  // a single turn: not piped
  const TreePlaces<BF16, INDEXED, SEGS> places(segs, bh, b, h);
  const char *const dk = a.dk + (int64_t)b * a.dk_b + (int64_t)h * a.dk_h, *const dv = a.dv + (int64_t)b * a.dv_b + (int64_t)h * a.dv_h;

  // What this thread brings in: vector my_vec of rows my_row + kRowsAt u.
  const int my_row = tid / kVecs, my_vec = tid % kVecs;
  struct Rows {
    pkv_u32x4 k[kLoads], v[kLoads];
  };
  using Found = typename TreePlaces<BF16, INDEXED, SEGS>::Found;
  auto find = [&](int first, int count, Found (&at)[kLoads]) {
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int r = my_row + kRowsAt * u;
      at[u] = places.find((uint32_t)(first + (r < count ? r : count - 1)));
    }
  };
  auto fetch = [&](const Found (&found)[kLoads], Rows &r) {
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const AttPlace<ONE> at = places.place(found[u]);
      if constexpr (ONE) {
        r.k[u] = __builtin_nontemporal_load((const pkv_u32x4 *)(places.k + (uint64_t)at.off) + my_vec);
        r.v[u] = __builtin_nontemporal_load((const pkv_u32x4 *)(places.v + (uint64_t)at.off) + my_vec);
      } else {
        r.k[u] = __builtin_nontemporal_load((const __attribute__((address_space(1))) pkv_u32x4 *)at.k + my_vec);
        r.v[u] = __builtin_nontemporal_load((const __attribute__((address_space(1))) pkv_u32x4 *)at.v + my_vec);
      }
    }
  };
  auto put = [&](const Rows &r, int buffer) {
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int row = my_row + kRowsAt * u, at = buffer * 2 * kTensor + row * kRow + 16 * (my_vec ^ (row & 15));
      *(pkv_u32x4 *)(lds + at) = r.k[u];
      *(pkv_u32x4 *)(lds + at + kTensor) = r.v[u];
    }
  };
  W w;
  pkv_u32x4 k[8];
  auto get_k = [&](int buffer) {
    constexpr int kTiles = BF16 ? 2 : 1, kC = BF16 ? 4 : 8;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int c = 0; c < kC; ++c)
        k[kC * t + c] = *(const pkv_u32x4 *)(lds + buffer * 2 * kTensor + (key_wave * W::kKeys + 16 * t + n) * kRow + 16 * ((4 * c + j) ^ n));
  };
  // bf16: a transposing read takes four rows times 16 dims with 16 lanes, eight bytes of a row each, and gives a lane one dim of the four.
  auto v_of = [&](int buffer) {
    return [&, buffer](int m) {
      const char *const rows = lds + buffer * 2 * kTensor + kTensor + key_wave * W::kKeys * kRow;
      pkv_u32x4 x;
      if constexpr (BF16) {
        const int r = 4 * j + (n >> 2), at = r * (int)kRow + 16 * ((2 * m + ((n >> 1) & 1)) ^ r) + 8 * (n & 1);
        const tree_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tree_lds_s16x4 *)(rows + at));
        const tree_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tree_lds_s16x4 *)(rows + at + 16 * kRow));
        const pkv_u32x2 a2 = __builtin_bit_cast(pkv_u32x2, lo), b2 = __builtin_bit_cast(pkv_u32x2, hi);
        x = pkv_u32x4{a2.x, a2.y, b2.x, b2.y};
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = tree_key(e, j);
          x[e] = *(const uint32_t *)(rows + r * kRow + 16 * ((16 * (m >> 2) + n) ^ r) + 4 * (m & 3));
        }
      }
      return x;
    };
  };

  int token[NT];
  tree_begin<BF16, NT>(w, a, b, h, r0, token);
  Found places_of[2][kLoads];
  Rows ahead[2];
  auto first_of = [&](int i) { return (split + (i < n_full ? i : n_full - 1) * n_splits) * kTurnKeys; };  // past the last: read again, never used
  if (n_full > 0) {
    Found first[2][kLoads];
    find(first_of(0), kTurnKeys, first[0]);
    find(first_of(1), kTurnKeys, first[1]);
    find(first_of(2), kTurnKeys, places_of[1]);
    find(first_of(3), kTurnKeys, places_of[0]);
    fetch(first[0], ahead[0]);
    fetch(first[1], ahead[1]);
    put(ahead[0], 0);
    fetch(places_of[1], ahead[0]);
  }
  // Turn i is in LDS or on its way there, turn i + 1 in registers, turn i + 2 requested, the places of turn i + 3 known.  Places are asked
  // for before rows: a wait for them is then not for the rows as well.
  auto turn = [&](int i, Rows &after, const Found (&third)[kLoads], Found (&fourth)[kLoads]) {
    __syncthreads();  // turn i is there, and everybody is done with turn i - 1
    put(after, (i + 1) & 1);
    find(first_of(i + 4), kTurnKeys, fourth);
    fetch(third, after);
    if (i >= n_full) return;  // the whole workgroup
    float s[NT][W::kE];
    get_k(i & 1);
#pragma unroll
    for (int t = 0; t < NT; ++t) tree_scores(w, k, t, s[t]);
    pkv_u32x4 p[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) p[t] = tree_weights<false>(w, t, s[t], 0u, a.scale_log2e);
    tree_output(w, p, v_of(i & 1));
  };
  for (int i = 0; i < n_full; i += 2) {  // no way round the second: waits count what was asked for since on every path
    turn(i, ahead[1], places_of[0], places_of[1]);
    turn(i + 1, ahead[0], places_of[1], places_of[0]);
  }

  // The cached keys behind the last full turn, and the drafted tokens, a turn of them at a time, dealt out behind the full ones.
  const int n_tail = rest > 0 ? 1 : 0, n_more = n_tail + (a.n_draft - 1) / kTurnKeys + 1;
  for (int i = n_mine > n_full ? -1 : 0, turn0 = (split - all_full % n_splits + n_splits) % n_splits; i < 0 || turn0 < n_more; ++i) {
    const bool whole = i < 0, draft = !whole && turn0 >= n_tail;
    const int first = whole ? split * kTurnKeys : draft ? (turn0 - n_tail) * kTurnKeys : all_full * kTurnKeys, left = (draft ? a.n_draft : (int)total) - first;
    const int count = left < kTurnKeys ? left : kTurnKeys;
    if (draft) {
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        const int r = my_row + kRowsAt * u, at = first + (r < count ? r : count - 1);
        ahead[0].k[u] = ((const pkv_u32x4 *)(dk + (int64_t)at * a.dk_t))[my_vec];
        ahead[0].v[u] = ((const pkv_u32x4 *)(dv + (int64_t)at * a.dv_t))[my_vec];
      }
    } else {
      find(first, count, places_of[0]);
      fetch(places_of[0], ahead[0]);
    }
    __syncthreads();
    put(ahead[0], 0);
    __syncthreads();
    const int here = count - key_wave * W::kKeys < W::kKeys ? count - key_wave * W::kKeys : W::kKeys;
    if (here > 0) {
      get_k(0);
      tree_masked_step<BF16, true, NT>(w, a, b, draft ? dv : nullptr, first + key_wave * W::kKeys, here, token,
                                       (float(*)[33])(lds + 2 * kTensor + wave * 2112), k, v_of(0));
    }
    if (!whole) turn0 += n_splits;
  }
  tree_finish<BF16, true, NT, RW, kWideWaves>(w, a, part, *(float(*)[kWideWaves][16])lds, *(float(*)[kWideWaves][16])(lds + kWideWaves * 64),
                                        *(float(*)[kWideWaves][16][132])(lds + kWideWaves * 128));
}

// One wave a query row: lane l weighs split l and holds dims 2 l, 2 l + 1 of the output.
template <bool BF16>
__global__ __launch_bounds__(256) void pkv_tree_merge_kernel(const float *__restrict__ ws_o, const float *__restrict__ ws_ml, void *__restrict__ out,
                                                             const int32_t *__restrict__ row_keys, int n_splits, uint32_t rows, uint32_t n_rows,
                                                             uint32_t n_draft, uint32_t group, uint32_t n_kv_heads, int by_keys, uint32_t total,
                                                             int n_bh, int slots) {
  const uint32_t at = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + threadIdx.x / PKV_WAVE);  // below 2^30: 65535 * 8192 rows
  const int lane = pkv_lane();
  if (at >= n_rows) return;
  const uint32_t bh = at / rows, row = at - bh * rows;
  int first_split = bh * n_splits;
  if (by_keys) {
    const TreeShare t = tree_share(row_keys, total, n_bh, slots, by_keys);
    n_splits = __builtin_amdgcn_readlane(t.n, bh), first_split = __builtin_amdgcn_readlane(t.first, bh);
  }
  const int64_t first = (int64_t)first_split * rows + row;
  float m = -INFINITY, l = 0.f;
  if (lane < n_splits) m = ws_ml[(first + (int64_t)lane * rows) * 2], l = ws_ml[(first + (int64_t)lane * rows) * 2 + 1];
  const float mx = pkv_wave_max(m), base = mx == -INFINITY ? 0.f : mx;
  const float c = __builtin_amdgcn_exp2f(m - base), all = pkv_wave_sum(l * c);
  const float weight = all == 0.f ? 0.f : c / all;
  float x = 0.f, y = 0.f;
  const float *const parts = ws_o + first * 128;
  for (int s = 0; s < n_splits; s += 16) {
    float2 o[16];
#pragma unroll
    for (int i = 0; i < 16; ++i)  // past the last split: the last again, as zeros
      o[i] = *(const float2 *)(parts + (int64_t)(s + i < n_splits ? s + i : n_splits - 1) * rows * 128 + 2 * lane);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(weight), s + i));
      const bool in = s + i < n_splits;
      x = fmaf(in ? o[i].x : 0.f, f, x), y = fmaf(in ? o[i].y : 0.f, f, y);
    }
  }
  const uint32_t b = bh / n_kv_heads, h = bh - b * n_kv_heads, u = row / group;
  const int64_t to = (((int64_t)b * n_draft + u) * n_kv_heads * group + h * group + (row - u * group)) * 128 + 2 * lane;
  if constexpr (BF16) *(uint32_t *)((uint16_t *)out + to) = tree_pack(x, y);
  else *(float2 *)((float *)out + to) = float2{x, y};
}

struct TreePlan {
  int nt, rw, row_tiles, n_splits, turn;
};

TreePlan tree_plan(int dtype, int bs, int n_kv_heads, int rows, int64_t total) {
  TreePlan p;
  const bool bf = dtype == PKV_DTYPE_BF16;
  p.rw = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  const int64_t bh = (int64_t)bs * n_kv_heads;
  auto split = [&](int nt) {
    p.nt = nt;
    const int per_wg = 16 * nt * p.rw;
    p.turn = (p.rw == 1 ? kTreeWaves : kWideWaves / p.rw) * (bf ? 32 : 16);  // keys a workgroup takes at a time
    p.row_tiles = (rows + per_wg - 1) / per_wg;
    int64_t s = kTreeWorkgroups / (bh * p.row_tiles), most = (total + p.turn - 1) / p.turn;
    if (s > most) s = most;
    if (s > kTreeMaxSplits) s = kTreeMaxSplits;
    // Few keys: no join, which is a launch (2.5 us of the host's time), rather than workgroups side by side.  us on the GPU, two launches / one, 8 KV heads:
    // 180 keys, 12 rows 8.3 / 6.7, 160 rows 13.2 / 11.4; 380 keys, 12 rows 9.5 / 8.8, 20 rows 11.3 / 12.0; fp32, 120 keys, 12 rows 10.9 / 9.2, 160 rows 16.1 / 22.5.
    if (total <= (bf ? 384 : p.rw == 1 ? 192 : 0)) s = 1;
    p.n_splits = (int)(s < 1 ? 1 : s);
  };
  // Two row tiles a wave read K and V from LDS once for both, but leave half the workgroups, which costs more where their share of keys is short:
  // us, one / two: 8 x 8 x 1617 keys, 256 rows 38 / 50; 1 x 8 x 4096, 512 rows 30 / 35; 2 x 8 x 16384, 128 rows 44 / 42; 1 x 8 x 32768, 256 rows
  // (two always) 62 to 65.  Measured as they are built: the kernel of two tiles spills.  fp32 has no registers for two.
  split(1);
  if (bf && rows > 64) {
    split(2);
    if (total / p.n_splits < 1024) split(1);
  }
  return p;
}

size_t tree_ws_floats(const TreePlan &p, int64_t n_rows) { return p.n_splits == 1 ? 0 : (size_t)n_rows * p.n_splits * 130; }

bool tree_shape_ok(int bs, int n_kv_heads, int group, int n_draft) {
  return bs > 0 && n_kv_heads > 0 && (int64_t)bs * n_kv_heads <= 65535 && group > 0 && n_draft > 0 && n_draft <= 1024 &&
         (int64_t)n_draft * group <= 8192;
}

}  // namespace

extern "C" size_t pkv_tree_attention_ws_bytes(int dtype, int bs, int n_kv_heads, int group, int n_draft, int64_t total_keys) {
  if (!tree_shape_ok(bs, n_kv_heads, group, n_draft) || total_keys < 0) return 0;
  return tree_ws_floats(tree_plan(dtype, bs, n_kv_heads, n_draft * group, total_keys), (int64_t)bs * n_kv_heads * n_draft * group) * 4;
}

extern "C" int pkv_tree_attention(const pkv_tree_args *a, void *stream) {
  PKV_REQUIRE(a != nullptr && a->q && a->out && a->draft_k && a->draft_v, "pkv_tree_attention: null pointer");
  PKV_REQUIRE(a->dtype == PKV_DTYPE_F32 || a->dtype == PKV_DTYPE_BF16, "unknown dtype %d", a->dtype);
  PKV_REQUIRE(tree_shape_ok(a->bs, a->n_kv_heads, a->group, a->n_draft),
              "pkv_tree_attention: bad shape bs=%d kv_heads=%d group=%d drafted=%d (at most 1024 drafted tokens, 8192 query rows a KV head)",
              a->bs, a->n_kv_heads, a->group, a->n_draft);
  PKV_REQUIRE(a->n_segments >= 0 && a->n_segments <= PKV_ATTN_MAX_SEGMENTS, "0..%d key segments", PKV_ATTN_MAX_SEGMENTS);
  const bool bf = a->dtype == PKV_DTYPE_BF16;
  const int64_t es = bf ? 2 : 4, vec = 16 / es;
  PKV_REQUIRE(pkv_aligned(a->q, 16) && pkv_aligned(a->out, 16) && pkv_aligned(a->draft_k, 16) && pkv_aligned(a->draft_v, 16),
              "pkv_tree_attention: 16-byte aligned buffers required");
  const int64_t strides[] = {a->q_stride_b, a->q_stride_t, a->dk_stride_b, a->dk_stride_h, a->dk_stride_t,
                             a->dv_stride_b, a->dv_stride_h, a->dv_stride_t};
  for (int64_t x : strides) PKV_REQUIRE(x % vec == 0 && x >= 0, "pkv_tree_attention: strides must be multiples of 16 bytes");
  PKV_REQUIRE((a->n_draft - 1) * a->dk_stride_t * es < ((int64_t)1 << 32) && (a->n_draft - 1) * a->dv_stride_t * es < ((int64_t)1 << 32),
              "pkv_tree_attention: a sequence's drafted rows must lie within 4 GiB");
  PKV_REQUIRE(!a->mask || (a->mask_stride_b >= 0 && a->mask_stride_t >= 0), "pkv_tree_attention: bad mask strides");
  PKV_REQUIRE(!a->row_keys || pkv_aligned(a->row_keys, 4), "pkv_tree_attention: row_keys must be int32");
  AttSegs sg;
  int64_t total;
  bool indexed;
  const int rc = collect_segments(a->dtype, a->segments, a->n_segments, sg, total, indexed);
  if (rc) return rc;
  PKV_REQUIRE(total < ((int64_t)1 << 23), "pkv_tree_attention: at most 2^23 - 1 keys (got %lld)", (long long)total);
  const int rows = a->n_draft * a->group;
  const int64_t n_rows = (int64_t)a->bs * a->n_kv_heads * rows;
  const TreePlan p = tree_plan(a->dtype, a->bs, a->n_kv_heads, rows, total);
  const size_t need = tree_ws_floats(p, n_rows) * sizeof(float);
  if (need && (!a->ws || a->ws_bytes < need || !pkv_aligned(a->ws, 16))) {
    pkv_set_error("pkv_tree_attention: workspace of %zu bytes required, got %zu", need, a->ws ? a->ws_bytes : (size_t)0);
    return PKV_ENOMEM;
  }
  TreeCall c;
  memset(&c, 0, sizeof c);
  c.q = a->q, c.q_stride_b = a->q_stride_b, c.q_stride_t = a->q_stride_t;
  c.n_kv_heads = a->n_kv_heads, c.group = a->group, c.n_draft = a->n_draft;
  c.total = (uint32_t)total, c.row_keys = a->row_keys;
  c.dk = (const char *)a->draft_k, c.dk_b = a->dk_stride_b * es, c.dk_h = a->dk_stride_h * es, c.dk_t = a->dk_stride_t * es;
  c.dv = (const char *)a->draft_v, c.dv_b = a->dv_stride_b * es, c.dv_h = a->dv_stride_h * es, c.dv_t = a->dv_stride_t * es;
  c.mask = a->mask, c.mask_b = a->mask_stride_b, c.mask_t = a->mask_stride_t;
  c.scale_log2e = a->scale * 1.4426950408889634f;
  c.ws_o = (float *)a->ws, c.ws_ml = c.ws_o ? c.ws_o + n_rows * p.n_splits * 128 : nullptr;
  c.out = a->out;
  AttOne one;
  const bool is_one = as_one_tensor(sg, (int)es, one);
  hipStream_t s = (hipStream_t)stream;
  c.n_splits = p.n_splits, c.row_tiles = p.row_tiles, c.n_pairs = a->bs * a->n_kv_heads * p.n_splits;
  c.n_bh = a->bs * a->n_kv_heads;
  if (a->row_keys && p.n_splits > 1 && c.n_bh <= PKV_WAVE) c.by_keys = 1 + __builtin_ctz(p.turn);
  const dim3 grid = tree_grid(c);
  const dim3 block((p.rw == 1 ? kTreeWaves : kWideWaves) * PKV_WAVE);
#define PKV_TREE(IDX, S, SHARES)                                                                                     \
  do {                                                                                                               \
    if (p.rw == 1) PKV_TREE_LAUNCH((pkv_tree_partial_kernel<BF, IDX, decltype(S), SHARES>), S);                      \
    else if (p.rw == 2) PKV_TREE_LAUNCH((pkv_tree_wide_kernel<BF, 1, 2, IDX, decltype(S), SHARES>), S);              \
    else if (p.nt == 1) PKV_TREE_LAUNCH((pkv_tree_wide_kernel<BF, 1, 4, IDX, decltype(S), SHARES>), S);              \
    else PKV_TREE_LAUNCH((pkv_tree_wide_kernel<BF, BF ? 2 : 1, 4, IDX, decltype(S), SHARES>), S);  /* two: bf16 */     \
  } while (0)
#define PKV_TREE_LAUNCH(KERNEL, S) hipLaunchKernelGGL(KERNEL, grid, block, 0, s, c, S)
#define PKV_TREE_S                                                              \
  do {                                                                          \
    if (c.by_keys && is_one) { if (indexed) PKV_TREE(true, one, true); else PKV_TREE(false, one, true); } \
    else if (c.by_keys) { if (indexed) PKV_TREE(true, sg, true); else PKV_TREE(false, sg, true); }        \
    else if (is_one) { if (indexed) PKV_TREE(true, one, false); else PKV_TREE(false, one, false); }       \
    else { if (indexed) PKV_TREE(true, sg, false); else PKV_TREE(false, sg, false); }                     \
  } while (0)
  if (bf) {
    constexpr bool BF = true;
    PKV_TREE_S;
  } else {
    constexpr bool BF = false;
    PKV_TREE_S;
  }
#undef PKV_TREE_S
#undef PKV_TREE_LAUNCH
#undef PKV_TREE
  PKV_LAUNCH_CHECK("pkv_tree_partial_kernel");
  if (p.n_splits == 1) return PKV_OK;
  const dim3 merge((unsigned)((n_rows + 3) / 4));
  if (bf)
    hipLaunchKernelGGL(pkv_tree_merge_kernel<true>, merge, dim3(256), 0, s, c.ws_o, c.ws_ml, c.out, c.row_keys, c.n_splits, (uint32_t)rows,
                       (uint32_t)n_rows, (uint32_t)c.n_draft, (uint32_t)c.group, (uint32_t)c.n_kv_heads, c.by_keys, c.total, c.n_bh, c.n_pairs);
  else
    hipLaunchKernelGGL(pkv_tree_merge_kernel<false>, merge, dim3(256), 0, s, c.ws_o, c.ws_ml, c.out, c.row_keys, c.n_splits, (uint32_t)rows,
                       (uint32_t)n_rows, (uint32_t)c.n_draft, (uint32_t)c.group, (uint32_t)c.n_kv_heads, c.by_keys, c.total, c.n_bh, c.n_pairs);
  PKV_LAUNCH_CHECK("pkv_tree_merge_kernel");
  return PKV_OK;
}
