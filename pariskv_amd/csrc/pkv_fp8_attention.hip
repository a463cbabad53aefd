// Attention over a K/V cache in eight bits (pkv_fp8_cache.hip): softmax(scale q K^T) V with K = code * scale of its block, V the same, for
// one query token a sequence or several, of which each sees the cached rows up to its own.  (No counterpart in the reference, whose
// caches are bf16.)
//
// A KV head's T * G query rows (T tokens, G query heads) share its keys: 256 bytes a key, which bound it.  Codes become bf16 numbers in
// registers, exactly (v_cvt_scalef32_pk_bf16_fp8, two to an instruction), and go to the matrix cores as such; a key's scale is
// multiplied into its score, a value's into its weight.
//   scores   S^T[key][row] = K[key][dim] . Q^T[dim][row], v_mfma_f32_16x16x32_bf16: lane (n, j) has bytes 16 j .. and 64 + 16 j .. of key n of a tile
//            of 16, and receives the scores of row n for keys 4 j .. 4 j + 3 ...
//   output   O[row][dim] += P[row][key] . V[key][dim]: ... which is where this product wants the weights: nothing is moved.
// bf16 queries: weights are rounded to bf16 (half a step of 2^-8 each) and the normaliser is the sum of the rounded ones.
// fp32 queries: q and the weights as sums of three bf16 numbers each, which hold their 24 bits; products with codes are exact.
// Softmax over all keys a row sees in one pass, with a running base and sum in fp32.
#include "pkv_attn.h"
#include "pkv_fp8.h"

#pragma clang fp contract(fast)

namespace {

constexpr int kWaves = 4, kStep = 64, kMaxSplits = 64;

struct Seg {
  int64_t idx_stride;
  const int64_t *idx;
  uint32_t end;    // exclusive, in the concatenated key order
  int32_t delta;   // row - concatenated key
  uint32_t limit;  // rows that idx may name
};
struct Call {
  const char *q;
  int64_t q_stride_b, q_stride_t;  // bytes
  const uint8_t *k, *v;
  const float *k_scale, *v_scale;
  int64_t capacity, n_blocks;
  const int32_t *row_keys;
  float scale_log2e;
  float *ws_o, *ws_ml;  // [row of (b, h)][split][query row][128], [..][2]
  void *out;
  int n_kv_heads, group, n_tokens, lg_block, n_segments, n_splits, n_pairs;
  uint32_t total;
  Seg seg[PKV_ATTN_MAX_SEGMENTS];
};

__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
  const pkv_f32x2 v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, pkv_bf16x2));
}
// Key of a half step (32 keys) that element e of lane (., j) belongs to.
__device__ __forceinline__ int key_of(int e, int j) { return 16 * (e >> 2) + 4 * j + (e & 3); }

// PARTS: bf16 numbers that make up a number of q and of the weights.
template <int PARTS>
struct Wave {
  pkv_u32x4 q[PARTS][4];
  // Weights are 2^(score - use).  use moves, and the sums with it, when a score is above it by more than lim = 8, so that most steps neither
  // look for the row's maximum across lanes nor touch the sums; lim = -inf: the row has seen nothing yet.
  float use, lim;
  pkv_f32x4 l;     // sums: of rows 4 j + i (PARTS = 1); of row n, this lane's keys, in the first element
  pkv_f32x4 o[8];  // o[m][i]: row 4 j + i, dim 8 n + m
};

// x as a sum of bf16 numbers, part by part.
__device__ __forceinline__ void split_off(float (&x)[8], pkv_u32x4 &part) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    part[d] = bf16x2(x[2 * d], x[2 * d + 1]);
    x[2 * d] -= __uint_as_float(part[d] << 16), x[2 * d + 1] -= __uint_as_float(part[d] & 0xffff0000u);
  }
}

// Scores (times log2 e) into weights of the keys in `bits` (MASKED; else of all); p stays as numbers, for bf16 rounded.
template <bool MASKED, int PARTS>
__device__ __forceinline__ void weights(Wave<PARTS> &w, const float (&s)[8], uint32_t bits, float (&p)[8]) {
  const int j = pkv_lane() >> 4;
  float x[8], top = -INFINITY;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = !MASKED || ((bits >> e) & 1u) ? s[e] : -INFINITY;
    top = fmaxf(top, x[e]);
  }
  if (__any(top - w.use > w.lim)) {
    top = pkv_pair_max<32>(pkv_pair_max<16>(top));
    const bool fresh = w.lim < 0.f, moves = top > -INFINITY && (fresh || top > w.use);
    const float next = moves ? top : w.use, corr = fresh ? 0.f : __builtin_amdgcn_exp2f(w.use - next);
    w.use = next, w.lim = moves ? 8.f : w.lim;
    float cr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) cr[i] = __shfl(corr, 4 * j + i, PKV_WAVE);
#pragma unroll
    for (int m = 0; m < 8; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) w.o[m][i] *= cr[i];
    if constexpr (PARTS == 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w.l[i] *= cr[i];
    } else {
      w.l[0] *= corr;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(x[e] - w.use);
  if constexpr (PARTS == 1) {
    const pkv_u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
    pkv_u32x4 a;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      a[d] = bf16x2(p[2 * d], p[2 * d + 1]);
      p[2 * d] = __uint_as_float(a[d] << 16), p[2 * d + 1] = __uint_as_float(a[d] & 0xffff0000u);
    }
    w.l = mfma_bf16(a, ones, w.l);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) w.l[0] += p[e];
  }
}

// The m-th operand (dim 8 n + m) out of eight codes of each of the lane's eight keys.
__device__ __forceinline__ void turn_v(const pkv_u32x2 (&v)[8], int half, pkv_u32x4 (&out)[4]) {
  // dims 4 half .. 4 half + 3: two keys' bytes side by side, dim by dim, then to bf16
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const uint32_t a = v[2 * d][half], b = v[2 * d + 1][half];
    const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x05010400u), hi = __builtin_amdgcn_perm(b, a, 0x07030602u);
    out[0][d] = fp8_bf16x2<false>(lo), out[1][d] = fp8_bf16x2<true>(lo), out[2][d] = fp8_bf16x2<false>(hi), out[3][d] = fp8_bf16x2<true>(hi);
  }
}

// Half a step: 32 keys.  k: two tiles of 16; kx, vx: the scales of the lane's keys (K's with scale log2 e); first: of the 32, in the key order.
template <bool MASKED, int PARTS>
__device__ __forceinline__ void half_step(Wave<PARTS> &w, const pkv_u32x4 (&k)[2][2], pkv_u32x2 (&v)[8], const float (&kx)[8], const float (&vx)[8],
                                          int first, int n_here, int limit) {
  const int j = pkv_lane() >> 4;
  pkv_f32x4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    pkv_u32x4 a, b;
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      a[2 * d] = fp8_bf16x2<false>(k[0][c >> 1][2 * (c & 1) + d]), a[2 * d + 1] = fp8_bf16x2<true>(k[0][c >> 1][2 * (c & 1) + d]);
      b[2 * d] = fp8_bf16x2<false>(k[1][c >> 1][2 * (c & 1) + d]), b[2 * d + 1] = fp8_bf16x2<true>(k[1][c >> 1][2 * (c & 1) + d]);
    }
#pragma unroll
    for (int p = PARTS - 1; p >= 0; --p) s0 = mfma_bf16(a, w.q[p][c], s0), s1 = mfma_bf16(b, w.q[p][c], s1);
  }
  float s[8], p[8];
  uint32_t bits = 0xffu, there = 0xffu;
  if constexpr (MASKED) {
    bits = there = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int key = first + key_of(e, j);
      bits |= key < limit ? 1u << e : 0u, there |= key < n_here ? 1u << e : 0u;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) s[e] = (e < 4 ? s0[e & 3] : s1[e & 3]) * kx[e];
  weights<MASKED, PARTS>(w, s, bits, p);
#pragma unroll
  for (int e = 0; e < 8; ++e) p[e] *= MASKED && !((bits >> e) & 1u) ? 0.f : vx[e];
  pkv_u32x4 a[PARTS];
  if constexpr (PARTS == 1) {
#pragma unroll
    for (int d = 0; d < 4; ++d) a[0][d] = bf16x2(p[2 * d], p[2 * d + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < PARTS; ++i) split_off(p, a[i]);
  }
  bool odd = false;
  if constexpr (MASKED) {
    // Keys that are not there were read again: zeros.  A NaN among the values is for the rows that see its key and for no other, but in the
    // product it would be one for all: zero there, and put into the rows below.
    uint32_t any = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t keep = (there >> e) & 1u ? 0xffffffffu : 0u;
#pragma unroll
      for (int i = 0; i < 2; ++i) v[e][i] &= keep, any |= (v[e][i] & 0x7f7f7f7fu) + 0x01010101u;
    }
    odd = __any((any & 0x80808080u) != 0u);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    pkv_u32x4 b[4];
    turn_v(v, h, b);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      if (MASKED && odd) {
        pkv_u32x4 is_nan, seen;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const uint32_t lo = (b[m][d] & 0x7fffu) > 0x7f80u ? 0xffffu : 0u, hi = (b[m][d] & 0x7fff0000u) > 0x7f800000u ? 0xffff0000u : 0u;
          is_nan[d] = (lo | hi) & 0x3f803f80u, b[m][d] &= ~(lo | hi);
          seen[d] = ((bits >> (2 * d)) & 1u ? 0x3f80u : 0u) | ((bits >> (2 * d + 1)) & 1u ? 0x3f800000u : 0u);
        }
        const pkv_f32x4 hits = mfma_bf16(seen, is_nan, pkv_f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (hits[i] > 0.f) w.o[4 * h + m][i] = NAN;
      }
#pragma unroll
      for (int i = PARTS - 1; i >= 0; --i) w.o[4 * h + m] = mfma_bf16(a[i], b[m], w.o[4 * h + m]);
    }
  }
}

// Row of concatenated key jj.
template <bool INDEXED>
__device__ __forceinline__ uint32_t row_of(const Call &a, int bh, uint32_t jj) {
  uint32_t r = jj + (uint32_t)a.seg[0].delta;
#pragma unroll
  for (int t = 1; t < PKV_ATTN_MAX_SEGMENTS; ++t) r = jj >= a.seg[t - 1].end ? jj + (uint32_t)a.seg[t].delta : r;
  if constexpr (INDEXED) {
    uint32_t lo = 0;
#pragma unroll
    for (int t = 0; t < PKV_ATTN_MAX_SEGMENTS; ++t) {
      const uint32_t hi = a.seg[t].end;
      if (t < a.n_segments && a.seg[t].idx && jj >= lo && jj < hi) {
        const int64_t x = a.seg[t].idx[(int64_t)bh * a.seg[t].idx_stride + (jj - lo)];
        r = lo + (uint32_t)a.seg[t].delta + (uint32_t)(x < 0 ? 0 : x >= a.seg[t].limit ? a.seg[t].limit - 1 : x);
      }
      lo = hi;
    }
  }
  return r;
}

template <bool BF16, bool INDEXED>
__global__ __launch_bounds__(kWaves * PKV_WAVE, 2) void pkv_fp8_attention_kernel(Call a) {
  constexpr int PARTS = BF16 ? 1 : 3;
  // Workgroups go to the eight dies in turn, and the row tiles of one split read the same keys: they are eight numbers apart.
  const int pair = (int)blockIdx.y * 8 + (blockIdx.x & 7), tile = (int)blockIdx.x >> 3;
  if (pair >= a.n_pairs) return;  // the whole workgroup
  const int bh = (unsigned)pair / (unsigned)a.n_splits, split = pair - bh * a.n_splits;
  const int b = (unsigned)bh / (unsigned)a.n_kv_heads, h = bh - b * a.n_kv_heads;
  const int tid = threadIdx.x, lane = pkv_lane(), wave = __builtin_amdgcn_readfirstlane(tid / PKV_WAVE), n = lane & 15, j = lane >> 4;
  const int rows = a.n_tokens * a.group, my_row = tile * 16 + n < rows ? tile * 16 + n : rows - 1, token = (unsigned)my_row / (unsigned)a.group;
  int total = (int)a.total;
  if (a.row_keys) total = a.row_keys[bh] < total ? a.row_keys[bh] : total;
  const int limit = total - (a.n_tokens - 1 - token), full = total - (a.n_tokens - 1);

  Wave<PARTS> w;
  const char *const qp = a.q + b * a.q_stride_b + token * a.q_stride_t + (int64_t)(h * a.group + my_row - token * a.group) * (BF16 ? 256 : 512);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int dim = 64 * (c >> 1) + 16 * j + 8 * (c & 1);  // of the eight of bytes 16 j + 64 (c / 2) + 8 (c % 2) ..
    if constexpr (BF16) {
      w.q[0][c] = *(const pkv_u32x4 *)(qp + dim * 2);
    } else {
      float x[8];
      fp8_load8<false>(qp + dim * 4, x);
#pragma unroll
      for (int i = 0; i < PARTS; ++i) split_off(x, w.q[i][c]);
    }
  }
  w.use = 0.f, w.lim = -INFINITY, w.l = pkv_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int m = 0; m < 8; ++m) w.o[m] = pkv_f32x4{0.f, 0.f, 0.f, 0.f};

  const uint8_t *const kb = a.k + (int64_t)bh * a.capacity * 128, *const vb = a.v + (int64_t)bh * a.capacity * 128;
  const float *const ks = a.k_scale + (int64_t)bh * a.n_blocks, *const vs = a.v_scale + (int64_t)bh * a.n_blocks;
  const int turns = kWaves * a.n_splits;
  for (int first = (split * kWaves + wave) * kStep; first < total; first += turns * kStep) {
    const uint32_t my_key = (uint32_t)(first + lane < total ? first + lane : total - 1), row = row_of<INDEXED>(a, bh, my_key);
    const float my_k = ks[row >> a.lg_block] * a.scale_log2e, my_v = vs[row >> a.lg_block];
    pkv_u32x4 k[2][2][2];
    pkv_u32x2 v[2][8];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint8_t *const p = kb + (uint64_t)(uint32_t)__shfl((int)row, 32 * s + 16 * t + n, PKV_WAVE) * 128 + 16 * j;
        k[s][t][0] = *(const pkv_u32x4 *)p, k[s][t][1] = *(const pkv_u32x4 *)(p + 64);
      }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        v[s][e] = *(const pkv_u32x2 *)(vb + (uint64_t)(uint32_t)__shfl((int)row, 32 * s + key_of(e, j), PKV_WAVE) * 128 + 8 * n);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      float kx[8], vx[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) kx[e] = __shfl(my_k, 32 * s + key_of(e, j), PKV_WAVE), vx[e] = __shfl(my_v, 32 * s + key_of(e, j), PKV_WAVE);
      if (first + kStep <= full) half_step<false, PARTS>(w, k[s], v[s], kx, vx, first + 32 * s, total, limit);
      else half_step<true, PARTS>(w, k[s], v[s], kx, vx, first + 32 * s, total, limit);
    }
  }

  // The waves meet and leave their result, or the split's part of it.
  __shared__ float s_m[kWaves][16], s_l[kWaves][16];
  __shared__ alignas(16) float s_o[kWaves][16][132];
  if (j == 0) s_m[wave][n] = w.lim < 0.f ? -INFINITY : w.use;
  if constexpr (PARTS == 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n == 0) s_l[wave][4 * j + i] = w.l[i];
  } else {
    const float l = pkv_pair_add<32>(pkv_pair_add<16>(w.l[0]));
    if (j == 0) s_l[wave][n] = l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    *(float4 *)&s_o[wave][4 * j + i][8 * n] = float4{w.o[0][i], w.o[1][i], w.o[2][i], w.o[3][i]};
    *(float4 *)&s_o[wave][4 * j + i][8 * n + 4] = float4{w.o[4][i], w.o[5][i], w.o[6][i], w.o[7][i]};
  }
  __syncthreads();
  for (int e = tid; e < 16 * 32; e += kWaves * PKV_WAVE) {  // four dims at a time
    const int r = e >> 5, d = 4 * (e & 31), row = tile * 16 + r;
    if (row >= rows) continue;
    float mx = s_m[0][r];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) mx = fmaxf(mx, s_m[i][r]);
    const float base = mx == -INFINITY ? 0.f : mx;
    float ls = 0.f;
    pkv_f32x4 os = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      const float c = __builtin_amdgcn_exp2f(s_m[i][r] - base);
      const pkv_f32x4 x = *(const pkv_f32x4 *)&s_o[i][r][d];
      ls = fmaf(s_l[i][r], c, ls);
#pragma unroll
      for (int u = 0; u < 4; ++u) os[u] = fmaf(x[u], c, os[u]);
    }
    if (a.n_splits == 1) {
      const int u = (unsigned)row / (unsigned)a.group;
      const int64_t to = (((int64_t)b * a.n_tokens + u) * a.n_kv_heads * a.group + h * a.group + (row - u * a.group)) * 128 + d;
      const float share = ls == 0.f ? 0.f : 1.0f / ls;  // 0: nothing seen
#pragma unroll
      for (int i = 0; i < 4; ++i) os[i] *= share;
      if constexpr (BF16) *(pkv_u32x2 *)((uint16_t *)a.out + to) = pkv_u32x2{bf16x2(os[0], os[1]), bf16x2(os[2], os[3])};
      else *(pkv_f32x4 *)((float *)a.out + to) = os;
    } else {
      const int64_t at = (int64_t)pair * rows + row;
      *(pkv_f32x4 *)(a.ws_o + at * 128 + d) = os;
      if (d == 0) *(float2 *)(a.ws_ml + at * 2) = float2{mx, ls};
    }
  }
}

// One wave a query row: lane l weighs split l and holds dims 2 l, 2 l + 1 of the output.
template <bool BF16>
__global__ __launch_bounds__(256) void pkv_fp8_join_kernel(const float *__restrict__ ws_o, const float *__restrict__ ws_ml, void *__restrict__ out,
                                                           int n_splits, uint32_t rows, uint32_t n_rows, uint32_t n_tokens, uint32_t group,
                                                           uint32_t n_kv_heads) {
  const uint32_t at = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + threadIdx.x / PKV_WAVE);
  const int lane = pkv_lane();
  if (at >= n_rows) return;
  const uint32_t bh = at / rows, row = at - bh * rows;
  const int64_t first = (int64_t)bh * n_splits * rows + row;
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
  const int64_t to = (((int64_t)b * n_tokens + u) * n_kv_heads * group + h * group + (row - u * group)) * 128 + 2 * lane;
  if constexpr (BF16) *(uint32_t *)((uint16_t *)out + to) = bf16x2(x, y);
  else *(float2 *)((float *)out + to) = float2{x, y};
}

int splits_of(int64_t bh, int row_tiles, int64_t total) {
  const int64_t turn = kWaves * kStep, most = (total + turn - 1) / turn;
  int64_t s = (1024 + bh * row_tiles - 1) / (bh * row_tiles);
  if (s > most) s = most;
  if (s > kMaxSplits) s = kMaxSplits;
  return (int)(s < 1 ? 1 : s);
}

bool shape_ok(int bs, int n_kv_heads, int group, int n_tokens) {
  return bs > 0 && n_kv_heads > 0 && (int64_t)bs * n_kv_heads <= 65535 && group > 0 && n_tokens > 0 && n_tokens <= 1024 && (int64_t)n_tokens * group <= 8192;
}

}  // namespace

extern "C" size_t pkv_fp8_attention_ws_bytes(int bs, int n_kv_heads, int group, int n_tokens, int64_t total_keys) {
  if (!shape_ok(bs, n_kv_heads, group, n_tokens) || total_keys < 0) return 0;
  const int rows = n_tokens * group, s = splits_of((int64_t)bs * n_kv_heads, (rows + 15) / 16, total_keys);
  return s == 1 ? 0 : (size_t)bs * n_kv_heads * s * rows * 130 * sizeof(float);
}

extern "C" int pkv_fp8_attention(const pkv_fp8_attn_args *a, void *stream) {
  PKV_REQUIRE(a && a->q && a->out, "pkv_fp8_attention: null pointer");
  if (const int rc = pkv_fp8_kv_check(&a->cache, "pkv_fp8_attention")) return rc;
  const int bs = a->cache.bs, H = a->cache.n_kv_heads;
  PKV_REQUIRE(a->dtype == PKV_DTYPE_F32 || a->dtype == PKV_DTYPE_BF16, "unknown dtype %d", a->dtype);
  PKV_REQUIRE(shape_ok(bs, H, a->group, a->n_tokens),
              "pkv_fp8_attention: bad shape bs=%d kv_heads=%d group=%d tokens=%d (at most 1024 tokens, 8192 query rows a KV head)", bs, H, a->group, a->n_tokens);
  PKV_REQUIRE(a->n_segments >= 0 && a->n_segments <= PKV_ATTN_MAX_SEGMENTS, "0..%d key segments", PKV_ATTN_MAX_SEGMENTS);
  const int64_t es = a->dtype == PKV_DTYPE_BF16 ? 2 : 4;
  PKV_REQUIRE(pkv_aligned(a->q, 16) && pkv_aligned(a->out, 16) && a->q_stride_b * es % 16 == 0 && a->q_stride_t * es % 16 == 0,
              "pkv_fp8_attention: 16-byte aligned buffers and strides required");
  PKV_REQUIRE(!a->row_keys || pkv_aligned(a->row_keys, 4), "pkv_fp8_attention: row_keys must be int32");
  Call c;
  memset(&c, 0, sizeof c);
  int64_t total = 0;
  bool indexed = false;
  for (int i = 0; i < a->n_segments; ++i) {
    const pkv_fp8_segment &g = a->segments[i];
    PKV_REQUIRE(g.n_rows >= 0 && g.row0 >= 0 && g.row0 <= a->cache.capacity, "segment %d: rows out of range", i);
    if (g.n_rows == 0) continue;
    Seg &to = c.seg[c.n_segments++];
    if (g.idx) {
      PKV_REQUIRE(pkv_aligned(g.idx, 8) && g.idx_stride >= g.n_rows && g.row0 < a->cache.capacity, "segment %d: indexed rows need idx_stride >= n_rows", i);
      to.idx = g.idx, to.idx_stride = g.idx_stride, to.limit = (uint32_t)(a->cache.capacity - g.row0), indexed = true;
    } else {
      PKV_REQUIRE(g.row0 + g.n_rows <= a->cache.capacity, "segment %d: rows %lld.. (%lld of them) of %lld", i, (long long)g.row0, (long long)g.n_rows,
                  (long long)a->cache.capacity);
    }
    to.delta = (int32_t)(g.row0 - total);
    total += g.n_rows;
    PKV_REQUIRE(total <= PKV_FP8_MAX_ROWS, "pkv_fp8_attention: at most %lld keys", (long long)PKV_FP8_MAX_ROWS);
    to.end = (uint32_t)total;
  }
  for (int i = c.n_segments; i < PKV_ATTN_MAX_SEGMENTS; ++i) c.seg[i].end = 0xffffffffu;
  if (c.n_segments) c.seg[c.n_segments - 1].end = 0xffffffffu;
  const int rows = a->n_tokens * a->group, row_tiles = (rows + 15) / 16;
  const int64_t bh = (int64_t)bs * H, n_rows = bh * rows;
  c.n_splits = splits_of(bh, row_tiles, total), c.n_pairs = (int)(bh * c.n_splits);
  const size_t need = c.n_splits == 1 ? 0 : (size_t)n_rows * c.n_splits * 130 * sizeof(float);
  if (need && (!a->ws || a->ws_bytes < need || !pkv_aligned(a->ws, 16))) {
    pkv_set_error("pkv_fp8_attention: workspace of %zu bytes required, got %zu", need, a->ws ? a->ws_bytes : (size_t)0);
    return PKV_ENOMEM;
  }
  c.q = (const char *)a->q, c.q_stride_b = a->q_stride_b * es, c.q_stride_t = a->q_stride_t * es;
  c.k = a->cache.k, c.v = a->cache.v, c.k_scale = a->cache.k_scale, c.v_scale = a->cache.v_scale;
  c.capacity = a->cache.capacity, c.n_blocks = a->cache.capacity / a->cache.block, c.lg_block = __builtin_ctz(a->cache.block);
  c.row_keys = a->row_keys, c.scale_log2e = a->scale * 1.4426950408889634f, c.total = (uint32_t)total;
  c.ws_o = (float *)a->ws, c.ws_ml = need ? c.ws_o + (size_t)n_rows * c.n_splits * 128 : nullptr, c.out = a->out;
  c.n_kv_heads = H, c.group = a->group, c.n_tokens = a->n_tokens;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid(8u * row_tiles, (unsigned)((c.n_pairs + 7) / 8)), block(kWaves * PKV_WAVE);
  const bool bf = a->dtype == PKV_DTYPE_BF16;
  if (bf && indexed) hipLaunchKernelGGL((pkv_fp8_attention_kernel<true, true>), grid, block, 0, s, c);
  else if (bf) hipLaunchKernelGGL((pkv_fp8_attention_kernel<true, false>), grid, block, 0, s, c);
  else if (indexed) hipLaunchKernelGGL((pkv_fp8_attention_kernel<false, true>), grid, block, 0, s, c);
  else hipLaunchKernelGGL((pkv_fp8_attention_kernel<false, false>), grid, block, 0, s, c);
  PKV_LAUNCH_CHECK("pkv_fp8_attention_kernel");
  if (c.n_splits == 1) return PKV_OK;
  const dim3 join((unsigned)((n_rows + 3) / 4));
  if (bf) hipLaunchKernelGGL(pkv_fp8_join_kernel<true>, join, dim3(256), 0, s, c.ws_o, c.ws_ml, c.out, c.n_splits, (uint32_t)rows, (uint32_t)n_rows,
                             (uint32_t)c.n_tokens, (uint32_t)c.group, (uint32_t)H);
  else hipLaunchKernelGGL(pkv_fp8_join_kernel<false>, join, dim3(256), 0, s, c.ws_o, c.ws_ml, c.out, c.n_splits, (uint32_t)rows, (uint32_t)n_rows,
                          (uint32_t)c.n_tokens, (uint32_t)c.group, (uint32_t)H);
  PKV_LAUNCH_CHECK("pkv_fp8_join_kernel");
  return PKV_OK;
}
