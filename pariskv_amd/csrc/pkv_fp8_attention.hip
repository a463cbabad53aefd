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
// bf16 queries: weights are rounded to bf16 (half a step, 2^-8 of themselves), times their values' scales for the product and as they are for the normaliser: the same
// ones where scales are powers of two.
// fp32 queries: q and the weights as sums of three bf16 numbers each, which hold their 24 bits; products with codes are exact.
// Softmax over all keys a row sees in one pass, with a running base and sum in fp32.
#include "pkv_attn.h"
#include "pkv_fp8.h"

#pragma clang fp contract(fast)

namespace {

constexpr int kWaves = 4, kStep = 64, kJoinSplits = 16, kMaxSplits = 16 * kJoinSplits;

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
  bool once;  // a key is read by one workgroup only
  uint32_t total;
  Seg seg[PKV_ATTN_MAX_SEGMENTS];
};

__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
  const pkv_f32x2 v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, pkv_bf16x2));
}
// Key of a half step (32 keys) that element e of lane (., j) belongs to.
__device__ __forceinline__ int key_of(int e, int j) { return 16 * (e >> 2) + 4 * j + (e & 3); }

// PARTS: bf16 numbers that make up a number of q and of the weights.  One tile of 16 query rows.
template <int PARTS>
struct Tile {
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

// Products of q and codes, times kx (a key's scale, and scale log2 e), into weights of the keys in `bits` (MASKED; else of all).
template <bool MASKED, int PARTS>
__device__ __forceinline__ void weights(Tile<PARTS> &w, const float (&s)[8], const float (&kx)[8], uint32_t bits, float (&p)[8]) {
  const int j = pkv_lane() >> 4;
  float x[8], top = -INFINITY;  // scores above use
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = !MASKED || ((bits >> e) & 1u) ? fmaf(s[e], kx[e], -w.use) : -INFINITY;
    top = fmaxf(top, x[e]);
  }
  if (__any(top > w.lim)) {
    top = pkv_pair_max<32>(pkv_pair_max<16>(top));
    const bool fresh = w.lim < 0.f, moves = top > -INFINITY && (fresh || top > 0.f);
    const float next = moves ? w.use + top : w.use, down = w.use - next, corr = fresh ? 0.f : __builtin_amdgcn_exp2f(down);
    w.use = next, w.lim = moves ? 8.f : w.lim;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] += down;
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
  for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(x[e]);
  if constexpr (PARTS == 1) {
    const pkv_u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
    pkv_u32x4 a;
#pragma unroll
    for (int d = 0; d < 4; ++d) a[d] = bf16x2(p[2 * d], p[2 * d + 1]);
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

// The codes of half a step, 32 keys, that a lane multiplies: of two tiles of keys, and eight dims of its eight keys' values.
struct Half {
  pkv_u32x4 k[2][2];
  pkv_u32x2 v[8];
  // in LDS: row i of K at 128 i, of V 4096 further, 16-byte vector v of it at v ^ (i mod 8), so that rows of an operand are on different banks
  __device__ __forceinline__ void from_lds(const uint8_t *at) {
    const int lane = pkv_lane(), n = lane & 15, j = lane >> 4;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) k[t][i] = *(const pkv_u32x4 *)(at + (16 * t + n) * 128 + 16 * ((4 * i + j) ^ (n & 7)));
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = *(const pkv_u32x2 *)(at + 4096 + key_of(e, j) * 128 + 16 * ((n >> 1) ^ (key_of(e, j) & 7)) + 8 * (n & 1));
  }
};

// Half a step.  kx, vx: the scales of the lane's keys (K's with scale log2 e); first: of the 32, in the key order.
template <bool MASKED, int PARTS, int NT>
__device__ __forceinline__ void half_step(Tile<PARTS> (&w)[NT], Half &x, const float (&kx)[8], const float (&vx)[8], int first, int n_here,
                                          const int (&limit)[NT]) {
  const int j = pkv_lane() >> 4;
  pkv_f32x4 s0[NT], s1[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) s0[t] = s1[t] = pkv_f32x4{0.f, 0.f, 0.f, 0.f};
  const pkv_u32x4(&k)[2][2] = x.k;
  pkv_u32x2(&v)[8] = x.v;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    pkv_u32x4 a, b;
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      a[2 * d] = fp8_bf16x2<false>(k[0][c >> 1][2 * (c & 1) + d]), a[2 * d + 1] = fp8_bf16x2<true>(k[0][c >> 1][2 * (c & 1) + d]);
      b[2 * d] = fp8_bf16x2<false>(k[1][c >> 1][2 * (c & 1) + d]), b[2 * d + 1] = fp8_bf16x2<true>(k[1][c >> 1][2 * (c & 1) + d]);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int p = PARTS - 1; p >= 0; --p) s0[t] = mfma_bf16(a, w[t].q[p][c], s0[t]), s1[t] = mfma_bf16(b, w[t].q[p][c], s1[t]);
  }
  uint32_t bits[NT], there = 0xffu;
  pkv_u32x4 a[NT][PARTS];
  if constexpr (MASKED) {
    there = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) there |= first + key_of(e, j) < n_here ? 1u << e : 0u;
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    bits[t] = 0xffu;
    if constexpr (MASKED) {
      bits[t] = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) bits[t] |= first + key_of(e, j) < limit[t] ? 1u << e : 0u;
    }
    float s[8], p[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = e < 4 ? s0[t][e & 3] : s1[t][e & 3];
    weights<MASKED, PARTS>(w[t], s, kx, bits[t], p);
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] *= MASKED && !((bits[t] >> e) & 1u) ? 0.f : vx[e];
    if constexpr (PARTS == 1) {
#pragma unroll
      for (int d = 0; d < 4; ++d) a[t][0][d] = bf16x2(p[2 * d], p[2 * d + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < PARTS; ++i) split_off(p, a[t][i]);
    }
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
        pkv_u32x4 is_nan;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const uint32_t lo = (b[m][d] & 0x7fffu) > 0x7f80u ? 0xffffu : 0u, hi = (b[m][d] & 0x7fff0000u) > 0x7f800000u ? 0xffff0000u : 0u;
          is_nan[d] = (lo | hi) & 0x3f803f80u, b[m][d] &= ~(lo | hi);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          pkv_u32x4 seen;
#pragma unroll
          for (int d = 0; d < 4; ++d) seen[d] = ((bits[t] >> (2 * d)) & 1u ? 0x3f80u : 0u) | ((bits[t] >> (2 * d + 1)) & 1u ? 0x3f800000u : 0u);
          const pkv_f32x4 hits = mfma_bf16(seen, is_nan, pkv_f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (hits[i] > 0.f) w[t].o[4 * h + m][i] = NAN;
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = PARTS - 1; i >= 0; --i) w[t].o[4 * h + m] = mfma_bf16(a[t][i], b[m], w[t].o[4 * h + m]);
    }
  }
}

// The kStep rows of keys jj .. lie one behind the other in a segment, at a distance of a multiple of four from their numbers.  (Fields of segments as
// values in scalar registers: picked by a lane they would be loaded from memory, and waited for with all that is under way.)
__device__ __forceinline__ bool is_plain(const Call &a, uint32_t jj) {
  bool plain = false;
  uint32_t lo = 0;
#pragma unroll
  for (int t = 0; t < PKV_ATTN_MAX_SEGMENTS; ++t) {
    const uint32_t end = att_field(a.seg[t].end), off = (uint32_t)att_field(a.seg[t].delta) | (a.seg[t].idx ? 1u : 0u);
    plain |= jj >= lo && jj + kStep <= end && (off & 3u) == 0;
    lo = end;
  }
  return plain && jj + kStep <= a.total;  // the last segment's end is open
}

// Row of concatenated key jj (plain: of a step for which is_plain says so).
template <bool INDEXED>
__device__ __forceinline__ uint32_t row_of(const Call &a, int bh, uint32_t jj, bool plain) {
  int32_t d = att_field(a.seg[0].delta);
#pragma unroll
  for (int t = 1; t < PKV_ATTN_MAX_SEGMENTS; ++t) {
    const int32_t next = att_field(a.seg[t].delta);
    d = jj >= att_field(a.seg[t - 1].end) ? next : d;
  }
  uint32_t r = jj + (uint32_t)d;
  if (INDEXED && !plain) {
    uint32_t lo = 0;
#pragma unroll
    for (int t = 0; t < PKV_ATTN_MAX_SEGMENTS; ++t) {
      const uint32_t hi = att_field(a.seg[t].end);
      if (t < a.n_segments && a.seg[t].idx && jj >= lo && jj < hi) {
        const int64_t x = a.seg[t].idx[(int64_t)bh * a.seg[t].idx_stride + (jj - lo)];
        r = lo + (uint32_t)a.seg[t].delta + (uint32_t)(x < 0 ? 0 : x >= a.seg[t].limit ? a.seg[t].limit - 1 : x);
      }
      lo = hi;
    }
  }
  return r;
}

// Until at most LEFT of this wave's loads are on their way, and none of its reads of LDS.
template <int LEFT>
__device__ __forceinline__ void wait_for() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LEFT) : "memory");
}
typedef const __attribute__((address_space(1))) void *global_at;
typedef __attribute__((address_space(3))) void *lds_at;

// A wave takes steps of 64 keys, dealt round the waves of all splits.  Rows go straight from memory to LDS, half a step at a time into a part of the
// wave's own: a half is asked for as soon as the one before in its place has been used, and no registers wait for it.  But the scales of the next step are multiplied with
// scale log2 e where they are loaded, in front of the first half's products, and loads come back in order: a wave waits for both halves there, and has nothing under way while it
// multiplies the first.  4 x 8 heads x 65536 keys (541 MB): 85 to 101 us and 4.6 the join; of 106 in all, 101 without any arithmetic and 51 without the loads (a plain read of
// as many bytes takes 77); rows kept by the caches 120; straight to registers, half a step ahead, 115 to 125.  More than 16 query rows: two tiles of them a wave, which share the codes' conversion: 1 x 8 x 32768
// keys, 256 rows 65 us, one tile 105.  Where several workgroups read a key, for their tiles of rows, the caches keep it: 65 and 74 us.
template <bool BF16, int NT, bool INDEXED>
__global__ __launch_bounds__(kWaves * PKV_WAVE, 2) void pkv_fp8_attention_kernel(Call a) {
  constexpr int PARTS = BF16 ? 1 : 3, kHalf = 8192;
  __shared__ alignas(16) uint8_t lds[kWaves * 2 * kHalf];
  // Workgroups go to the eight dies in turn, and the row tiles of one split read the same keys: they are eight numbers apart.
  const int pair = (int)blockIdx.y * 8 + (blockIdx.x & 7), tile = (int)blockIdx.x >> 3;
  if (pair >= a.n_pairs) return;  // the whole workgroup
  const int bh = (unsigned)pair / (unsigned)a.n_splits, split = pair - bh * a.n_splits;
  const int b = (unsigned)bh / (unsigned)a.n_kv_heads, h = bh - b * a.n_kv_heads;
  const int tid = threadIdx.x, lane = pkv_lane(), wave = __builtin_amdgcn_readfirstlane(tid / PKV_WAVE), n = lane & 15, j = lane >> 4;
  const int rows = a.n_tokens * a.group;
  int total = (int)a.total;
  if (a.row_keys) total = a.row_keys[bh] < total ? a.row_keys[bh] : total;
  const int full = total - (a.n_tokens - 1);

  Tile<PARTS> w[NT];
  int limit[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = (tile * NT + t) * 16 + n, my_row = r < rows ? r : rows - 1, token = (unsigned)my_row / (unsigned)a.group;  // past the last: not stored
    limit[t] = total - (a.n_tokens - 1 - token);
    const char *const qp = a.q + b * a.q_stride_b + token * a.q_stride_t + (int64_t)(h * a.group + my_row - token * a.group) * (BF16 ? 256 : 512);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int dim = 64 * (c >> 1) + 16 * j + 8 * (c & 1);  // of the eight of bytes 16 j + 64 (c / 2) + 8 (c % 2) ..
      if constexpr (BF16) {
        w[t].q[0][c] = *(const pkv_u32x4 *)(qp + dim * 2);
      } else {
        float x[8];
        fp8_load8<false>(qp + dim * 4, x);
#pragma unroll
        for (int i = 0; i < PARTS; ++i) split_off(x, w[t].q[i][c]);
      }
    }
    w[t].use = 0.f, w[t].lim = -INFINITY, w[t].l = pkv_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int m = 0; m < 8; ++m) w[t].o[m] = pkv_f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const uint8_t *const kb = a.k + (int64_t)bh * a.capacity * 128, *const vb = a.v + (int64_t)bh * a.capacity * 128;  // below 2^31 bytes each
  const float *const ks = a.k_scale + (int64_t)bh * a.n_blocks, *const vs = a.v_scale + (int64_t)bh * a.n_blocks;
  uint8_t *const mine = lds + wave * 2 * kHalf;
  // Lane l of a step knows the place and the scales of its key l.  plain: the step's rows lie one behind the other, and four keys from a multiple of
  // four on are in one block: addresses are sums and a lane's eight keys of half a step have two scales.  Else both come from the lanes that know
  // them, by exchanges through LDS, which take it 16 cycles each.
  struct Place {
    uint32_t row;
    float k, v;
    bool plain;
  };
  auto place = [&](int first) {
    Place p;
    p.plain = is_plain(a, (uint32_t)first);
    p.row = row_of<INDEXED>(a, bh, (uint32_t)(first + lane < total ? first + lane : total - 1), p.plain);
    p.k = ks[p.row >> a.lg_block] * a.scale_log2e, p.v = vs[p.row >> a.lg_block];
    return p;
  };
  auto fetch = [&](const Place &p, int s) {  // eight loads
    __builtin_amdgcn_sched_barrier(0);
    uint32_t row[4];
    if (p.plain) {  // the whole wave
      const uint32_t row0 = __builtin_amdgcn_readfirstlane(p.row) + 32 * s + (lane >> 3);
#pragma unroll
      for (int u = 0; u < 4; ++u) row[u] = row0 + 8 * u;
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u) row[u] = (uint32_t)__shfl((int)p.row, 32 * s + 8 * u + (lane >> 3), PKV_WAVE);
    }
#define PKV_FETCH(POLICY)                                                                                                                     \
  _Pragma("unroll") for (int u = 0; u < 4; ++u) {                                                                                             \
    const uint32_t at = row[u] * 128u + 16u * ((lane & 7) ^ (lane >> 3));                                                                     \
    __builtin_amdgcn_global_load_lds((global_at)(kb + at), (lds_at)(mine + s * kHalf + u * 1024), 16, 0, POLICY);                             \
    __builtin_amdgcn_global_load_lds((global_at)(vb + at), (lds_at)(mine + s * kHalf + 4096 + u * 1024), 16, 0, POLICY);                      \
  }
    if (a.once) PKV_FETCH(2) else PKV_FETCH(0)  // 2: streaming
#undef PKV_FETCH
    __builtin_amdgcn_sched_barrier(0);
  };
  auto scales = [&](const Place &p, int s, float (&kx)[8], float (&vx)[8]) {
    if (p.plain) {  // the whole wave
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float k = __shfl(p.k, 32 * s + 16 * t + 4 * j, PKV_WAVE), v = __shfl(p.v, 32 * s + 16 * t + 4 * j, PKV_WAVE);
#pragma unroll
        for (int e = 0; e < 4; ++e) kx[4 * t + e] = k, vx[4 * t + e] = v;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) kx[e] = __shfl(p.k, 32 * s + key_of(e, j), PKV_WAVE), vx[e] = __shfl(p.v, 32 * s + key_of(e, j), PKV_WAVE);
    }
  };
  auto compute = [&](const Place &p, int s) {
    float kx[8], vx[8];
    Half x;
    x.from_lds(mine + s * kHalf);
    scales(p, s, kx, vx);
    half_step<false, PARTS, NT>(w, x, kx, vx, 0, 0, limit);
  };
  const int turn = kWaves * a.n_splits * kStep;
  int first = (split * kWaves + wave) * kStep;
  if (first + kStep <= full) {  // the whole wave; steps that all rows see in full
    Place here = place(first), next = here;
    fetch(here, 0);
    fetch(here, 1);
    for (;;) {
      const bool more = first + turn + kStep <= full;
      wait_for<8>();  // the first half is there
      if (more) next = place(first + turn);
      compute(here, 0);
      if (more) {
        fetch(next, 0);
        wait_for<8>();  // the second half is there
      } else {
        wait_for<0>();
      }
      compute(here, 1);
      first += turn;
      if (!more) break;
      fetch(next, 1);
      here = next;
    }
  }
  for (; first < total; first += turn) {
    const Place here = place(first);
    wait_for<63>();  // its reads of the last step are done; loads need not be
    fetch(here, 0);
    fetch(here, 1);
    wait_for<0>();
#pragma unroll 1
    for (int s = 0; s < 2; ++s) {
      float kx[8], vx[8];
      Half x;
      x.from_lds(mine + s * kHalf);
      scales(here, s, kx, vx);
      half_step<true, PARTS, NT>(w, x, kx, vx, first + 32 * s, total, limit);
    }
  }

  // The waves meet, a tile of 16 rows at a time, and leave their result, or the split's part of it.
  float(*const s_m)[16] = (float(*)[16])lds, (*const s_l)[16] = (float(*)[16])(lds + 64 * kWaves), (*const s_o)[16][132] = (float(*)[16][132])(lds + 128 * kWaves);
  static_assert(128 * kWaves + kWaves * 16 * 132 * 4 <= (int)sizeof lds, "room for it");
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    __syncthreads();
    if (j == 0) s_m[wave][n] = w[t].lim < 0.f ? -INFINITY : w[t].use;
    if constexpr (PARTS == 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n == 0) s_l[wave][4 * j + i] = w[t].l[i];
    } else {
      const float l = pkv_pair_add<32>(pkv_pair_add<16>(w[t].l[0]));
      if (j == 0) s_l[wave][n] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      *(float4 *)&s_o[wave][4 * j + i][8 * n] = float4{w[t].o[0][i], w[t].o[1][i], w[t].o[2][i], w[t].o[3][i]};
      *(float4 *)&s_o[wave][4 * j + i][8 * n + 4] = float4{w[t].o[4][i], w[t].o[5][i], w[t].o[6][i], w[t].o[7][i]};
    }
    __syncthreads();
    for (int e = tid; e < 16 * 32; e += kWaves * PKV_WAVE) {  // four dims at a time
      const int r = e >> 5, d = 4 * (e & 31), row = (tile * NT + t) * 16 + r;
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
}

// 16 splits of a query row a wave, so that all partial results are one memory round trip: WAVES of them a row, or four rows a workgroup.  Lane l weighs split l of
// the wave and holds dims 2 l, 2 l + 1.  us with the join, 64 splits, one wave a row in four rounds / four waves: 1 x 8 x 32768 keys 19.5 / 17.5,
// 1 x 8 x 8000 10.3 / 9.3.
template <bool BF16, int WAVES>
__global__ __launch_bounds__(WAVES > 4 ? WAVES * PKV_WAVE : 256) void pkv_fp8_join_kernel(const float *__restrict__ ws_o, const float *__restrict__ ws_ml,
                                                                                          void *__restrict__ out, int n_splits, uint32_t rows, uint32_t n_rows,
                                                                                          uint32_t n_tokens, uint32_t group, uint32_t n_kv_heads) {
  __shared__ float s_m[WAVES], s_l[WAVES];
  __shared__ float2 s_o[WAVES][PKV_WAVE];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / PKV_WAVE), lane = pkv_lane(), s0 = WAVES > 1 ? wave * kJoinSplits : 0;
  const uint32_t at = WAVES > 1 ? blockIdx.x : blockIdx.x * 4 + wave;
  if (at >= n_rows) return;  // WAVES > 1: no such workgroup
  const uint32_t bh = at / rows, row = at - bh * rows;
  const int64_t first = (int64_t)bh * n_splits * rows + row;
  const float *const parts = ws_o + first * 128;
  float2 o[kJoinSplits];
#pragma unroll
  for (int i = 0; i < kJoinSplits; ++i)  // past the last split: the last again, as zeros
    o[i] = *(const float2 *)(parts + (int64_t)(s0 + i < n_splits ? s0 + i : n_splits - 1) * rows * 128 + 2 * lane);
  float m = -INFINITY, l = 0.f;
  if (lane < kJoinSplits && s0 + lane < n_splits) {
    const float2 ml = *(const float2 *)(ws_ml + (first + (int64_t)(s0 + lane) * rows) * 2);
    m = ml.x, l = ml.y;
  }
  float mx = pkv_wave_max(m);
  const float c = __builtin_amdgcn_exp2f(m - (mx == -INFINITY ? 0.f : mx));
  float all = pkv_wave_sum(l * c), x = 0.f, y = 0.f;
#pragma unroll
  for (int i = 0; i < kJoinSplits; ++i) {
    const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(c), i));
    const bool in = s0 + i < n_splits;
    x = fmaf(in ? o[i].x : 0.f, f, x), y = fmaf(in ? o[i].y : 0.f, f, y);
  }
  if constexpr (WAVES > 1) {
    s_o[wave][lane] = float2{x, y};
    if (lane == 0) s_m[wave] = mx, s_l[wave] = all;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) mx = fmaxf(mx, s_m[w]);
    const float base = mx == -INFINITY ? 0.f : mx;
    all = x = y = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float f = __builtin_amdgcn_exp2f(s_m[w] - base);
      all = fmaf(s_l[w], f, all), x = fmaf(s_o[w][lane].x, f, x), y = fmaf(s_o[w][lane].y, f, y);
    }
  }
  const float share = all == 0.f ? 0.f : 1.0f / all;  // 0: nothing seen
  x *= share, y *= share;
  const uint32_t b = bh / n_kv_heads, h = bh - b * n_kv_heads, u = row / group;
  const int64_t to = (((int64_t)b * n_tokens + u) * n_kv_heads * group + h * group + (row - u * group)) * 128 + 2 * lane;
  if constexpr (BF16) *(uint32_t *)((uint16_t *)out + to) = bf16x2(x, y);
  else *(float2 *)((float *)out + to) = float2{x, y};
}

// Row tiles of 16 a wave.
int tiles_a_wave(int dtype, int rows) { return dtype == PKV_DTYPE_BF16 && rows > 16 ? 2 : 1; }

// Workgroups: two to a compute unit, as many as fit there at a time, for bf16 and not one more: a second round starts anew for what is left.  us, up to 512 of
// them / rounded up / up to 1024: 3 x 8 x 20000 keys, 32 rows 35.2 / 42.7 / 42.2; 3 x 7 x 9000, 20 rows 20.4 / 22.6 / 23.6; 1 x 8 x 32768, 256 rows 65 / 65 / 71.
// Four where a wave of one row tile has sixteen steps or more, and the rounds even out what memory does: 4 x 8 x 65536 keys, 4 rows 110 / 110 / 105;
// 7 x 8 x 30000 (fewer) 84.4 / 90 / 84.6.  fp32, whose steps are longer, rounds up: 3 x 4 x 9001, 35 rows 17.5, not so 19.1 (but 3 x 3 x 20000, 24 rows 23.2 and 21.3);
// one row tile up to 1024, 4 x 2 x 20000 19.1.
// Two row tiles a wave: two steps at least where that leaves each compute unit a workgroup, since a workgroup's 32 rows of results cost as much as a step:
// 4 x 8 x 4096 keys, 32 rows 17.6, one step 20.3; 4 x 8 x 1000 (128 of them) 14.3 and 12.0.
// Up to 512 keys are two steps a wave of one workgroup, which saves the join: 1 x 8 x 300 keys 7.5 us, split in two 8.3 and a launch more; 600 keys 9.7 and
// 8.4.  At most 64 a row tile, or a workgroup to a compute unit if that is more: 1 x 8 x 32768 keys, 64 splits 17.3, 128 21.9; 1 x 1 x 65536 keys 14.8,
// 256 splits 11.8.
int splits_of(int dtype, int64_t bh, int rows, int64_t total) {
  const int nt = tiles_a_wave(dtype, rows), row_tiles = (rows + 16 * nt - 1) / (16 * nt);
  const int64_t turn = kWaves * kStep, most = (total + turn - 1) / turn, tiles = bh * row_tiles;
  int64_t s;
  if (most <= 2) s = 1;
  else if (dtype == PKV_DTYPE_BF16) s = row_tiles == 1 && tiles <= 512 && most >= 16 * (512 / tiles) ? 1024 / tiles : 512 / tiles;
  else s = ((row_tiles > 1 ? 512 : 1024) + tiles - 1) / tiles;
  if (s > most) s = most;
  const int64_t two = (most + 1) / 2 > 256 / tiles ? (most + 1) / 2 : 256 / tiles;
  if (nt > 1 && s > two) s = two;
  int64_t cap = kMaxSplits / tiles;  // kMaxSplits: a workgroup to each compute unit
  if (cap < 64) cap = 64;
  if (s > cap) s = cap;
  return (int)(s < 1 ? 1 : s);
}

bool shape_ok(int bs, int n_kv_heads, int group, int n_tokens) {
  return bs > 0 && n_kv_heads > 0 && (int64_t)bs * n_kv_heads <= 65535 && group > 0 && n_tokens > 0 && n_tokens <= 1024 && (int64_t)n_tokens * group <= 8192;
}

}  // namespace

extern "C" size_t pkv_fp8_attention_ws_bytes(int dtype, int bs, int n_kv_heads, int group, int n_tokens, int64_t total_keys) {
  if (!shape_ok(bs, n_kv_heads, group, n_tokens) || total_keys < 0) return 0;
  const int rows = n_tokens * group, s = splits_of(dtype, (int64_t)bs * n_kv_heads, rows, total_keys);
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
    PKV_REQUIRE(g.n_rows >= 0 && g.n_rows <= PKV_FP8_MAX_ROWS && g.row0 >= 0 && g.row0 <= a->cache.capacity, "segment %d: rows out of range", i);
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
  const int rows = a->n_tokens * a->group, nt = tiles_a_wave(a->dtype, rows), row_tiles = (rows + 16 * nt - 1) / (16 * nt);
  const int64_t bh = (int64_t)bs * H, n_rows = bh * rows;
  c.n_splits = splits_of(a->dtype, bh, rows, total), c.n_pairs = (int)(bh * c.n_splits);
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
  c.n_kv_heads = H, c.group = a->group, c.n_tokens = a->n_tokens, c.once = row_tiles == 1;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid(8u * row_tiles, (unsigned)((c.n_pairs + 7) / 8)), block(kWaves * PKV_WAVE);
  const bool bf = a->dtype == PKV_DTYPE_BF16;
#define PKV_FP8_ATTENTION(BF16, NT)                                                                                 \
  do {                                                                                                              \
    if (indexed) hipLaunchKernelGGL((pkv_fp8_attention_kernel<BF16, NT, true>), grid, block, 0, s, c);              \
    else hipLaunchKernelGGL((pkv_fp8_attention_kernel<BF16, NT, false>), grid, block, 0, s, c);                     \
  } while (0)
  if (bf && nt == 2) PKV_FP8_ATTENTION(true, 2);
  else if (bf) PKV_FP8_ATTENTION(true, 1);
  else PKV_FP8_ATTENTION(false, 1);
#undef PKV_FP8_ATTENTION
  PKV_LAUNCH_CHECK("pkv_fp8_attention_kernel");
  if (c.n_splits == 1) return PKV_OK;
#define PKV_FP8_JOIN(BF16, WAVES)                                                                                                                    \
  hipLaunchKernelGGL((pkv_fp8_join_kernel<BF16, WAVES>), dim3((unsigned)(WAVES > 1 ? n_rows : (n_rows + 3) / 4)), dim3(WAVES > 4 ? WAVES * PKV_WAVE : 256), 0, s, \
                     c.ws_o, c.ws_ml, c.out, c.n_splits, (uint32_t)rows, (uint32_t)n_rows, (uint32_t)c.n_tokens, (uint32_t)c.group, (uint32_t)H)
  if (bf) {
    if (c.n_splits <= kJoinSplits) PKV_FP8_JOIN(true, 1);
    else if (c.n_splits <= 4 * kJoinSplits) PKV_FP8_JOIN(true, 4);
    else PKV_FP8_JOIN(true, 16);
  } else {
    if (c.n_splits <= kJoinSplits) PKV_FP8_JOIN(false, 1);
    else if (c.n_splits <= 4 * kJoinSplits) PKV_FP8_JOIN(false, 4);
    else PKV_FP8_JOIN(false, 16);
  }
#undef PKV_FP8_JOIN
  PKV_LAUNCH_CHECK("pkv_fp8_join_kernel");
  return PKV_OK;
}
