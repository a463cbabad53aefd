// Attention of the drafted tokens of a tree over the cached keys and over each other: the verification step of speculative
// decoding.  (No counterpart in the reference, whose decode step takes one token a sequence.)
//
// A KV head's T * G query rows (T drafted tokens, G query heads) share its keys, so K and V (2 * 128 elements a key) are read once for
// all of them: up to some 64 rows the bytes bound it, beyond 256 the matrix instructions.  Rows go to the matrix cores 16 at
// a time, a wave holds NT such tiles; the four waves of a workgroup take keys in turns of their own and merge through LDS; the key axis is
// split over workgroups, whose partial results a second launch joins.  Nothing but the merge goes through LDS:
//   scores   S^T[key][row] = K[key][dim] . Q^T[dim][row]: lane (n, j) receives the scores of row n for four keys 4j .. 4j+3 of a
//            tile of 16 ...
//   output   O[row][dim] += P[row][key] . V[key][dim]: ... which is where this product wants the probabilities.
//            Columns n of instruction m are the dims 8n + m, so that rows of V are read whole.
// bf16: v_mfma_f32_16x16x32_bf16, 32 keys a step (see pkv_attn.h, whose one-token step this is for many rows); the probabilities
//       are rounded to bf16 for the second product, half a step of their own type each, and summed unrounded.
// fp32: v_mfma_f32_16x16x4_f32, 16 keys a step; no rounding.
// Softmax over all keys a row sees in one pass with the running maximum and sum, fp32.
#include "pkv_attn.h"

#pragma clang fp contract(fast)

namespace {

constexpr int kTreeWaves = 4, kTreeMaxSplits = 64;

struct TreeCall {
  const void *q;
  int64_t q_stride_b, q_stride_t;  // elements
  int n_kv_heads, group, n_draft;
  uint32_t total;                  // cached keys
  uint32_t per_split;              // a multiple of what the waves take in one step
  const int32_t *row_keys;
  const char *dk, *dv;
  int64_t dk_b, dk_h, dk_t, dv_b, dv_h, dv_t;  // bytes
  const uint8_t *mask;
  int64_t mask_b, mask_t;
  float scale_log2e;
  float *ws_o, *ws_ml;  // [row of (b, h)][split][query row][128], [..][2]
  void *out;
};

template <bool BF16, int NT>
struct TreeWave {
  static constexpr int kQ = BF16 ? 4 : 8;   // 16-byte vectors of a query row in a lane
  static constexpr int kE = BF16 ? 8 : 4;   // keys of a step in a lane
  static constexpr int kKeys = BF16 ? 32 : 16;
  static constexpr uint32_t kRow = BF16 ? 256 : 512;
  pkv_u32x4 q[NT][kQ];
  float m[NT], l[NT];
  pkv_f32x4 o[NT][8];
};

__device__ __forceinline__ pkv_f32x4 mfma_f32(float a, float b, pkv_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// Key of the step that element e of lane (., j) belongs to.
__device__ __forceinline__ int tree_key(int e, int j) { return 16 * (e >> 2) + 4 * j + (e & 3); }

// One step's keys into the wave's rows.  kv_at(key of the step, address of K, of V); sees(tile, e): whether the lane's row sees its key
// e; count: keys of the step that there are (the others are read again and count for nothing).
template <bool BF16, int NT, bool DRAFT, typename At, typename Sees>
__device__ __forceinline__ void tree_step(TreeWave<BF16, NT> &w, At at, Sees sees, int count, float scale_log2e) {
  using W = TreeWave<BF16, NT>;
  const int lane = pkv_lane(), n = lane & 15, j = lane >> 4;
  pkv_u32x4 k[8], v[8];
  if constexpr (BF16) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const char *kp, *vp;
      at(16 * t + n, kp, vp);
#pragma unroll
      for (int c = 0; c < 4; ++c) k[4 * t + c] = *(const pkv_u32x4 *)(kp + 64 * c + 16 * j);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const char *kp, *vp;
      at(tree_key(e, j), kp, vp);
      v[e] = *(const pkv_u32x4 *)(vp + 16 * n);
    }
  } else {
    const char *kp, *vp;
    at(n, kp, vp);
#pragma unroll
    for (int c = 0; c < 8; ++c) k[c] = *(const pkv_u32x4 *)(kp + 64 * c + 16 * j);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      at(tree_key(e, j), kp, vp);
      v[2 * e] = *(const pkv_u32x4 *)(vp + 32 * n);
      v[2 * e + 1] = *(const pkv_u32x4 *)(vp + 32 * n + 16);
    }
  }
  // Keys that are not there: zeros, so that nothing of a key read again reaches the sums.
  if (count < W::kKeys) {
#pragma unroll
    for (int e = 0; e < W::kE; ++e)
      if (tree_key(e, j) >= count) {
        if constexpr (BF16) v[e] = pkv_u32x4{0u, 0u, 0u, 0u};
        else v[2 * e] = v[2 * e + 1] = pkv_u32x4{0u, 0u, 0u, 0u};
      }
  }
  // A drafted value that is not finite belongs to the rows that see it and to no other; in the product it would reach all of the
  // tile as 0 * inf.  It is taken out there and added for its rows below.
  pkv_u32x4 odd[8];
  bool any_odd = false;
  if constexpr (DRAFT) {
    uint32_t found = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      odd[i] = v[i];
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const uint32_t x = v[i][d];
        if constexpr (BF16) {
          const uint32_t lo = (x & 0x7f80u) == 0x7f80u ? 0xffffu : 0u, hi = (x & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u;
          v[i][d] = x & ~(lo | hi), odd[i][d] = x & (lo | hi), found |= lo | hi;
        } else {
          const uint32_t bad = (x & 0x7f800000u) == 0x7f800000u ? 0xffffffffu : 0u;
          v[i][d] = x & ~bad, odd[i][d] = x & bad, found |= bad;
        }
      }
    }
    any_odd = __any(found != 0);
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    float s[W::kE];
    if constexpr (BF16) {
      pkv_f32x4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 4; ++c) s0 = mfma_bf16(k[c], w.q[t][c], s0), s1 = mfma_bf16(k[4 + c], w.q[t][c], s1);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] = e < 4 ? s0[e & 3] : s1[e & 3];
    } else {
      pkv_f32x4 s0 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 8; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) s0 = mfma_f32(__uint_as_float(k[c][i]), __uint_as_float(w.q[t][c][i]), s0);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] = s0[e];
    }
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < W::kE; ++e) {
      s[e] = (DRAFT ? sees(t, e) : tree_key(e, j) < count) ? s[e] * scale_log2e : -INFINITY;
      mx = fmaxf(mx, s[e]);
    }
    const float m_new = fmaxf(w.m[t], pkv_pair_max<32>(pkv_pair_max<16>(mx)));
    const float base = m_new == -INFINITY ? 0.f : m_new;  // a row that has seen nothing yet
    const float corr = __builtin_amdgcn_exp2f(w.m[t] - base);
    w.m[t] = m_new;
    float p[W::kE], sum = 0.f;
#pragma unroll
    for (int e = 0; e < W::kE; ++e) p[e] = __builtin_amdgcn_exp2f(s[e] - base), sum += p[e];
    w.l[t] = fmaf(w.l[t], corr, sum);
    float cr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) cr[i] = __shfl(corr, 4 * j + i, PKV_WAVE);
#pragma unroll
    for (int m = 0; m < 8; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) w.o[t][m][i] *= cr[i];
    if constexpr (BF16) {
      const pkv_u32x4 pa = {pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]), pack_bf16x2(p[4], p[5]), pack_bf16x2(p[6], p[7])};
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        const uint32_t sel = (m & 1) ? 0x07060302u : 0x05040100u;  // element m of each of the eight rows
        pkv_u32x4 b;
#pragma unroll
        for (int d = 0; d < 4; ++d) b[d] = __builtin_amdgcn_perm(v[2 * d + 1][m >> 1], v[2 * d][m >> 1], sel);
        w.o[t][m] = mfma_bf16(pa, b, w.o[t][m]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int m = 0; m < 8; ++m) w.o[t][m] = mfma_f32(p[e], __uint_as_float(v[2 * e + (m >> 2)][m & 3]), w.o[t][m]);
    }
    if constexpr (DRAFT) {
      if (any_odd) {  // the whole wave
#pragma unroll
        for (int e = 0; e < W::kE; ++e)
          for (int from = 0; from < 4; ++from) {  // key tree_key(e, from): its value in the lanes (n, from), row r's weight in lane (r, from)
            float x[8];
#pragma unroll
            for (int m = 0; m < 8; ++m) {
              if constexpr (BF16) {
                const uint32_t d = (uint32_t)__shfl((int)odd[e][m >> 1], n + 16 * from, PKV_WAVE);
                x[m] = __uint_as_float(m & 1 ? d & 0xffff0000u : d << 16);
              } else {
                x[m] = __uint_as_float((uint32_t)__shfl((int)odd[2 * e + (m >> 2)][m & 3], n + 16 * from, PKV_WAVE));
              }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float pr = __shfl(p[e], 4 * j + i + 16 * from, PKV_WAVE);
#pragma unroll
              for (int m = 0; m < 8; ++m)
                if (pr != 0.f && x[m] != 0.f) w.o[t][m][i] += pr * x[m];
            }
          }
      }
    }
  }
}

// grid (splits, tiles of 16 NT query rows, rows of (b, h))
template <bool BF16, int NT, bool INDEXED, typename SEGS>
__global__ __launch_bounds__(kTreeWaves * PKV_WAVE) void pkv_tree_partial_kernel(TreeCall a, SEGS segs) {
  using W = TreeWave<BF16, NT>;
  constexpr bool ONE = __is_same(SEGS, AttOne);
  const int split = blockIdx.x, n_splits = gridDim.x, r0 = blockIdx.y * 16 * NT, bh = blockIdx.z;
  const int b = bh / a.n_kv_heads, h = bh % a.n_kv_heads, rows = a.n_draft * a.group;
  const int tid = threadIdx.x, lane = tid & (PKV_WAVE - 1), wave = tid / PKV_WAVE, n = lane & 15, j = lane >> 4;
  constexpr int es = BF16 ? 2 : 4;

  uint32_t total = a.total;
  if (a.row_keys) {
    const int rk = a.row_keys[bh];
    total = rk <= 0 ? 0u : (uint32_t)rk < total ? (uint32_t)rk : total;
  }
  const uint32_t per_wave = a.per_split / kTreeWaves;  // a multiple of a step's keys
  const uint32_t k0 = (uint32_t)split * a.per_split + (uint32_t)wave * per_wave;
  const uint32_t k1 = k0 + per_wave < total ? k0 + per_wave : total;  // k1 <= k0: nothing for this wave

  W w;
  int token[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = r0 + 16 * t + n, rr = r < rows ? r : rows - 1;  // rows past the last repeat it and are not stored
    token[t] = rr / a.group;
    const char *qp = (const char *)a.q + ((int64_t)b * a.q_stride_b + (int64_t)token[t] * a.q_stride_t +
                                          (int64_t)(h * a.group + rr % a.group) * 128) * es + 16 * j;
#pragma unroll
    for (int c = 0; c < W::kQ; ++c) w.q[t][c] = *(const pkv_u32x4 *)(qp + 64 * c);
    w.m[t] = -INFINITY, w.l[t] = 0.f;
#pragma unroll
    for (int m = 0; m < 8; ++m) w.o[t][m] = pkv_f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const char *kbase = nullptr, *vbase = nullptr;
  if constexpr (ONE) {
    const int64_t slab = (int64_t)b * segs.stride_b + (int64_t)h * segs.stride_h;
    kbase = segs.k + slab, vbase = segs.v + slab;
  }
  AttPlace<ONE> mine;  // of key (block of 64) + lane
  for (uint32_t at = k0; at < k1; at += W::kKeys) {
    const int in_block = (int)(at - k0) & (PKV_WAVE - 1);
    if (in_block == 0) mine = att_place<INDEXED, W::kRow>(segs, bh, b, h, at + lane < k1 ? at + lane : k1 - 1);
    const int count = k1 - at < (uint32_t)W::kKeys ? (int)(k1 - at) : W::kKeys;
    tree_step<BF16, NT, false>(
        w,
        [&](int key, const char *&kp, const char *&vp) {
          if constexpr (ONE) {
            const uint64_t off = mine.from(in_block + key).off;
            kp = kbase + off, vp = vbase + off;
          } else {
            kp = mine.k_from(in_block + key), vp = mine.v_from(in_block + key);
          }
        },
        [](int, int) { return true; }, count, a.scale_log2e);
  }
  if (split == n_splits - 1) {  // the drafted tokens, a step's keys a wave in turn
    for (int u0 = wave * W::kKeys; u0 < a.n_draft; u0 += kTreeWaves * W::kKeys) {
      const int count = a.n_draft - u0 < W::kKeys ? a.n_draft - u0 : W::kKeys;
      tree_step<BF16, NT, true>(
          w,
          [&](int key, const char *&kp, const char *&vp) {
            const int64_t u = u0 + (key < count ? key : count - 1);
            kp = a.dk + (int64_t)b * a.dk_b + (int64_t)h * a.dk_h + u * a.dk_t;
            vp = a.dv + (int64_t)b * a.dv_b + (int64_t)h * a.dv_h + u * a.dv_t;
          },
          [&](int t, int e) {
            const int key = tree_key(e, j), u = u0 + (key < count ? key : count - 1);
            const bool on = a.mask ? a.mask[(int64_t)b * a.mask_b + (int64_t)token[t] * a.mask_t + u] != 0 : u <= token[t];
            return on && key < count;
          },
          count, a.scale_log2e);
    }
  }

  // the waves of the workgroup, a tile of rows at a time
  __shared__ float s_m[kTreeWaves][16], s_l[kTreeWaves][16];
  __shared__ alignas(16) float s_o[kTreeWaves][16][128 + 4];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const float l = pkv_pair_add<32>(pkv_pair_add<16>(w.l[t]));
    if (t > 0) __syncthreads();
    if (j == 0) s_m[wave][n] = w.m[t], s_l[wave][n] = l;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      *(float4 *)&s_o[wave][4 * j + i][8 * n] = float4{w.o[t][0][i], w.o[t][1][i], w.o[t][2][i], w.o[t][3][i]};
      *(float4 *)&s_o[wave][4 * j + i][8 * n + 4] = float4{w.o[t][4][i], w.o[t][5][i], w.o[t][6][i], w.o[t][7][i]};
    }
    __syncthreads();
    for (int e = tid; e < 16 * 128; e += kTreeWaves * PKV_WAVE) {
      const int r = e >> 7, d = e & 127, row = r0 + 16 * t + r;
      if (row >= rows) break;  // rows come in order
      float mx = s_m[0][r];
#pragma unroll
      for (int i = 1; i < kTreeWaves; ++i) mx = fmaxf(mx, s_m[i][r]);
      const float base = mx == -INFINITY ? 0.f : mx;
      float ls = 0.f, os = 0.f;
#pragma unroll
      for (int i = 0; i < kTreeWaves; ++i) {
        const float c = __builtin_amdgcn_exp2f(s_m[i][r] - base);
        ls = fmaf(s_l[i][r], c, ls), os = fmaf(s_o[i][r][d], c, os);
      }
      if (n_splits == 1) {
        const float y = ls == 0.f ? 0.f : os / ls;  // nothing seen
        const int64_t to = (((int64_t)b * a.n_draft + row / a.group) * a.n_kv_heads * a.group + h * a.group + row % a.group) * 128 + d;
        if constexpr (BF16) ((uint16_t *)a.out)[to] = pkv_f32_to_bf16_bits(y);
        else ((float *)a.out)[to] = y;
      } else {
        const int64_t at = ((int64_t)bh * n_splits + split) * rows + row;
        a.ws_o[at * 128 + d] = os;
        if (d == 0) a.ws_ml[at * 2] = mx, a.ws_ml[at * 2 + 1] = ls;
      }
    }
  }
}

// One wave a query row: lane l weighs split l and holds dims 2 l, 2 l + 1 of the output.
template <bool BF16>
__global__ __launch_bounds__(256) void pkv_tree_merge_kernel(const float *__restrict__ ws_o, const float *__restrict__ ws_ml, int n_splits,
                                                             int rows, int64_t n_rows, int n_draft, int group, int n_kv_heads,
                                                             void *__restrict__ out) {
  const int64_t at = (int64_t)blockIdx.x * 4 + threadIdx.x / PKV_WAVE;
  const int lane = pkv_lane();
  if (at >= n_rows) return;
  const int64_t bh = at / rows;
  const int row = (int)(at % rows), b = (int)(bh / n_kv_heads), h = (int)(bh % n_kv_heads);
  const int64_t first = bh * n_splits * rows + row;
  float m = -INFINITY, l = 0.f;
  if (lane < n_splits) m = ws_ml[(first + (int64_t)lane * rows) * 2], l = ws_ml[(first + (int64_t)lane * rows) * 2 + 1];
  const float mx = pkv_wave_max(m), base = mx == -INFINITY ? 0.f : mx;
  const float c = __builtin_amdgcn_exp2f(m - base), all = pkv_wave_sum(l * c);
  const float weight = all == 0.f ? 0.f : c / all;
  float x = 0.f, y = 0.f;
  for (int s = 0; s < n_splits; ++s) {
    const float2 o = *(const float2 *)(ws_o + (first + (int64_t)s * rows) * 128 + 2 * lane);
    const float f = __shfl(weight, s, PKV_WAVE);
    x = fmaf(o.x, f, x), y = fmaf(o.y, f, y);
  }
  const int64_t to = (((int64_t)b * n_draft + row / group) * n_kv_heads * group + h * group + row % group) * 128 + 2 * lane;
  if constexpr (BF16) *(uint32_t *)((uint16_t *)out + to) = pack_bf16x2(x, y);
  else *(float2 *)((float *)out + to) = float2{x, y};
}

struct TreePlan {
  int nt, row_tiles, n_splits;
  uint32_t per_split;
};

TreePlan tree_plan(int dtype, int bs, int n_kv_heads, int rows, int64_t total) {
  TreePlan p;
  const bool bf = dtype == PKV_DTYPE_BF16;
  p.nt = 1;
  p.row_tiles = (rows + 16 * p.nt - 1) / (16 * p.nt);
  const int step = kTreeWaves * (bf ? 32 : 16);
  int64_t s = 1024 / ((int64_t)bs * n_kv_heads * p.row_tiles), most = (total + step - 1) / step;
  if (s > most) s = most;
  if (s > kTreeMaxSplits) s = kTreeMaxSplits;
  if (s < 1) s = 1;
  int64_t per = (total + s - 1) / s;
  per = (per + step - 1) / step * step;
  if (per < step) per = step;
  p.per_split = (uint32_t)per;
  p.n_splits = (int)(total > 0 ? (total + per - 1) / per : 1);
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
  c.total = (uint32_t)total, c.per_split = p.per_split, c.row_keys = a->row_keys;
  c.dk = (const char *)a->draft_k, c.dk_b = a->dk_stride_b * es, c.dk_h = a->dk_stride_h * es, c.dk_t = a->dk_stride_t * es;
  c.dv = (const char *)a->draft_v, c.dv_b = a->dv_stride_b * es, c.dv_h = a->dv_stride_h * es, c.dv_t = a->dv_stride_t * es;
  c.mask = a->mask, c.mask_b = a->mask_stride_b, c.mask_t = a->mask_stride_t;
  c.scale_log2e = a->scale * 1.4426950408889634f;
  c.ws_o = (float *)a->ws, c.ws_ml = c.ws_o ? c.ws_o + n_rows * p.n_splits * 128 : nullptr;
  c.out = a->out;
  AttOne one;
  const bool is_one = as_one_tensor(sg, (int)es, one);
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)p.n_splits, (unsigned)p.row_tiles, (unsigned)(a->bs * a->n_kv_heads)), block(kTreeWaves * PKV_WAVE);
#define PKV_TREE(BF, NT, IDX, S) hipLaunchKernelGGL((pkv_tree_partial_kernel<BF, NT, IDX, decltype(S)>), grid, block, 0, s, c, S)
#define PKV_TREE_S(BF, NT)                                                            \
  do {                                                                                \
    if (is_one) { if (indexed) PKV_TREE(BF, NT, true, one); else PKV_TREE(BF, NT, false, one); } \
    else { if (indexed) PKV_TREE(BF, NT, true, sg); else PKV_TREE(BF, NT, false, sg); }          \
  } while (0)
  if (bf) PKV_TREE_S(true, 1);
  else PKV_TREE_S(false, 1);
#undef PKV_TREE_S
#undef PKV_TREE
  PKV_LAUNCH_CHECK("pkv_tree_partial_kernel");
  if (p.n_splits == 1) return PKV_OK;
  const dim3 merge((unsigned)((n_rows + 3) / 4));
  if (bf)
    hipLaunchKernelGGL(pkv_tree_merge_kernel<true>, merge, dim3(256), 0, s, (const float *)c.ws_o, (const float *)c.ws_ml, p.n_splits, rows,
                       n_rows, a->n_draft, a->group, a->n_kv_heads, a->out);
  else
    hipLaunchKernelGGL(pkv_tree_merge_kernel<false>, merge, dim3(256), 0, s, (const float *)c.ws_o, (const float *)c.ws_ml, p.n_splits, rows,
                       n_rows, a->n_draft, a->group, a->n_kv_heads, a->out);
  PKV_LAUNCH_CHECK("pkv_tree_merge_kernel");
  return PKV_OK;
}
