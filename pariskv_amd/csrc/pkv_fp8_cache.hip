// A K/V cache in eight bits: rows quantised as they are written, and read back.  (No counterpart in the reference, whose caches are bf16.)
//
// Row r of head h of sequence b is 128 e4m3 codes; the rows of a block of 16, 32, 64 or 128 share one scale each for K and for V
// (pkv_fp8.h).  Rows written behind others in a block keep those: the scale is the larger (in magnitude) of what stands there and what the new rows
// need, and where it grows the older rows' codes are rounded again under it.  Rows from the block's first one on start it anew.
#include "pkv_fp8.h"

namespace {

constexpr int kStoreThreads = 256, kStoreRows = kStoreThreads / 16;  // 16 lanes a row, eight values each

struct StoreArgs {
  const char *x[2];  // K, V
  int64_t stride_b[2], stride_t[2], stride_h[2];  // bytes
  uint8_t *codes[2];
  float *scales[2];
  const int32_t *start, *length;  // or null
  int64_t start0, capacity, n_blocks;
  int n_tokens, n_heads;
};

// One workgroup a block of rows of K or of V: everything in registers, one reduction, no second look at the input.  The bytes bound it: 8192 tokens x
// 8 heads (50 MB) 10.4 us, 4.85 TB/s (11.6 with codes that the caches keep); one token 3.4 us, a launch.
// grid (blocks that the rows may reach into, (b, h), K or V)
template <bool BF16, int BLOCK>
__global__ __launch_bounds__(kStoreThreads) void pkv_fp8_store_kernel(StoreArgs a) {
  constexpr int kIter = BLOCK / kStoreRows;
  __shared__ uint32_t s_top[kStoreThreads / PKV_WAVE];
  const int tid = threadIdx.x, kv = blockIdx.z, b = (unsigned)blockIdx.y / (unsigned)a.n_heads, h = blockIdx.y - b * a.n_heads;
  const int64_t start = a.start ? a.start[b] : a.start0;
  int n = a.length ? a.length[b] : a.n_tokens;
  n = n < a.n_tokens ? n : a.n_tokens;
  if (start < 0 || start >= a.capacity || n <= 0) return;  // nothing of this sequence (the whole workgroup)
  if (n > a.capacity - start) n = (int)(a.capacity - start);
  const int64_t block = start / BLOCK + blockIdx.x, row0 = block * BLOCK;
  if (row0 >= start + n) return;
  const int64_t bh = blockIdx.y;
  uint8_t *const codes = a.codes[kv] + (bh * a.capacity + row0) * 128 + (tid & 15) * 8;
  float *const scale_at = a.scales[kv] + bh * a.n_blocks + block;
  const int before = start > row0 ? (int)(start - row0) : 0;  // rows of the block that are there already
  const float was = before ? *scale_at : 0.f;

  float x[kIter][8];
  uint32_t top = 0;
  const char *const src = a.x[kv] + b * a.stride_b[kv] + h * a.stride_h[kv] + (tid & 15) * (BF16 ? 16 : 32);
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int64_t t = row0 + i * kStoreRows + (tid >> 4) - start;
    if (t >= 0 && t < n) {
      fp8_load8<BF16>(src + t * a.stride_t[kv], x[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t m = fp8_magnitude(x[i][e]);
        top = m > top ? m : top;
      }
    }
  }
  top = pkv_wave_max(top);
  if (pkv_lane() == 0) s_top[tid / PKV_WAVE] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kStoreThreads / PKV_WAVE; ++w) top = s_top[w] > top ? s_top[w] : top;
  const float need = fp8_pow2(fp8_exponent(top)), scale = fabsf(was) > need ? was : need;  // a scale that the caller set may be negative
  const float inv = 1.0f / scale;  // exact where the scale is a power of two, as it is unless the caller set it
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int r = i * kStoreRows + (tid >> 4);
    const int64_t t = row0 + r - start;
    if (t >= 0 && t < n) __builtin_nontemporal_store(fp8_codes8(x[i], inv), (pkv_u32x2 *)(codes + r * 128));
    else if (r < before && was != scale) {
      const pkv_u32x2 old = *(const pkv_u32x2 *)(codes + r * 128);
      float y[8];
      fp8_values4(old.x, y), fp8_values4(old.y, y + 4);
      *(pkv_u32x2 *)(codes + r * 128) = fp8_codes8(y, was * inv);
    }
  }
  if (tid == 0) *scale_at = scale;
}

// Rows of K and V as values: 16 lanes a row, eight codes each; kReadUnroll rows a lane under way.  The bytes bound it: 32 768 rows x 8 heads to bf16
// (201 MB) 31 us, 6.5 TB/s, 42 with stores that the caches keep; 8968 rows x 24 heads to fp32 (275 MB) 41.4 us, and 61.8 with 32 bytes a lane side by side;
// 515 selected rows x 12 to fp32 5.4 us, two memory round trips.
struct ReadArgs {
  const uint8_t *codes[2];
  const float *scales[2];
  const int64_t *idx;  // or null
  int64_t idx_stride, row0, n_rows, capacity, n_blocks, total;  // total: rows of all (b, h)
  char *out[2];
  int64_t out_b[2], out_h[2], out_row[2];  // bytes
  int n_heads, lg_block;
};
constexpr int kReadThreads = 256, kReadUnroll = 4;
typedef float fp8_f32x4 __attribute__((ext_vector_type(4)));

template <bool BF16>
__global__ __launch_bounds__(kReadThreads) void pkv_fp8_read_kernel(ReadArgs a) {
  const int tid = threadIdx.x, kv = blockIdx.y, lane = tid & 15;
  const int64_t first = (int64_t)blockIdx.x * (kReadThreads / 16 * kReadUnroll) + (tid >> 4);
  pkv_u32x2 w[kReadUnroll];
  float scale[kReadUnroll];
#pragma unroll
  for (int u = 0; u < kReadUnroll; ++u) {
    const int64_t at = first + u * (kReadThreads / 16);
    w[u] = pkv_u32x2{0u, 0u}, scale[u] = 0.f;
    if (at < a.total) {
      const int64_t bh = at / a.n_rows, i = at - bh * a.n_rows, pick = a.idx ? a.idx[bh * a.idx_stride + i] : i, r = a.row0 + pick;
      if ((uint64_t)pick < (uint64_t)(a.capacity - a.row0)) {  // a selected row that is not there: zeros
        const uint8_t *const from = a.codes[kv] + (bh * a.capacity + r) * 128;
        if constexpr (BF16) w[u] = *(const pkv_u32x2 *)(from + lane * 8);
        else w[u] = pkv_u32x2{*(const uint32_t *)(from + lane * 4), *(const uint32_t *)(from + 64 + lane * 4)};  // stores of 16 bytes side by side
        scale[u] = a.scales[kv][bh * a.n_blocks + (r >> a.lg_block)];
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kReadUnroll; ++u) {
    const int64_t at = first + u * (kReadThreads / 16);
    if (at >= a.total) continue;
    const int64_t bh = at / a.n_rows, i = at - bh * a.n_rows, b = bh / a.n_heads, h = bh - b * a.n_heads;
    char *const to = a.out[kv] + b * a.out_b[kv] + h * a.out_h[kv] + i * a.out_row[kv] + lane * 16;
    float x[8];
    fp8_values4(w[u].x, x), fp8_values4(w[u].y, x + 4);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= scale[u];
    if constexpr (BF16) {
      pkv_u32x4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = (uint32_t)pkv_f32_to_bf16_bits(x[2 * e]) | ((uint32_t)pkv_f32_to_bf16_bits(x[2 * e + 1]) << 16);
      __builtin_nontemporal_store(o, (pkv_u32x4 *)to);
    } else {
      __builtin_nontemporal_store(fp8_f32x4{x[0], x[1], x[2], x[3]}, (fp8_f32x4 *)to);
      __builtin_nontemporal_store(fp8_f32x4{x[4], x[5], x[6], x[7]}, (fp8_f32x4 *)(to + 256));
    }
  }
}

}  // namespace

int pkv_fp8_kv_check(const pkv_fp8_kv *c, const char *who) {
  PKV_REQUIRE(c && c->k && c->v && c->k_scale && c->v_scale, "%s: null cache", who);
  PKV_REQUIRE(c->bs > 0 && c->n_kv_heads > 0 && (int64_t)c->bs * c->n_kv_heads <= 65535 && c->capacity > 0 && c->capacity <= PKV_FP8_MAX_ROWS,
              "%s: bad cache bs=%d kv_heads=%d capacity=%lld", who, c->bs, c->n_kv_heads, (long long)c->capacity);
  PKV_REQUIRE(c->block == 16 || c->block == 32 || c->block == 64 || c->block == 128, "%s: blocks of 16, 32, 64 or 128 rows (got %d)", who, c->block);
  PKV_REQUIRE(c->capacity % c->block == 0, "%s: the capacity must be a multiple of the block", who);
  PKV_REQUIRE(pkv_aligned(c->k, 16) && pkv_aligned(c->v, 16) && pkv_aligned(c->k_scale, 4) && pkv_aligned(c->v_scale, 4),
              "%s: 16-byte aligned codes required", who);
  return PKV_OK;
}

extern "C" int pkv_fp8_store(const pkv_fp8_kv *cache, const void *k, const void *v, int dtype, int64_t n_tokens, int64_t k_stride_b,
                             int64_t k_stride_t, int64_t k_stride_h, int64_t v_stride_b, int64_t v_stride_t, int64_t v_stride_h,
                             int64_t start, const int32_t *starts, const int32_t *lengths, void *stream) {
  if (const int rc = pkv_fp8_kv_check(cache, "pkv_fp8_store")) return rc;
  PKV_REQUIRE(k && v, "pkv_fp8_store: null pointer");
  PKV_REQUIRE(dtype == PKV_DTYPE_F32 || dtype == PKV_DTYPE_BF16, "unknown dtype %d", dtype);
  PKV_REQUIRE(n_tokens > 0 && n_tokens <= cache->capacity, "pkv_fp8_store: 1..capacity tokens (got %lld)", (long long)n_tokens);
  PKV_REQUIRE(starts || (start >= 0 && start <= cache->capacity - n_tokens), "pkv_fp8_store: rows %lld.. (%lld of them) of %lld",
              (long long)start, (long long)n_tokens, (long long)cache->capacity);
  PKV_REQUIRE(pkv_aligned(k, 16) && pkv_aligned(v, 16) && pkv_aligned(starts, 4) && pkv_aligned(lengths, 4), "pkv_fp8_store: 16-byte aligned rows required");
  const int64_t es = dtype == PKV_DTYPE_BF16 ? 2 : 4;
  const int64_t strides[] = {k_stride_b, k_stride_t, k_stride_h, v_stride_b, v_stride_t, v_stride_h};
  for (int64_t s : strides) PKV_REQUIRE(s * es % 16 == 0, "pkv_fp8_store: strides must be multiples of 16 bytes");
  StoreArgs a;
  a.x[0] = (const char *)k, a.x[1] = (const char *)v;
  a.stride_b[0] = k_stride_b * es, a.stride_t[0] = k_stride_t * es, a.stride_h[0] = k_stride_h * es;
  a.stride_b[1] = v_stride_b * es, a.stride_t[1] = v_stride_t * es, a.stride_h[1] = v_stride_h * es;
  a.codes[0] = cache->k, a.codes[1] = cache->v, a.scales[0] = cache->k_scale, a.scales[1] = cache->v_scale;
  a.start = starts, a.length = lengths, a.start0 = start, a.capacity = cache->capacity, a.n_blocks = cache->capacity / cache->block;
  a.n_tokens = (int)n_tokens, a.n_heads = cache->n_kv_heads;
  // where the starts are not known here, as many blocks as rows at the worst of them reach into
  const int64_t blocks = starts ? (n_tokens + cache->block - 2) / cache->block + 1 : (start + n_tokens - 1) / cache->block - start / cache->block + 1;
  const dim3 grid((unsigned)blocks, (unsigned)(cache->bs * cache->n_kv_heads), 2);
#define PKV_STORE(BF)                                                                                                          \
  do {                                                                                                                         \
    if (cache->block == 16) hipLaunchKernelGGL((pkv_fp8_store_kernel<BF, 16>), grid, dim3(kStoreThreads), 0, (hipStream_t)stream, a);       \
    else if (cache->block == 32) hipLaunchKernelGGL((pkv_fp8_store_kernel<BF, 32>), grid, dim3(kStoreThreads), 0, (hipStream_t)stream, a);  \
    else if (cache->block == 64) hipLaunchKernelGGL((pkv_fp8_store_kernel<BF, 64>), grid, dim3(kStoreThreads), 0, (hipStream_t)stream, a);  \
    else hipLaunchKernelGGL((pkv_fp8_store_kernel<BF, 128>), grid, dim3(kStoreThreads), 0, (hipStream_t)stream, a);                         \
  } while (0)
  if (dtype == PKV_DTYPE_BF16) PKV_STORE(true);
  else PKV_STORE(false);
#undef PKV_STORE
  PKV_LAUNCH_CHECK("pkv_fp8_store_kernel");
  return PKV_OK;
}

extern "C" int pkv_fp8_read(const pkv_fp8_kv *cache, int64_t row0, int64_t n_rows, const int64_t *idx, int64_t idx_stride, int dtype, void *out_k,
                            void *out_v, int64_t ok_stride_b, int64_t ok_stride_h, int64_t ok_stride_row, int64_t ov_stride_b, int64_t ov_stride_h,
                            int64_t ov_stride_row, void *stream) {
  if (const int rc = pkv_fp8_kv_check(cache, "pkv_fp8_read")) return rc;
  PKV_REQUIRE(out_k && out_v, "pkv_fp8_read: null pointer");
  PKV_REQUIRE(dtype == PKV_DTYPE_F32 || dtype == PKV_DTYPE_BF16, "unknown dtype %d", dtype);
  PKV_REQUIRE(n_rows > 0 && n_rows < ((int64_t)1 << 31) && row0 >= 0 && row0 < cache->capacity && (idx || row0 + n_rows <= cache->capacity) &&
                  (!idx || idx_stride >= n_rows),
              "pkv_fp8_read: rows %lld.. (%lld of them) of %lld", (long long)row0, (long long)n_rows, (long long)cache->capacity);
  PKV_REQUIRE(pkv_aligned(out_k, 16) && pkv_aligned(out_v, 16) && pkv_aligned(idx, 8), "pkv_fp8_read: 16-byte aligned rows required");
  const int64_t es = dtype == PKV_DTYPE_BF16 ? 2 : 4;
  const int64_t strides[] = {ok_stride_b, ok_stride_h, ok_stride_row, ov_stride_b, ov_stride_h, ov_stride_row};
  for (int64_t s : strides) PKV_REQUIRE(s * es % 16 == 0, "pkv_fp8_read: strides must be multiples of 16 bytes");
  ReadArgs a;
  a.codes[0] = cache->k, a.codes[1] = cache->v, a.scales[0] = cache->k_scale, a.scales[1] = cache->v_scale;
  a.idx = idx, a.idx_stride = idx_stride, a.row0 = row0, a.n_rows = n_rows, a.capacity = cache->capacity;
  a.n_blocks = cache->capacity / cache->block, a.total = (int64_t)cache->bs * cache->n_kv_heads * n_rows;
  a.out[0] = (char *)out_k, a.out[1] = (char *)out_v;
  a.out_b[0] = ok_stride_b * es, a.out_h[0] = ok_stride_h * es, a.out_row[0] = ok_stride_row * es;
  a.out_b[1] = ov_stride_b * es, a.out_h[1] = ov_stride_h * es, a.out_row[1] = ov_stride_row * es;
  a.n_heads = cache->n_kv_heads, a.lg_block = __builtin_ctz(cache->block);
  const int64_t per = kReadThreads / 16 * kReadUnroll, groups = (a.total + per - 1) / per;
  PKV_REQUIRE(groups < ((int64_t)1 << 31), "pkv_fp8_read: too many rows");
  const dim3 grid((unsigned)groups, 2);
  if (dtype == PKV_DTYPE_BF16) hipLaunchKernelGGL(pkv_fp8_read_kernel<true>, grid, dim3(kReadThreads), 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL(pkv_fp8_read_kernel<false>, grid, dim3(kReadThreads), 0, (hipStream_t)stream, a);
  PKV_LAUNCH_CHECK("pkv_fp8_read_kernel");
  return PKV_OK;
}
