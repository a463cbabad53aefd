// Rows in eight bits, each with a scale of its own (pkv_fp8.h), as the products with eight-bit matrices take them: the
// root-mean-square norm with the residual's addition in front (pkv_add_rmsnorm with eight-bit rows for its norm), or rows as they are.
// (No counterpart in the reference, whose activations stay bf16.)
//
// A row is read once and held in registers; the sum of its squares is a sum of 64-bit numbers, where those of bf16 numbers are exact
// (16 bits of mantissa each): what a code rounds to does not depend on the order.
#include "pkv_fp8.h"

namespace {

constexpr int kMaxWidth = 16384, kReps = 2, E = 8;  // E: neighbouring elements a thread takes at a time

__device__ __forceinline__ double fp8_wave_sum(double v) {
#pragma unroll
  for (int m = 1; m < PKV_WAVE; m <<= 1) v += __shfl_xor(v, m, PKV_WAVE);
  return v;
}

struct RowsArgs {
  const char *x;
  const uint16_t *residual, *weight;
  int64_t x_stride, code_stride;  // bytes
  double eps;
  int width, padded;
  uint16_t *out_sum;
  uint8_t *codes;
  float *scales;
};

// Eight elements at any address of whole elements, or the `left` of them that the row still has with zeros behind them.  The memory takes 16-byte
// accesses at any alignment: 4096 rows of 4095 with the residual take 28.6 us (element by element: 52.2), of 4096 23.4.
template <bool BF16>
__device__ __forceinline__ void load_any(const char *p, int left, float (&v)[E]) {
  if (left >= E) {
    struct __attribute__((packed)) Raw {
      uint32_t w[BF16 ? 4 : 8];
    } raw;
    __builtin_memcpy(&raw, p, sizeof raw);
#pragma unroll
    for (int e = 0; e < E; ++e)
      v[e] = __uint_as_float(!BF16 ? raw.w[BF16 ? 0 : e] : e & 1 ? raw.w[e / 2] & 0xffff0000u : raw.w[e / 2] << 16);
    return;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = e >= left ? 0.f : BF16 ? pkv_bf16_bits_to_f32(((const uint16_t *)p)[e]) : ((const float *)p)[e];
}

// ALIGNED: whole 16-byte vectors everywhere.  THREADS: as many as a row takes with eight elements a thread, once or twice (kReps).  us, with the residual, 256 threads and
// as often as it takes / this: 16384 x 1024 29.9 / 22.1 (5.3 TB/s; a copy reaches 4.8), 20000 x 200 29.9 / 13.5, 4096 x 4096 22.9, 2048 x 8192 25.8 / 23.1, 1 x 16384 8.3 / 5.4.
template <bool NORM, bool BF16, bool ALIGNED, int THREADS>
__global__ __launch_bounds__(THREADS) void pkv_fp8_rows_kernel(RowsArgs a) {
  constexpr int kRowThreads = THREADS, kRowWaves = THREADS / PKV_WAVE;
  __shared__ double s_sum[kRowWaves];
  __shared__ uint32_t s_top[kRowWaves];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const char *const x = a.x + row * a.x_stride;
  float v[kReps][E], w[NORM ? kReps : 1][E];
  double sum = 0.0;
  uint32_t top = 0;
#pragma unroll
  for (int r = 0; r < kReps; ++r) {
    const int at = (r * kRowThreads + tid) * E, left = a.width - at;
    if (left <= 0) continue;
    const char *const from = x + (int64_t)at * (BF16 ? 2 : 4);
    if constexpr (ALIGNED) fp8_load8<BF16>(from, v[r]);
    else load_any<BF16>(from, left, v[r]);
    if constexpr (NORM) {
      if constexpr (ALIGNED) fp8_load8<true>((const char *)(a.weight + at), w[r]);
      else load_any<true>((const char *)(a.weight + at), left, w[r]);
      if (a.residual) {
        const char *const res = (const char *)(a.residual + row * a.width + at);
        float add[E];
        if constexpr (ALIGNED) fp8_load8<true>(res, add);
        else load_any<true>(res, left, add);
#pragma unroll
        for (int e = 0; e < E; ++e) v[r][e] = pkv_bf16_round(v[r][e] + add[e]);
      }
      if (a.out_sum) {
        uint16_t *const to = a.out_sum + row * a.width + at;
        pkv_u32x4 o;
#pragma unroll
        for (int p = 0; p < 4; ++p) o[p] = (__float_as_uint(v[r][2 * p]) >> 16) | (__float_as_uint(v[r][2 * p + 1]) & 0xffff0000u);
        if constexpr (ALIGNED) {
          __builtin_nontemporal_store(o, (pkv_u32x4 *)to);
        } else if (left >= E) {
          __builtin_memcpy(to, &o, sizeof o);
        } else {
#pragma unroll
          for (int e = 0; e < E - 1; ++e)
            if (e < left) to[e] = (uint16_t)(__float_as_uint(v[r][e]) >> 16);
        }
      }
#pragma unroll
      for (int e = 0; e < E; ++e) sum += (double)v[r][e] * (double)v[r][e];
    }
  }
  if constexpr (NORM) {
    sum = fp8_wave_sum(sum);
    if (pkv_lane() == 0) s_sum[tid / PKV_WAVE] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < kRowWaves; ++i) sum += s_sum[i];
    const float inv = (float)(1.0 / sqrt(sum / (double)a.width + a.eps));
#pragma unroll
    for (int r = 0; r < kReps; ++r) {
      const int left = a.width - (r * kRowThreads + tid) * E;
      if (left <= 0) continue;
#pragma unroll
      for (int e = 0; e < E; ++e) v[r][e] = ALIGNED || e < left ? v[r][e] * inv * w[r][e] : 0.f;  // past the row zeros, also where inv is a NaN
    }
  }
#pragma unroll
  for (int r = 0; r < kReps; ++r) {
    if ((r * kRowThreads + tid) * E >= a.width) continue;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t m = fp8_magnitude(v[r][e]);
      top = m > top ? m : top;
    }
  }
  top = pkv_wave_max(top);
  if (pkv_lane() == 0) s_top[tid / PKV_WAVE] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRowWaves; ++i) top = s_top[i] > top ? s_top[i] : top;
  const int e2 = fp8_exponent(top);
  const float shrink = fp8_pow2(-e2);
  uint8_t *const codes = a.codes + row * a.code_stride;
#pragma unroll
  for (int r = 0; r < kReps; ++r) {
    const int at = (r * kRowThreads + tid) * E;
    if (at >= a.width) continue;
    *(pkv_u32x2 *)(codes + at) = fp8_codes8(v[r], shrink);  // zeros behind the row's last element: a row holds whole chunks of 128
  }
  const int pad = (a.width + E - 1) / E * E + tid * E;
  if (pad < a.padded) *(pkv_u32x2 *)(codes + pad) = pkv_u32x2{0, 0};
  if (tid == 0) a.scales[row] = fp8_pow2(e2);
}

template <bool NORM, bool BF16, bool ALIGNED>
int launch_as(const RowsArgs &a, int64_t rows, hipStream_t s) {
  // Few rows: eight elements a thread once, up to 512 threads.  us, with the residual, once / twice: 1 x 4096 3.4 / 3.8, 300 x 1024 3.6 / 4.0, 700 x 4096 7.5 / 7.2,
  // 300 x 8192 8.1 / 7.0.
  const int threads = (a.width + E - 1) / E, most = rows <= 512 && threads <= 512 ? threads : (threads + kReps - 1) / kReps;
#define PKV_ROWS(THREADS) \
  hipLaunchKernelGGL((pkv_fp8_rows_kernel<NORM, BF16, ALIGNED, THREADS>), dim3((unsigned)rows), dim3(THREADS), 0, s, a)
  if (most <= 64) PKV_ROWS(64);
  else if (most <= 128) PKV_ROWS(128);
  else if (most <= 256) PKV_ROWS(256);
  else if (most <= 512) PKV_ROWS(512);
  else PKV_ROWS(1024);
#undef PKV_ROWS
  static_assert(1024 * E * kReps == kMaxWidth, "no wider row");
  PKV_LAUNCH_CHECK("pkv_fp8_rows_kernel");
  return PKV_OK;
}
template <bool NORM, bool BF16>
int launch(RowsArgs a, int64_t rows, bool aligned, hipStream_t s) {
  constexpr int64_t kMost = (int64_t)1 << 21;  // rows of a launch, which has fewer than 2^32 threads; the next ones begin at a multiple of 16 bytes where these do
  for (;;) {
    const int64_t n = rows < kMost ? rows : kMost;
    if (const int rc = aligned ? launch_as<NORM, BF16, true>(a, n, s) : launch_as<NORM, BF16, false>(a, n, s)) return rc;
    if ((rows -= n) == 0) return PKV_OK;
    a.x += n * a.x_stride, a.codes += n * a.code_stride, a.scales += n;
    if (a.residual) a.residual += n * a.width;
    if (a.out_sum) a.out_sum += n * a.width;
  }
}

int shape_ok(const char *who, int64_t rows, int64_t width, const void *codes, int64_t code_stride, const void *scales) {
  PKV_REQUIRE(rows > 0 && rows < ((int64_t)1 << 31) && width > 0 && width <= kMaxWidth, "%s: 1..%d columns, at least one row (got %lld x %lld)", who,
              kMaxWidth, (long long)rows, (long long)width);
  PKV_REQUIRE(pkv_aligned(codes, 16) && code_stride % 16 == 0 && code_stride >= (int64_t)pkv_align_up((size_t)width, 128) && pkv_aligned(scales, 4),
              "%s: rows of codes must be 16-byte aligned and hold whole chunks of 128", who);
  return PKV_OK;
}

}  // namespace

extern "C" int pkv_add_rmsnorm_fp8(const void *x, const void *residual, const void *weight, double eps, int64_t rows, int64_t width,
                                   void *out_sum, uint8_t *codes, int64_t code_stride, float *scales, void *stream) {
  PKV_REQUIRE(x && weight && codes && scales, "pkv_add_rmsnorm_fp8: null pointer");
  if (const int rc = shape_ok("pkv_add_rmsnorm_fp8", rows, width, codes, code_stride, scales)) return rc;
  PKV_REQUIRE(pkv_aligned(x, 2) && pkv_aligned(residual, 2) && pkv_aligned(weight, 2) && pkv_aligned(out_sum, 2), "pkv_add_rmsnorm_fp8: bf16 operands");
  RowsArgs a;
  a.x = (const char *)x, a.residual = (const uint16_t *)residual, a.weight = (const uint16_t *)weight, a.x_stride = width * 2, a.eps = eps;
  a.width = (int)width, a.padded = (int)pkv_align_up((size_t)width, 128), a.out_sum = (uint16_t *)out_sum, a.codes = codes, a.code_stride = code_stride, a.scales = scales;
  const bool aligned = width % 8 == 0 && pkv_aligned(x, 16) && pkv_aligned(residual, 16) && pkv_aligned(weight, 16) && pkv_aligned(out_sum, 16);
  return launch<true, true>(a, rows, aligned, (hipStream_t)stream);
}

extern "C" int pkv_fp8_rows(const void *x, int dtype, int64_t x_stride, int64_t rows, int64_t width, uint8_t *codes, int64_t code_stride, float *scales,
                            void *stream) {
  PKV_REQUIRE(x && codes && scales, "pkv_fp8_rows: null pointer");
  PKV_REQUIRE(dtype == PKV_DTYPE_F32 || dtype == PKV_DTYPE_BF16, "unknown dtype %d", dtype);
  if (const int rc = shape_ok("pkv_fp8_rows", rows, width, codes, code_stride, scales)) return rc;
  const int64_t es = dtype == PKV_DTYPE_BF16 ? 2 : 4;
  PKV_REQUIRE(pkv_aligned(x, es) && x_stride >= 0, "pkv_fp8_rows: rows of whole elements");
  RowsArgs a;
  memset(&a, 0, sizeof a);
  a.x = (const char *)x, a.x_stride = x_stride * es, a.width = (int)width, a.padded = (int)pkv_align_up((size_t)width, 128);
  a.codes = codes, a.code_stride = code_stride, a.scales = scales;
  const bool aligned = width % 8 == 0 && x_stride * es % 16 == 0 && pkv_aligned(x, 16);
  if (dtype == PKV_DTYPE_BF16) return launch<false, true>(a, rows, aligned, (hipStream_t)stream);
  return launch<false, false>(a, rows, aligned, (hipStream_t)stream);
}
