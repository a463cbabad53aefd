// Products of few rows with matrices of 4-bit weights and group scales: the projections of a decode step, or of a step over
// several drafted tokens, at a quarter of the bytes.  (No counterpart in the reference, whose projections are bf16 GEMMs,
// model_hub/qwen.py:327-383.)
//
// y[m][n] = sum_k x[m][k] s[n][g(k)] (q[n][k] - z[n][g(k)]) = sum_g s[n][g] (sum_k x (16 + q) - (16 + z[n][g]) sum_k x)
//
// 16 + q is a bf16 number that a rotation, an AND and an OR make of a code (the code goes into the upper four mantissa bits of 16.0;
// 16 is the smallest number whose mantissa has room for it, so that the difference cancels as little as it can): 7 vector instructions for 8
// weights.  Both sums over k come from v_mfma_f32_16x16x32_bf16, the second with a matrix of ones, which leaves sum x in the
// registers where it is needed; products of bf16 numbers are exact in fp32, as are the codes, and sums are fp32.
#include "pkv_common.h"

namespace {

typedef __bf16 w4_bf16x8 __attribute__((ext_vector_type(8)));
typedef float w4_f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTileRows = 16, kTileCols = 128, kTileBytes = 1024;
constexpr int kWaves = 4;

__device__ __forceinline__ w4_f32x4 w4_mfma(pkv_u32x4 a, pkv_u32x4 b, w4_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(w4_bf16x8, a), __builtin_bit_cast(w4_bf16x8, b), c, 0, 0, 0);
}

// The eight codes of a word as bf16 numbers 16 + q, in column order.
__device__ __forceinline__ pkv_u32x4 w4_expand(uint32_t w) {
  const uint32_t keep = 0x00780078u, sixteen = 0x41804180u;
  return pkv_u32x4{(w & keep) | sixteen, ((w >> 4) & keep) | sixteen, ((w >> 8) & keep) | sixteen,
                   (__builtin_amdgcn_alignbit(w, w, 12) & keep) | sixteen};
}

struct W4Matrix {
  const char *tiles;      // [row tile][chunk of 128 columns] of kTileBytes
  const uint32_t *words;  // [row tile][group][16]
};

// grid (row tiles, tiles of 16 MT rows of x), four waves that take the chunks in turn and meet in LDS.
template <int MT, int G, bool GATED>
__global__ __launch_bounds__(kWaves * PKV_WAVE) void pkv_w4_kernel(const uint16_t *__restrict__ x, int64_t x_stride, int64_t rows,
                                                                   W4Matrix wa, W4Matrix wb, int64_t n_out, int64_t k, int chunks,
                                                                   const uint16_t *__restrict__ bias, void *__restrict__ y,
                                                                   int out_f32) {
  constexpr int kParts = GATED ? 2 : 1, kGroups = kTileCols / G, kSteps = G / 32;
  const int lane = threadIdx.x & (PKV_WAVE - 1), wave = threadIdx.x / PKV_WAVE, n = lane & 15, j = lane >> 4;
  const int64_t tile = blockIdx.x, m0 = (int64_t)blockIdx.y * 16 * MT;
  const pkv_u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u}, none = {0u, 0u, 0u, 0u};
  w4_f32x4 tot[kParts][MT];
#pragma unroll
  for (int p = 0; p < kParts; ++p)
#pragma unroll
    for (int t = 0; t < MT; ++t) tot[p][t] = w4_f32x4{0.f, 0.f, 0.f, 0.f};
  for (int c = wave; c < chunks; c += kWaves) {
    pkv_u32x4 w[kParts], xv[MT][4], sc[kParts][kGroups];
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      const W4Matrix &m = p ? wb : wa;
      w[p] = __builtin_nontemporal_load((const pkv_u32x4 *)(m.tiles + (tile * chunks + c) * kTileBytes) + lane);
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
        sc[p][g] = *(const pkv_u32x4 *)(m.words + ((tile * chunks + c) * kGroups + g) * kTileRows + 4 * j);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int64_t row = m0 + 16 * t + n, col = (int64_t)c * kTileCols + 32 * s + 8 * j;
        xv[t][s] = row < rows && col < k ? *(const pkv_u32x4 *)(x + row * x_stride + col) : none;
      }
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      w4_f32x4 acc[kParts][MT], xs[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        xs[t] = w4_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int p = 0; p < kParts; ++p) acc[p][t] = w4_f32x4{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int s = g * kSteps + i;
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
          const pkv_u32x4 a = w4_expand(w[p][s]);
#pragma unroll
          for (int t = 0; t < MT; ++t) acc[p][t] = w4_mfma(a, xv[t][s], acc[p][t]);
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) xs[t] = w4_mfma(ones, xv[t][s], xs[t]);
      }
#pragma unroll
      for (int p = 0; p < kParts; ++p)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float scale = __uint_as_float(sc[p][g][r] & 0xffff0000u), zero = __uint_as_float(sc[p][g][r] << 16);
#pragma unroll
          for (int t = 0; t < MT; ++t) tot[p][t][r] = fmaf(scale, fmaf(-zero, xs[t][r], acc[p][t][r]), tot[p][t][r]);
        }
    }
  }
  // lane (n, j) has rows 4 j .. 4 j + 3 of the tile for row n of x; the waves' shares are added in their order
  __shared__ float s_part[kWaves][kParts][MT][16][17];
#pragma unroll
  for (int p = 0; p < kParts; ++p)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) s_part[wave][p][t][n][4 * j + r] = tot[p][t][r];
  __syncthreads();
  for (int e = threadIdx.x; e < MT * 256; e += kWaves * PKV_WAVE) {
    const int t = e >> 8, m = (e >> 4) & 15, r = e & 15;
    const int64_t row = m0 + 16 * t + m, col = tile * kTileRows + r;
    if (row >= rows || col >= n_out) continue;
    float v[kParts];
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      v[p] = s_part[0][p][t][m][r];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) v[p] += s_part[w][p][t][m][r];
    }
    float out = v[0];
    if (GATED) out = v[0] / (1.0f + __expf(-v[0])) * v[kParts - 1];
    if (bias) out += pkv_bf16_bits_to_f32(bias[col]);
    if (out_f32) ((float *)y)[row * n_out + col] = out;
    else ((uint16_t *)y)[row * n_out + col] = pkv_f32_to_bf16_bits(out);
  }
}

// Where column c of a 32-column step's word goes: see pkv_w4_pack in the header.
__device__ __forceinline__ uint32_t w4_place(uint32_t code, int e) {
  const int at = (3 + 4 * (e >> 1) + 16 * (e & 1)) & 31;
  return at == 0 ? code : (code << at) | (code >> (32 - at));
}

// One thread a 16-byte vector of a tile.
__global__ __launch_bounds__(256) void pkv_w4_pack_kernel(const uint8_t *__restrict__ codes, const uint16_t *__restrict__ scales,
                                                          const uint8_t *__restrict__ zeros, int64_t n, int64_t k, int group,
                                                          int chunks, int64_t n_tiles, char *__restrict__ tiles,
                                                          uint32_t *__restrict__ words) {
  const int64_t vec = (int64_t)blockIdx.x * 256 + threadIdx.x, tile_chunk = vec >> 6;
  const int lane = (int)(vec & 63), r = lane & 15, j = lane >> 4;
  if (tile_chunk >= n_tiles * chunks) return;
  const int64_t tile = tile_chunk / chunks, c = tile_chunk % chunks, row = tile * kTileRows + r, groups = k / group;
  pkv_u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int64_t col = c * kTileCols + 32 * s + 8 * j;
    if (row < n && col < k)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[s] |= w4_place(codes[row * k + col + e] & 15u, e);
  }
  ((pkv_u32x4 *)tiles)[vec] = v;
  const int per = kTileCols / group;  // groups of this chunk: lane j < per writes one of them
  if (j < per) {
    const int64_t g = c * per + j;
    const bool real = row < n && g < groups;
    const uint32_t s = real ? scales[row * groups + g] : 0u, z = real ? zeros[row * groups + g] & 15u : 0u;
    words[(tile_chunk * per + j) * kTileRows + r] = (s << 16) | (0x4180u + (z << 3));
  }
}

__global__ __launch_bounds__(256) void pkv_w4_unpack_kernel(const char *__restrict__ tiles, const uint32_t *__restrict__ words, int64_t n,
                                                            int64_t k, int group, int chunks, int64_t n_tiles, float *__restrict__ out) {
  const int64_t vec = (int64_t)blockIdx.x * 256 + threadIdx.x, tile_chunk = vec >> 6;
  const int lane = (int)(vec & 63), r = lane & 15, j = lane >> 4;
  if (tile_chunk >= n_tiles * chunks) return;
  const int64_t tile = tile_chunk / chunks, c = tile_chunk % chunks, row = tile * kTileRows + r;
  const pkv_u32x4 v = ((const pkv_u32x4 *)tiles)[vec];
  const int per = kTileCols / group;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int64_t col = c * kTileCols + 32 * s + 8 * j;
    if (row >= n || col >= k) continue;
    const uint32_t word = words[(tile_chunk * per + (32 * s) / group) * kTileRows + r];
    const float scale = __uint_as_float(word & 0xffff0000u), zero = __uint_as_float(word << 16);
    const pkv_u32x4 a = w4_expand(v[s]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float q = __uint_as_float(e & 1 ? a[e >> 1] & 0xffff0000u : a[e >> 1] << 16);
      out[row * k + col + e] = scale * (q - zero);
    }
  }
}

// 32 lanes a group.
template <bool BF16>
__global__ __launch_bounds__(256) void pkv_w4_quantize_kernel(const void *__restrict__ w, int64_t row_stride, int64_t n, int64_t k, int group,
                                                              uint8_t *__restrict__ codes, uint16_t *__restrict__ scales,
                                                              uint8_t *__restrict__ zeros) {
  const int64_t groups = k / group, at = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  const int l = threadIdx.x & 31;
  if (at >= n * groups) return;  // whole halves of a wave
  const int64_t row = at / groups, g = at % groups;
  float v[4], lo = 0.f, hi = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t e = row * row_stride + g * group + 32 * i + l;
    v[i] = 32 * i >= group ? 0.f : BF16 ? pkv_bf16_bits_to_f32(((const uint16_t *)w)[e]) : ((const float *)w)[e];
    lo = fminf(lo, v[i]), hi = fmaxf(hi, v[i]);
  }
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) lo = fminf(lo, __shfl_xor(lo, m, PKV_WAVE)), hi = fmaxf(hi, __shfl_xor(hi, m, PKV_WAVE));
  const float scale = pkv_bf16_round((hi - lo) / 15.0f);
  const bool some = scale >= 1.17549435e-38f;
  const float zero = some ? fminf(fmaxf(rintf(-lo / scale), 0.f), 15.f) : 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (32 * i < group)
      codes[row * k + g * group + 32 * i + l] = (uint8_t)(some ? fminf(fmaxf(rintf(v[i] / scale) + zero, 0.f), 15.f) : 0.f);
  if (l == 0) scales[at] = some ? (uint16_t)(__float_as_uint(scale) >> 16) : 0, zeros[at] = (uint8_t)zero;
}

bool w4_shape_ok(int64_t n, int64_t k, int group) {
  return (group == 32 || group == 64 || group == 128) && n > 0 && k > 0 && k % group == 0 && n < ((int64_t)1 << 31) &&
         k < ((int64_t)1 << 24) && (n + 15) / 16 * ((k + 127) / 128) < ((int64_t)1 << 32);
}
int64_t w4_tiles(int64_t n) { return (n + kTileRows - 1) / kTileRows; }
int64_t w4_chunks(int64_t k) { return (k + kTileCols - 1) / kTileCols; }
W4Matrix w4_matrix(const void *packed, int64_t n, int64_t k) {
  return {(const char *)packed, (const uint32_t *)((const char *)packed + w4_tiles(n) * w4_chunks(k) * kTileBytes)};
}

#define PKV_W4_SHAPE(what)                                                                                                       \
  PKV_REQUIRE(w4_shape_ok(n, k, group), what ": groups of 32, 64 or 128, k a multiple of them (got n=%lld k=%lld group=%d)", \
              (long long)n, (long long)k, group)

template <bool GATED>
int w4_launch(const void *x, int64_t x_stride, int64_t rows, W4Matrix a, W4Matrix b, int64_t n, int64_t k, int group, const void *bias,
              void *y, int out_f32, hipStream_t s) {
  const int mt = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  const int64_t row_tiles = (rows + 16 * mt - 1) / (16 * mt);
  PKV_REQUIRE(row_tiles <= 65535, "pkv_w4: too many rows (%lld)", (long long)rows);
  const dim3 grid((unsigned)w4_tiles(n), (unsigned)row_tiles);
#define PKV_W4(MT, G)                                                                                                              \
  hipLaunchKernelGGL((pkv_w4_kernel<MT, G, GATED>), grid, dim3(kWaves * PKV_WAVE), 0, s, (const uint16_t *)x, x_stride, rows, a, b, \
                     n, k, (int)w4_chunks(k), (const uint16_t *)bias, y, out_f32)
#define PKV_W4_G(MT)                     \
  do {                                   \
    if (group == 32) PKV_W4(MT, 32);     \
    else if (group == 64) PKV_W4(MT, 64); \
    else PKV_W4(MT, 128);                \
  } while (0)
  if (mt == 1) PKV_W4_G(1);
  else if (mt == 2) PKV_W4_G(2);
  else PKV_W4_G(4);
#undef PKV_W4_G
#undef PKV_W4
  PKV_LAUNCH_CHECK("pkv_w4_kernel");
  return PKV_OK;
}

int w4_check_x(const void *x, int64_t x_stride, int64_t rows, int64_t k, const void *y) {
  PKV_REQUIRE(x && y, "pkv_w4: null pointer");
  PKV_REQUIRE(rows > 0 && rows < ((int64_t)1 << 22), "pkv_w4: bad row count %lld", (long long)rows);
  PKV_REQUIRE(pkv_aligned(x, 16) && (rows == 1 || (x_stride % 8 == 0 && x_stride >= k)),
              "pkv_w4: rows of x must be 16-byte aligned and not overlap");
  return PKV_OK;
}

}  // namespace

extern "C" size_t pkv_w4_bytes(int64_t n, int64_t k, int group) {
  if (!w4_shape_ok(n, k, group)) return 0;
  return (size_t)(w4_tiles(n) * w4_chunks(k)) * (kTileBytes + kTileCols / group * kTileRows * 4);
}

extern "C" int pkv_w4_pack(const uint8_t *codes, const uint16_t *scales, const uint8_t *zeros, int64_t n, int64_t k, int group,
                           void *packed, void *stream) {
  PKV_REQUIRE(codes && scales && zeros && packed, "pkv_w4_pack: null pointer");
  PKV_W4_SHAPE("pkv_w4_pack");
  PKV_REQUIRE(pkv_aligned(packed, 16) && pkv_aligned(scales, 2), "pkv_w4_pack: 16-byte aligned buffer required");
  const W4Matrix m = w4_matrix(packed, n, k);
  const int64_t blocks = (w4_tiles(n) * w4_chunks(k) + 3) / 4;
  PKV_REQUIRE(blocks < ((int64_t)1 << 31), "pkv_w4_pack: too large");
  hipLaunchKernelGGL(pkv_w4_pack_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, codes, scales, zeros, n, k, group,
                     (int)w4_chunks(k), w4_tiles(n), (char *)m.tiles, (uint32_t *)m.words);
  PKV_LAUNCH_CHECK("pkv_w4_pack_kernel");
  return PKV_OK;
}

extern "C" int pkv_w4_unpack(const void *packed, int64_t n, int64_t k, int group, float *w, void *stream) {
  PKV_REQUIRE(packed && w, "pkv_w4_unpack: null pointer");
  PKV_W4_SHAPE("pkv_w4_unpack");
  PKV_REQUIRE(pkv_aligned(packed, 16) && pkv_aligned(w, 4), "pkv_w4_unpack: 16-byte aligned buffer required");
  const W4Matrix m = w4_matrix(packed, n, k);
  const int64_t blocks = (w4_tiles(n) * w4_chunks(k) + 3) / 4;
  PKV_REQUIRE(blocks < ((int64_t)1 << 31), "pkv_w4_unpack: too large");
  hipLaunchKernelGGL(pkv_w4_unpack_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, m.tiles, m.words, n, k, group,
                     (int)w4_chunks(k), w4_tiles(n), w);
  PKV_LAUNCH_CHECK("pkv_w4_unpack_kernel");
  return PKV_OK;
}

extern "C" int pkv_w4_quantize(const void *w, int dtype, int64_t row_stride, int64_t n, int64_t k, int group, uint8_t *codes,
                               uint16_t *scales, uint8_t *zeros, void *stream) {
  PKV_REQUIRE(w && codes && scales && zeros, "pkv_w4_quantize: null pointer");
  PKV_REQUIRE(dtype == PKV_DTYPE_F32 || dtype == PKV_DTYPE_BF16, "unknown dtype %d", dtype);
  PKV_W4_SHAPE("pkv_w4_quantize");
  PKV_REQUIRE(row_stride >= k || n == 1, "pkv_w4_quantize: rows must not overlap");
  const int64_t blocks = (n * (k / group) + 7) / 8;
  PKV_REQUIRE(blocks < ((int64_t)1 << 31), "pkv_w4_quantize: too large");
  if (dtype == PKV_DTYPE_BF16)
    hipLaunchKernelGGL(pkv_w4_quantize_kernel<true>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, w, row_stride, n, k, group,
                       codes, scales, zeros);
  else
    hipLaunchKernelGGL(pkv_w4_quantize_kernel<false>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, w, row_stride, n, k, group,
                       codes, scales, zeros);
  PKV_LAUNCH_CHECK("pkv_w4_quantize_kernel");
  return PKV_OK;
}

extern "C" int pkv_w4_linear(const void *x, int64_t x_stride, int64_t rows, const void *packed, int64_t n, int64_t k, int group,
                             const void *bias, void *y, int out_dtype, void *stream) {
  PKV_REQUIRE(packed && pkv_aligned(packed, 16), "pkv_w4_linear: 16-byte aligned weights required");
  PKV_REQUIRE(out_dtype == PKV_DTYPE_F32 || out_dtype == PKV_DTYPE_BF16, "unknown dtype %d", out_dtype);
  PKV_W4_SHAPE("pkv_w4_linear");
  const int rc = w4_check_x(x, x_stride, rows, k, y);
  if (rc) return rc;
  return w4_launch<false>(x, x_stride, rows, w4_matrix(packed, n, k), W4Matrix{}, n, k, group, bias, y, out_dtype == PKV_DTYPE_F32,
                          (hipStream_t)stream);
}

extern "C" int pkv_w4_silu_mul(const void *x, int64_t x_stride, int64_t rows, const void *gate, const void *up, int64_t n, int64_t k,
                               int group, void *y, void *stream) {
  PKV_REQUIRE(gate && up && pkv_aligned(gate, 16) && pkv_aligned(up, 16), "pkv_w4_silu_mul: 16-byte aligned weights required");
  PKV_W4_SHAPE("pkv_w4_silu_mul");
  const int rc = w4_check_x(x, x_stride, rows, k, y);
  if (rc) return rc;
  return w4_launch<true>(x, x_stride, rows, w4_matrix(gate, n, k), w4_matrix(up, n, k), n, k, group, nullptr, y, 0,
                         (hipStream_t)stream);
}
