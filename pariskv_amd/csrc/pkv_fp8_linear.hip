// Products of eight-bit rows with eight-bit matrices, a scale for each row of both: y[m][n] = sx[m] sw[n] sum_k xc[m][k] wc[n][k] + bias[n],
// codes e4m3.  (No counterpart in the reference, whose projections are bf16 GEMMs, model_hub/qwen.py:327-383.)
//
// Codes become bf16 numbers in registers, exactly (two to an instruction), and go to v_mfma_f32_16x16x32_bf16, whose products of them
// are exact and whose sums are fp32.  The instructions that take e4m3 codes themselves have twice the rate, but add eight neighbouring products
// up with nothing below 2^-13 of the largest of them: 2^16 + 4 is 2^16, and rows of normal numbers come out 1.5e-5 off.
// Which columns a lane has is free as long as both operands agree: lane (r, j) takes columns 16 j .. 16 j + 15 and 64 + 16 j .. of a chunk of 128,
// so that the rows of x are read 64 bytes side by side.  The matrix is laid out once in tiles of 16 rows x 128 columns in the order of the lanes.
#include "pkv_fp8.h"

namespace {

typedef __bf16 fp8_bf16x8 __attribute__((ext_vector_type(8)));
typedef float fp8_f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTileRows = 16, kTileCols = 128, kTileBytes = kTileRows * kTileCols;

struct Codes {  // 32 codes of a lane
  pkv_u32x4 half[2];
};
struct Operand {  // ... as bf16 numbers
  pkv_u32x4 part[4];
  __device__ __forceinline__ Operand(const Codes &c) {
#pragma unroll
    for (int p = 0; p < 4; ++p)
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        const uint32_t w = c.half[p >> 1][2 * (p & 1) + d];
        part[p][2 * d] = fp8_bf16x2<false>(w), part[p][2 * d + 1] = fp8_bf16x2<true>(w);
      }
  }
};
__device__ __forceinline__ fp8_f32x4 fp8_mfma(const Operand &a, const Operand &b, fp8_f32x4 c) {
#pragma unroll
  for (int p = 0; p < 4; ++p)
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(fp8_bf16x8, a.part[p]), __builtin_bit_cast(fp8_bf16x8, b.part[p]), c, 0, 0, 0);
  return c;
}

struct LinearArgs {
  const uint8_t *x;     // [m][chunks * 128]
  const float *sx;
  const uint8_t *tiles; // [row tile][chunk][half][lane] of 16 bytes
  const float *sw;      // [row tiles * 16]
  const uint16_t *bias; // or null
  void *y;
  int64_t m, n;
  int chunks, f32;
};

__device__ __forceinline__ void put(const LinearArgs &a, int64_t row, int64_t col, float sum, float sx) {
  float v = sum * sx * a.sw[col];
  if (a.bias) v += pkv_bf16_bits_to_f32(a.bias[col]);
  if (a.f32) ((float *)a.y)[row * a.n + col] = v;
  else ((uint16_t *)a.y)[row * a.n + col] = pkv_f32_to_bf16_bits(v);
}

// Few rows: the matrix is read once and the bytes bound it.  A workgroup takes 16 RT rows of the matrix and 16 MT of x, its waves every
// kStreamWaves-th chunk of columns, straight from memory into the operands; they meet in LDS, in their order.
constexpr int kStreamWaves = 8;
template <int MT, int RT>
__global__ __launch_bounds__(kStreamWaves * PKV_WAVE) void pkv_fp8_stream_kernel(LinearArgs a) {
  constexpr int kAhead = MT * RT > 4 ? 1 : MT + RT > 3 ? 2 : 4;  // chunks under way
  __shared__ fp8_f32x4 s_part[kStreamWaves][RT][MT][PKV_WAVE];
  const int tid = threadIdx.x, lane = pkv_lane(), wave = tid / PKV_WAVE, n = lane & 15, j = lane >> 4;
  const int64_t tiles = (a.n + kTileRows - 1) / kTileRows, m0 = (int64_t)blockIdx.y * 16 * MT, t0 = (int64_t)blockIdx.x * RT;
  const uint8_t *w_at[RT], *x_at[MT];
#pragma unroll
  for (int r = 0; r < RT; ++r) w_at[r] = a.tiles + (t0 + r < tiles ? t0 + r : tiles - 1) * a.chunks * kTileBytes + lane * 16;
#pragma unroll
  for (int t = 0; t < MT; ++t) x_at[t] = a.x + (m0 + 16 * t + n < a.m ? m0 + 16 * t + n : a.m - 1) * a.chunks * kTileCols + 16 * j;
  fp8_f32x4 acc[RT][MT];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[r][t] = fp8_f32x4{0.f, 0.f, 0.f, 0.f};
  for (int c0 = wave; c0 < a.chunks; c0 += kStreamWaves * kAhead) {
    Codes w[kAhead][RT], x[kAhead][MT];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int c = c0 + u * kStreamWaves;
      if (c >= a.chunks) break;  // the whole wave
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) w[u][r].half[h] = __builtin_nontemporal_load((const pkv_u32x4 *)(w_at[r] + (int64_t)c * kTileBytes + h * 1024));
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) x[u][t].half[h] = *(const pkv_u32x4 *)(x_at[t] + c * kTileCols + h * 64);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (c0 + u * kStreamWaves >= a.chunks) break;
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const Operand wo(w[u][r]);
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[r][t] = fp8_mfma(wo, Operand(x[u][t]), acc[r][t]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < MT; ++t) s_part[wave][r][t][lane] = acc[r][t];
  __syncthreads();
  // number e of the workgroup's: column e mod 16 RT of the matrix' rows, row e / (16 RT) of x
  for (int e = tid; e < 256 * RT * MT; e += kStreamWaves * PKV_WAVE) {
    const int col = e % (16 * RT), row = e / (16 * RT), r = col / 16, t = row / 16;
    const int at = (((col & 15) >> 2) * 16 + (row & 15)) * 4 + (col & 3);  // lane (row, col / 4), its element col mod 4
    float sum = ((const float *)s_part[0][r][t])[at];
#pragma unroll
    for (int w = 1; w < kStreamWaves; ++w) sum += ((const float *)s_part[w][r][t])[at];
    if (m0 + row < a.m && t0 * 16 + col < a.n) put(a, m0 + row, t0 * 16 + col, sum, a.sx[m0 + row]);
  }
}

// Many rows: 128 x 128 of y a workgroup, 64 x 64 a wave.  A chunk of both operands goes straight from memory to LDS in the order of the lanes.
constexpr int kBlock = 128, kBlockTiles = kBlock / 16;
typedef const __attribute__((address_space(1))) void *fp8_global;
typedef __attribute__((address_space(3))) void *fp8_lds;
__global__ __launch_bounds__(256) void pkv_fp8_block_kernel(LinearArgs a) {
  __shared__ alignas(16) uint8_t lds[2][kBlockTiles * kTileBytes];  // x, matrix
  const int tid = threadIdx.x, lane = pkv_lane(), wave = __builtin_amdgcn_readfirstlane(tid / PKV_WAVE), n = lane & 15, j = lane >> 4;
  const int64_t tiles = (a.n + kTileRows - 1) / kTileRows, m0 = (int64_t)blockIdx.y * kBlock, t0 = (int64_t)blockIdx.x * kBlockTiles;
  const int wm = wave & 1, wn = wave >> 1;
  // what this wave brings in: two tiles of each
  const uint8_t *x_at[2], *w_at[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int64_t row = m0 + (2 * wave + u) * 16 + n, tile = t0 + 2 * wave + u;
    x_at[u] = a.x + (row < a.m ? row : a.m - 1) * a.chunks * kTileCols + 16 * j;
    w_at[u] = a.tiles + (tile < tiles ? tile : tiles - 1) * a.chunks * kTileBytes + lane * 16;
  }
  fp8_f32x4 acc[4][4];
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[r][t] = fp8_f32x4{0.f, 0.f, 0.f, 0.f};
  for (int c = 0; c < a.chunks; ++c) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        __builtin_amdgcn_global_load_lds((fp8_global)(x_at[u] + c * kTileCols + h * 64), (fp8_lds)(lds[0] + (2 * wave + u) * kTileBytes + h * 1024), 16, 0, 0);
        __builtin_amdgcn_global_load_lds((fp8_global)(w_at[u] + (int64_t)c * kTileBytes + h * 1024), (fp8_lds)(lds[1] + (2 * wave + u) * kTileBytes + h * 1024), 16, 0, 0);
      }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    Codes x[4], w[4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        x[t].half[h] = *(const pkv_u32x4 *)(lds[0] + (4 * wm + t) * kTileBytes + h * 1024 + lane * 16);
        w[t].half[h] = *(const pkv_u32x4 *)(lds[1] + (4 * wn + t) * kTileBytes + h * 1024 + lane * 16);
      }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const Operand wo(w[r]);
#pragma unroll
      for (int t = 0; t < 4; ++t) acc[r][t] = fp8_mfma(wo, Operand(x[t]), acc[r][t]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int64_t row = m0 + (4 * wm + t) * 16 + n;
    if (row >= a.m) continue;
    const float sx = a.sx[row];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t col = (t0 + 4 * wn + r) * 16 + 4 * j + i;
        if (col < a.n) put(a, row, col, acc[r][t][i], sx);
      }
  }
}

// Codes [n][k] into tiles and back: one 16-byte vector of a tile a thread.
__global__ __launch_bounds__(256) void pkv_fp8_pack_kernel(const uint8_t *__restrict__ codes, const float *__restrict__ scales, int64_t n, int64_t k,
                                                           int64_t stride, int chunks, int64_t vecs, uint8_t *__restrict__ tiles, float *__restrict__ sw) {
  const int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t rows = (n + kTileRows - 1) / kTileRows * kTileRows;
  if (v < rows) sw[v] = v < n ? scales[v] : 0.f;
  if (v >= vecs) return;
  const int lane = (int)(v & 63), h = (int)(v >> 6) & 1;
  const int64_t tc = v >> 7, tile = tc / chunks, c = tc - tile * chunks;
  const int64_t row = tile * 16 + (lane & 15), col = c * kTileCols + h * 64 + (lane >> 4) * 16;
  uint8_t out[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) out[i] = row < n && col + i < k ? codes[row * stride + col + i] : (uint8_t)0;
  pkv_u32x4 o;
  memcpy(&o, out, 16);
  *(pkv_u32x4 *)(tiles + v * 16) = o;
}

__global__ __launch_bounds__(256) void pkv_fp8_unpack_kernel(const uint8_t *__restrict__ tiles, const float *__restrict__ sw, int64_t n, int64_t k,
                                                             int chunks, float *__restrict__ w) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= n * k) return;
  const int64_t row = e / k, col = e - row * k;
  const int in = (int)(col & 127);
  const uint8_t code = tiles[((row >> 4) * chunks + (col >> 7)) * kTileBytes + (in >> 6) * 1024 + (((in & 63) >> 4) * 16 + (row & 15)) * 16 + (in & 15)];
  w[e] = __builtin_amdgcn_cvt_pk_f32_fp8((int)code, false)[0] * sw[row];
}

int64_t row_tiles(int64_t n) { return (n + kTileRows - 1) / kTileRows; }
int chunks_of(int64_t k) { return (int)((k + kTileCols - 1) / kTileCols); }
size_t tile_bytes(int64_t n, int64_t k) { return (size_t)row_tiles(n) * chunks_of(k) * kTileBytes; }
bool matrix_ok(int64_t n, int64_t k) { return n > 0 && n < ((int64_t)1 << 31) - 16 && k > 0 && k <= ((int64_t)1 << 20); }

}  // namespace

extern "C" size_t pkv_fp8_bytes(int64_t n, int64_t k) {
  if (!matrix_ok(n, k)) return 0;
  return tile_bytes(n, k) + (size_t)row_tiles(n) * kTileRows * sizeof(float);
}

extern "C" int pkv_fp8_pack(const uint8_t *codes, int64_t row_stride, const float *scales, int64_t n, int64_t k, void *packed, void *stream) {
  PKV_REQUIRE(codes && scales && packed, "pkv_fp8_pack: null pointer");
  PKV_REQUIRE(matrix_ok(n, k) && row_stride >= k, "pkv_fp8_pack: bad matrix %lld x %lld", (long long)n, (long long)k);
  PKV_REQUIRE(pkv_aligned(packed, 16) && pkv_aligned(scales, 4), "pkv_fp8_pack: 16-byte aligned buffers required");
  const int64_t vecs = (int64_t)(tile_bytes(n, k) / 16);
  PKV_REQUIRE(vecs / 256 < ((int64_t)1 << 31), "pkv_fp8_pack: matrix too large");
  hipLaunchKernelGGL(pkv_fp8_pack_kernel, dim3((unsigned)((vecs + 255) / 256)), dim3(256), 0, (hipStream_t)stream, codes, scales, n, k, row_stride,
                     chunks_of(k), vecs, (uint8_t *)packed, (float *)((uint8_t *)packed + tile_bytes(n, k)));
  PKV_LAUNCH_CHECK("pkv_fp8_pack_kernel");
  return PKV_OK;
}

extern "C" int pkv_fp8_unpack(const void *packed, int64_t n, int64_t k, float *w, void *stream) {
  PKV_REQUIRE(packed && w, "pkv_fp8_unpack: null pointer");
  PKV_REQUIRE(matrix_ok(n, k) && pkv_aligned(packed, 16) && n * k / 256 < ((int64_t)1 << 31), "pkv_fp8_unpack: bad matrix %lld x %lld", (long long)n, (long long)k);
  hipLaunchKernelGGL(pkv_fp8_unpack_kernel, dim3((unsigned)((n * k + 255) / 256)), dim3(256), 0, (hipStream_t)stream, (const uint8_t *)packed,
                     (const float *)((const uint8_t *)packed + tile_bytes(n, k)), n, k, chunks_of(k), w);
  PKV_LAUNCH_CHECK("pkv_fp8_unpack_kernel");
  return PKV_OK;
}

extern "C" int pkv_fp8_linear(const uint8_t *x, const float *x_scales, int64_t rows, const void *packed, int64_t n, int64_t k, const void *bias,
                              void *y, int out_dtype, void *stream) {
  PKV_REQUIRE(x && x_scales && packed && y, "pkv_fp8_linear: null pointer");
  PKV_REQUIRE(out_dtype == PKV_DTYPE_F32 || out_dtype == PKV_DTYPE_BF16, "unknown dtype %d", out_dtype);
  PKV_REQUIRE(matrix_ok(n, k) && rows > 0 && rows <= ((int64_t)1 << 22), "pkv_fp8_linear: bad shape %lld rows, %lld x %lld", (long long)rows, (long long)n, (long long)k);
  PKV_REQUIRE(pkv_aligned(x, 16) && pkv_aligned(packed, 16) && pkv_aligned(x_scales, 4) && pkv_aligned(bias, 2) && pkv_aligned(y, 4), "pkv_fp8_linear: 16-byte aligned operands required");
  LinearArgs a;
  a.x = x, a.sx = x_scales, a.tiles = (const uint8_t *)packed, a.sw = (const float *)((const uint8_t *)packed + tile_bytes(n, k));
  a.bias = (const uint16_t *)bias, a.y = y, a.m = rows, a.n = n, a.chunks = chunks_of(k), a.f32 = out_dtype == PKV_DTYPE_F32;
  hipStream_t s = (hipStream_t)stream;
  const unsigned tiles = (unsigned)row_tiles(n);
  if (rows <= 16) hipLaunchKernelGGL((pkv_fp8_stream_kernel<1, 1>), dim3(tiles), dim3(kStreamWaves * PKV_WAVE), 0, s, a);
  else if (rows <= 32) hipLaunchKernelGGL((pkv_fp8_stream_kernel<2, 1>), dim3(tiles), dim3(kStreamWaves * PKV_WAVE), 0, s, a);
  else if (rows <= 128) hipLaunchKernelGGL((pkv_fp8_stream_kernel<4, 1>), dim3(tiles, (unsigned)((rows + 63) / 64)), dim3(kStreamWaves * PKV_WAVE), 0, s, a);
  else hipLaunchKernelGGL(pkv_fp8_block_kernel, dim3((tiles + kBlockTiles - 1) / kBlockTiles, (unsigned)((rows + kBlock - 1) / kBlock)), dim3(256), 0, s, a);
  PKV_LAUNCH_CHECK("pkv_fp8_linear");
  return PKV_OK;
}
