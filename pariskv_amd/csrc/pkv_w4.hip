// Products of few rows with matrices of 4-bit weights and group scales: the projections of a decode step, or of a step over
// several drafted tokens, at a quarter of the bytes.  (No counterpart in the reference, whose projections are bf16 GEMMs,
// model_hub/qwen.py:327-383.)
//
// y[m][n] = sum_k x[m][k] s[n][g(k)] (q[n][k] - z[n][g(k)]) = sum_g s[n][g] (sum_k x (16 + q) - (16 + z[n][g]) sum_k x)
//
// 16 + q is a bf16 number that a rotation, an AND and an OR make of a code (the code goes into the upper four mantissa bits of 16.0;
// 16 is the smallest number whose mantissa has room for it, so that the difference cancels as little as it can): 7 vector instructions for 8
// weights.  Both sums over k come from v_mfma_f32_16x16x32_bf16, the second with a matrix of ones, which leaves sum x in the
// registers where it is needed; products of bf16 numbers are exact in fp32, as are the codes, and sums are fp32.  (Where x stays in LDS the second
// is found once, as x is put there.)
#include "pkv_common.h"

namespace {

typedef __bf16 w4_bf16x8 __attribute__((ext_vector_type(8)));
typedef float w4_f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTileRows = 16, kTileCols = 128, kTileBytes = 1024;
constexpr int kWaves = 8;

__device__ __forceinline__ w4_f32x4 w4_mfma(pkv_u32x4 a, pkv_u32x4 b, w4_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(w4_bf16x8, a), __builtin_bit_cast(w4_bf16x8, b), c, 0, 0, 0);
}

// The eight codes of a word as bf16 numbers 16 + q, in column order.
__device__ __forceinline__ pkv_u32x4 w4_expand(uint32_t w) {
  uint32_t keep = 0x00780078u, sixteen = 0x41804180u;
  asm("" : "+s"(keep), "+v"(sixteen));  // in registers: AND and OR are one instruction, which takes no constants
  return pkv_u32x4{(w & keep) | sixteen, ((w >> 4) & keep) | sixteen, ((w >> 8) & keep) | sixteen,
                   (__builtin_amdgcn_alignbit(w, w, 12) & keep) | sixteen};
}

// Columns past k of a chunk, whose scales are zero: a sum with them has to be finite for that to make them nothing, so x has zeros there.
__device__ __forceinline__ pkv_u32x4 w4_columns(pkv_u32x4 x, int64_t col, int64_t k) {
  uint32_t keep = col < k ? 0xffffffffu : 0u;
  asm volatile("" : "+v"(keep));  // stays behind the caller's branch
  return pkv_u32x4{x.x & keep, x.y & keep, x.z & keep, x.w & keep};
}

struct W4Matrix {
  const char *tiles;      // [row tile][chunk of 128 columns] of kTileBytes
  const uint32_t *words;  // [row tile][group][16]
};

// One chunk of one row tile, of each of PARTS matrices: the codes of a lane and the words of its four rows' groups.
template <int G, int PARTS>
struct W4Chunk {
  static constexpr int kGroups = kTileCols / G;
  pkv_u32x4 w[PARTS], sc[PARTS][kGroups];
  // w_at, s_at: the lane's first vector and words of chunk 0
  __device__ __forceinline__ void load(const char *const (&w_at)[PARTS], const char *const (&s_at)[PARTS], int64_t c) {
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      w[p] = __builtin_nontemporal_load((const pkv_u32x4 *)(w_at[p] + c * kTileBytes));
#pragma unroll
      for (int g = 0; g < kGroups; ++g) sc[p][g] = *(const pkv_u32x4 *)(s_at[p] + (c * kGroups + g) * (kTileRows * 4));
    }
  }
};

// tot += chunk times x; x_of(t, s): columns 32 s + 8 j .. of the chunk of row n of tile t of x; sum_of(t, g): the sum of row n's columns of
// its group g, where the caller has it (SUMS), else a product with ones finds it.
template <int MT, int G, int PARTS, bool SUMS, typename Of, typename SumOf>
__device__ __forceinline__ void w4_chunk(const W4Chunk<G, PARTS> &c, Of x_of, SumOf sum_of, w4_f32x4 (&tot)[PARTS][MT]) {
  constexpr int kSteps = G / 32;
  const pkv_u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
  for (int g = 0; g < kTileCols / G; ++g) {
    w4_f32x4 acc[PARTS][MT], xs[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      xs[t] = w4_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int p = 0; p < PARTS; ++p) acc[p][t] = w4_f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int s = g * kSteps + i;
      pkv_u32x4 xv[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        xv[t] = x_of(t, s);
        if constexpr (!SUMS) xs[t] = w4_mfma(ones, xv[t], xs[t]);
      }
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        const pkv_u32x4 a = w4_expand(c.w[p][s]);
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[p][t] = w4_mfma(a, xv[t], acc[p][t]);
      }
    }
    float sum[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) sum[t] = SUMS ? sum_of(t, g) : xs[t][0];
#pragma unroll
    for (int p = 0; p < PARTS; ++p)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float scale = __uint_as_float(c.sc[p][g][r] & 0xffff0000u), zero = __uint_as_float(c.sc[p][g][r] << 16);
#pragma unroll
        for (int t = 0; t < MT; ++t) tot[p][t][r] = fmaf(scale, fmaf(-zero, sum[t], acc[p][t][r]), tot[p][t][r]);
      }
  }
}

struct W4Out {
  const uint16_t *bias;
  void *y;
  int f32;
};
template <int PARTS>
__device__ __forceinline__ void w4_store(const W4Out &o, int64_t at, int64_t col, const float (&v)[PARTS]) {
  float out = v[0];
  if (PARTS == 2) out = v[0] / (1.0f + __expf(-v[0])) * v[PARTS - 1];
  if (o.bias) out += pkv_bf16_bits_to_f32(o.bias[col]);
  if (o.f32) ((float *)o.y)[at] = out;
  else ((uint16_t *)o.y)[at] = pkv_f32_to_bf16_bits(out);
}

// x is read by rows and goes through LDS: a product wants 64 bytes of each of 16 rows, which lie a multiple of the interleaving of the L2's
// channels apart and came one after the other when they were read straight from there (4096 x 12288, 64 rows: 47 us, of them 12 of
// instructions).  In LDS vector c (of 16) of a chunk of row r lies at c ^ (r mod 16): the 16 rows of an operand are on different banks.

// 16 MT rows whose x fits into XKB KB of LDS: it stays there while a workgroup goes through its row tiles.  1 << lg of its waves share a
// tile, chunk c going to wave c mod (1 << lg), and meet in LDS after it; U chunks ahead are under way, over the ends of tiles too.
// A chunk costs a wave some 60 vector and 4 matrix instructions for its 1 KB.  151936 x 4096: 1 row 55 us (330 MB: 5.9 TB/s; a plain read
// reaches 7.1), 8 rows 63 us; with a workgroup to each 16 rows of the matrix, which reads x again for each of them, 75 and 94 us.
template <int MT, int G, bool GATED, int XKB, int U>
__global__ __launch_bounds__(kWaves * PKV_WAVE) void pkv_w4_resident_kernel(const uint16_t *__restrict__ x, int64_t x_stride, int64_t all_rows,
                                                                            W4Matrix wa, W4Matrix wb, int64_t n_out, int k, int chunks,
                                                                            int by_row_vecs, int lg, int each, int more,
                                                                            W4Out out) {
  constexpr int kParts = GATED ? 2 : 1, kFetch = XKB * 64 / (kWaves * PKV_WAVE) < 8 ? XKB * 64 / (kWaves * PKV_WAVE) : 8;
  __shared__ alignas(16) char lds[XKB * 1024];
  constexpr int kHalves = MT > 1 || (XKB == 64 && !GATED) ? 1 : 2;  // what fits; XKB = 64: for two workgroups a compute unit
  __shared__ float s_sum[XKB * 512 / G];                // of x, by row and group
  __shared__ w4_f32x4 s_part[kHalves][kWaves][kParts][MT][PKV_WAVE];  // rows 4 j .. 4 j + 3 for row n of x at 16 j + (n ^ 4 j): no two on one bank
  const int tid = threadIdx.x, lane = tid & (PKV_WAVE - 1), wave = __builtin_amdgcn_readfirstlane(tid / PKV_WAVE), n = lane & 15, j = lane >> 4;
  const int tiles = (int)((n_out + kTileRows - 1) / kTileRows), kg = wave & ((1 << lg) - 1), side = kWaves >> lg;
  const int64_t m0 = (int64_t)blockIdx.y * 16 * MT;
  const int rows = (int)(all_rows - m0 < 16 * MT ? all_rows - m0 : 16 * MT);
  x += m0 * x_stride;
  const int per_wave = (chunks + (1 << lg) - 1) >> lg, row_vecs = chunks * (kTileCols / 8), x_vecs = rows * row_vecs;
  const W4Matrix m[2] = {wa, wb};

  // x is asked for first: vectors tid, tid + 512, .. of its rows one after the other; past the end the last one again, past the columns the row's
  // first.  Vector v goes to v (as zeros where it is past the columns), its last four bits changed by its row, and the 16 lanes of a chunk add its
  // columns up.
  const bool ragged = G < kTileCols && k % kTileCols != 0;
  const int d_row = kWaves * PKV_WAVE * (unsigned)by_row_vecs >> 24, d_col = kWaves * PKV_WAVE - d_row * row_vecs;
  int f_row = (unsigned)tid * (unsigned)by_row_vecs >> 24, f_col = tid - f_row * row_vecs, p_row = f_row, p_col = f_col, put_at = 0;
  auto next = [&](int &row, int &col) {
    row += d_row, col += d_col;
    if (col >= row_vecs) col -= row_vecs, ++row;
  };
  auto fetch = [&](pkv_u32x4 (&got)[kFetch]) {
#pragma unroll
    for (int u = 0; u < kFetch; ++u) {
      const bool in = f_row < rows;
      const int row = in ? f_row : rows - 1, col = in ? f_col : row_vecs - 1;
      got[u] = *(const pkv_u32x4 *)(x + row * x_stride + (col * 8 < k ? col * 8 : 0));
      next(f_row, f_col);
    }
  };
  auto put = [&](pkv_u32x4 (&got)[kFetch]) {
#pragma unroll
    for (int u = 0; u < kFetch; ++u) {
      const bool in = p_row < rows;
      const int row = in ? p_row : rows - 1, col = in ? p_col : row_vecs - 1, v = row * row_vecs + col;
      asm volatile("" : "+v"(got[u]));  // arrived on every path, or its register's next use would wait for all of the ring
      if (put_at < x_vecs) {            // the whole workgroup
        if (ragged) got[u] = w4_columns(got[u], col * 8, k);
        *(pkv_u32x4 *)(lds + (v >> 4) * 256 + 16 * ((v ^ row) & 15)) = got[u];
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) sum += __uint_as_float(got[u][w] << 16) + __uint_as_float(got[u][w] & 0xffff0000u);
        sum += pkv_lane_xor_f<1>(sum);
        sum += pkv_lane_xor_f<2>(sum);
        if (G >= 64) sum += pkv_lane_xor_f<7>(sum);
        if (G >= 128) sum += pkv_lane_xor_f<15>(sum);
        if (in && v % (G / 8) == 0) s_sum[v / (G / 8)] = sum;
      }
      next(p_row, p_col);
      put_at += kWaves * PKV_WAVE;
    }
  };
  pkv_u32x4 got[kFetch];
  fetch(got);

  // the next chunk to ask for; past the last one it stays where it is
  int ask_tile = blockIdx.x * side + (wave >> lg), ask_i = 0, at_tile = ask_tile < tiles ? ask_tile : tiles - 1, at_c = 0;
  auto ask = [&](W4Chunk<G, kParts> &c) {
    const int now = (ask_i << lg) + kg;
    if (ask_tile < tiles) at_tile = ask_tile, at_c = now < chunks ? now : chunks - 1;  // scalars
    const char *w_at[kParts], *s_at[kParts];
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      w_at[p] = m[p].tiles + (int64_t)at_tile * chunks * kTileBytes + lane * 16;
      s_at[p] = (const char *)m[p].words + (int64_t)at_tile * chunks * (kTileCols / G) * (kTileRows * 4) + j * 16;
    }
    c.load(w_at, s_at, at_c);
    if (++ask_i == per_wave) ask_i = 0, ask_tile += gridDim.x * side;
  };
  W4Chunk<G, kParts> ring[U];
#pragma unroll
  for (int u = 0; u < U; ++u) ask(ring[u]);

  put(got);
  if constexpr (XKB * 64 > kFetch * kWaves * PKV_WAVE)
    while (put_at < x_vecs) fetch(got), put(got);
  __syncthreads();
  int my[MT];  // rows that are not there repeat the last; what is computed with them is not stored
#pragma unroll
  for (int t = 0; t < MT; ++t) my[t] = 16 * t + n < rows ? 16 * t + n : rows - 1;
  w4_f32x4 tot[kParts][MT];
#pragma unroll
  for (int p = 0; p < kParts; ++p)
#pragma unroll
    for (int t = 0; t < MT; ++t) tot[p][t] = w4_f32x4{0.f, 0.f, 0.f, 0.f};
  // One way through the loop, without a return inside: the waits for the ring count what came after on every path that might be.
  const int step = gridDim.x * side, steps = (each + ((int)blockIdx.x < more)) * per_wave;
  int tile = blockIdx.x * side, i = 0, half = 0;
  for (int at0 = 0; at0 < steps; at0 += U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = (i << lg) + kg;
      if (c < chunks && at0 + u < steps)  // the whole wave
        w4_chunk<MT, G, kParts, true>(
            ring[u],
            [&](int t, int s) { return *(const pkv_u32x4 *)(lds + my[t] * (row_vecs * 16) + c * 256 + 16 * ((4 * s + j) ^ (my[t] & 15))); },
            [&](int t, int g) { return s_sum[(my[t] * chunks + c) * (kTileCols / G) + g]; }, tot);
      ask(ring[u]);
      if (++i == per_wave && at0 + u < steps) {  // the whole workgroup
        // lane (n, j) has rows 4 j .. 4 j + 3 of the tile for row n of x; the waves' shares are added in their order
#pragma unroll
        for (int p = 0; p < kParts; ++p)
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            s_part[half][wave][p][t][16 * j + (n ^ 4 * j)] = tot[p][t];
            tot[p][t] = w4_f32x4{0.f, 0.f, 0.f, 0.f};
          }
        __syncthreads();  // with two halves, one is enough: the other is written next, by waves that are past this
        for (int q = tid >> 8; q < side; q += 2) {
          const int row0 = tid >> 4 & 15, at = ((tid & 12) << 4) + ((row0 ^ (tid & 12)) << 2) + (tid & 3);
          const int64_t col = (int64_t)(tile + q) * kTileRows + (tid & 15);
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            const int row = 16 * t + row0;
            if (row >= rows || col >= n_out) continue;
            float v[kParts];
#pragma unroll
            for (int p = 0; p < kParts; ++p) {
              v[p] = ((const float *)s_part[half][q << lg][p][t])[at];
              for (int w = 1; w < 1 << lg; ++w) v[p] += ((const float *)s_part[half][(q << lg) + w][p][t])[at];
            }
            w4_store<kParts>(out, (m0 + row) * n_out + col, col, v);
          }
        }
        tile += step, i = 0;
        if constexpr (kHalves == 2) half ^= 1;
        else __syncthreads();
      }
    }
  }
}

// More rows, or longer ones: a workgroup takes eight row tiles (of the gated block four, of both matrices), 16 MT rows of x and a run of chunks,
// two a round.  A wave takes every other chunk of two tiles, which share what it reads of x from LDS and the sums of its columns (a tile a wave:
// 24576 x 4096, 64 rows, 40 us instead of 30).  x is asked for three rounds ahead into registers and written to one of two LDS buffers a round
// ahead, weights are asked for two rounds ahead.  Where that leaves some of the chip idle the columns are split over workgroups, and a
// second launch adds the splits up.  4096 x 12288, 64 rows: 21 us, of them 6 rounds of 1.8 us: two waves' 250 vector and 48 matrix instructions each
// a SIMD, which take nearly the sum of their times.
// grid (groups of tiles, tiles of 16 MT rows of x, splits)
template <int MT, int G, bool GATED>
__global__ __launch_bounds__(kWaves * PKV_WAVE, 2) void pkv_w4_kernel(const uint16_t *__restrict__ x, int64_t x_stride, int64_t rows,
                                                                      W4Matrix wa, W4Matrix wb, int64_t n_out, int64_t k, int chunks,
                                                                      int per_split, W4Out out, float *__restrict__ ws) {
  constexpr int kParts = 2, kGroup = GATED ? 4 : 8, kRowVecs = 32, kSlab = 16 * MT * kRowVecs * 16;
  static_assert(kSlab == MT * kWaves * PKV_WAVE * 16, "MT loads of the workgroup a round");
  constexpr int kPart = kWaves * kParts * ((MT + 1) / 2) * PKV_WAVE * 16, kLds = 2 * kSlab > kPart ? 2 * kSlab : kPart;
  __shared__ alignas(16) char lds[kLds];
  const int tid = threadIdx.x, lane = tid & (PKV_WAVE - 1), wave = __builtin_amdgcn_readfirstlane(tid / PKV_WAVE), n = lane & 15, j = lane >> 4;
  const int kg = wave & 1, my_tile = wave >> 1;
  const int64_t tiles = (n_out + kTileRows - 1) / kTileRows, tile0 = (int64_t)blockIdx.x * kGroup, m0 = (int64_t)blockIdx.y * 16 * MT;
  const int m_rows = (int)(rows - m0 < 16 * MT ? rows - m0 : 16 * MT);
  const int first = blockIdx.z * per_split, last = first + per_split < chunks ? first + per_split : chunks, rounds = (last - first + 1) / 2;
  const W4Matrix m[2] = {wa, GATED ? wb : wa};
  const char *w_at[kParts], *s_at[kParts];
#pragma unroll
  for (int p = 0; p < kParts; ++p) {  // a tile of both matrices, or two of one
    int64_t tile = tile0 + my_tile + (GATED ? 0 : 4 * p);
    if (tile >= tiles) tile = tiles - 1;  // past the last: read again, not stored
    w_at[p] = m[p].tiles + tile * chunks * kTileBytes + lane * 16;
    s_at[p] = (const char *)m[p].words + tile * chunks * (kTileCols / G) * (kTileRows * 4) + j * 16;
  }
  auto chunk_of = [&](int i) { return first + 2 * (i < rounds ? i : rounds - 1); };  // past the last: the last again, not used
  auto weights = [&](int i, W4Chunk<G, kParts> &c) {
    const int at = chunk_of(i) + kg;
    c.load(w_at, s_at, at < last ? at : last - 1);
  };
  // Vector my_vec of rows my_row + 16 u of the slab; rows past the last repeat it, columns past the last are read as the
  // first and written as zeros: known for all of a round, so that the others do without (in every round it takes 1 to 3 %).
  const int my_row = tid / kRowVecs, my_vec = tid % kRowVecs;
  const uint16_t *x_at[MT];
#pragma unroll
  for (int u = 0; u < MT; ++u) x_at[u] = x + (m0 + (my_row + 16 * u < m_rows ? my_row + 16 * u : m_rows - 1)) * x_stride;
  auto fetch = [&](int i, pkv_u32x4 (&r)[MT]) {
    const int col = chunk_of(i) * kTileCols + my_vec * 8;
#pragma unroll
    for (int u = 0; u < MT; ++u) r[u] = *(const pkv_u32x4 *)(x_at[u] + (col < k ? col : 0));
  };
  auto put = [&](pkv_u32x4 (&r)[MT], int i) {
    const int buffer = i & 1, chunk = chunk_of(i);
    if (G < kTileCols && (chunk + 2) * kTileCols > k) {  // the whole workgroup
#pragma unroll
      for (int u = 0; u < MT; ++u) r[u] = w4_columns(r[u], chunk * kTileCols + my_vec * 8, k);
    }
#pragma unroll
    for (int u = 0; u < MT; ++u) {
      const int row = my_row + 16 * u;
      *(pkv_u32x4 *)(lds + buffer * kSlab + row * (kRowVecs * 16) + (my_vec >> 4) * 256 + 16 * ((my_vec & 15) ^ (row & 15))) = r[u];
    }
  };
  w4_f32x4 tot[kParts][MT];
#pragma unroll
  for (int p = 0; p < kParts; ++p)
#pragma unroll
    for (int t = 0; t < MT; ++t) tot[p][t] = w4_f32x4{0.f, 0.f, 0.f, 0.f};
  pkv_u32x4 ahead[2][MT];
  W4Chunk<G, kParts> ring[2];
  fetch(0, ahead[0]);
  weights(0, ring[0]);
  fetch(1, ahead[1]);
  weights(1, ring[1]);
  put(ahead[0], 0);
  fetch(2, ahead[0]);
  auto round = [&](int i, pkv_u32x4 (&after)[MT], W4Chunk<G, kParts> &now) {
    __syncthreads();  // round i is there, and everybody is done with round i - 1
    put(after, i + 1);
    fetch(i + 3, after);
    if (i < rounds && chunk_of(i) + kg < last)  // the whole wave
      w4_chunk<MT, G, kParts, false>(now, [&](int t, int s) {
        return *(const pkv_u32x4 *)(lds + (i & 1) * kSlab + (16 * t + n) * (kRowVecs * 16) + kg * 256 + 16 * ((4 * s + j) ^ n));
      }, [](int, int) { return 0.f; }, tot);
    weights(i + 2, now);
  };
  for (int i = 0; i < rounds; i += 2) {  // no way round the second: the waits count what came after on every path
    round(i, ahead[1], ring[0]);
    round(i + 1, ahead[0], ring[1]);
  }
  // Lane (n, j) has rows 4 j .. 4 j + 3 of its tiles for row n of x.  The two waves of a tile exchange halves of their shares: the one with the
  // odd chunks finishes the upper half of the rows of x (of 16 rows: none; of 48 both finish the middle).
  constexpr int kHalf = (MT + 1) / 2;
  w4_f32x4(*const part)[kParts][kHalf][PKV_WAVE] = (w4_f32x4(*)[kParts][kHalf][PKV_WAVE])lds;
  __syncthreads();
#pragma unroll
  for (int p = 0; p < kParts; ++p)
#pragma unroll
    for (int t = kHalf - 1; t >= 0; --t)
      if (kg) {
        part[wave][p][t][lane] = tot[p][t];
      } else {
        part[wave][p][t][lane] = tot[p][MT - kHalf + t];
        tot[p][MT - kHalf + t] = tot[p][t];
      }
  __syncthreads();
  if (MT == 1 && kg) return;
  const bool by_four = n_out % 4 == 0;
#pragma unroll
  for (int t = 0; t < kHalf; ++t) {
    const int row = 16 * (kg * (MT - kHalf) + t) + n;
    w4_f32x4 v[kParts];
#pragma unroll
    for (int p = 0; p < kParts; ++p) v[p] = tot[p][MT - kHalf + t] + part[wave ^ 1][p][t][lane];
    if (row >= m_rows) continue;
#pragma unroll
    for (int p = 0; p < (GATED && gridDim.z == 1 ? 1 : kParts); ++p) {
      const int64_t col = (tile0 + my_tile + (GATED ? 0 : 4 * p)) * kTileRows + 4 * j, at = (m0 + row) * n_out + col;
      if (gridDim.z > 1) {
        float *const to = ws + (GATED ? (int64_t)blockIdx.z * 2 + p : (int64_t)blockIdx.z) * rows * n_out + at;
        if (by_four && col < n_out) *(w4_f32x4 *)to = v[p];
        else
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (col + r < n_out) to[r] = v[p][r];
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (col + r >= n_out) continue;
          if (GATED) {
            const float both[2] = {v[0][r], v[1][r]};
            w4_store<2>(out, at + r, col + r, both);
          } else {
            const float one[1] = {v[p][r]};
            w4_store<1>(out, at + r, col + r, one);
          }
        }
      }
    }
  }
}

// The splits' shares (at most MOST), added in their order; all of them are asked for at once, those that are not there as the last one again.
constexpr int kMaxSplits = 16;
template <bool GATED, int MOST>
__global__ __launch_bounds__(256) void pkv_w4_sum_kernel(const float *__restrict__ ws, int splits, int64_t n_out, W4Out out) {
  constexpr int kParts = GATED ? 2 : 1;
  const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x, at = blockIdx.y * n_out + col, n_all = gridDim.y * n_out;
  if (col >= n_out) return;
  float got[kParts][MOST], v[kParts];
#pragma unroll
  for (int p = 0; p < kParts; ++p)
#pragma unroll
    for (int s = 0; s < MOST; ++s) got[p][s] = ws[((s < splits ? s : splits - 1) * (int64_t)kParts + p) * n_all + at];
#pragma unroll
  for (int p = 0; p < kParts; ++p) {
    v[p] = got[p][0];
#pragma unroll
    for (int s = 1; s < MOST; ++s) v[p] = s < splits ? v[p] + got[p][s] : v[p];
  }
  w4_store<kParts>(out, at, col, v);
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

// How a product is taken, 16 mt rows of x at a time: those that fit into LDS stay there (xkb: how much of it) while `workgroups` workgroups go through the
// matrix, 1 << lg waves to a tile; else they are streamed, the columns in `splits` runs of per_split chunks.
struct W4Plan {
  int xkb, mt, splits, per_split, lg;
  int64_t row_tiles, workgroups;
};
W4Plan w4_plan(int64_t rows, int64_t n, int64_t k, bool gated) {
  W4Plan p = {0, 1, 1, 0, 0, 1, 0};
  const int64_t chunks = w4_chunks(k), tiles = w4_tiles(n);
  p.mt = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  p.row_tiles = (rows + 16 * p.mt - 1) / (16 * p.mt);
  const int64_t x_bytes = (rows < 16 * p.mt ? rows : 16 * p.mt) * chunks * kTileCols * 2;
  // 16 rows of more than 3840 columns do not fit.  us, 15 rows (kept) / 16 (streamed), groups of 32, 64, 128: 6144 x 4096 12.6 / 12.1, 11.1 / 10.1,
  // 9.8 / 9.3; gated 12288 x 4096 21.3 / 24.5, 18.9 / 17.9, 16.4 / 15.2.
  // More than 16 rows, streamed / kept in LDS, us: 96164 x 640, 87 rows 57 / 36; 38959 x 1152, 51 rows 28 / 22, 24 rows 18.5 / 15.0; 3000 x 896,
  // 60 rows 11.4 / 8.8.  The gated block has to join two matrices' shares of more rows than there is room for: 12288 x 1536, 24 rows 9.6 / 12.6.
  const int xkb = p.mt > 1 ? 120 : x_bytes <= 16 * 1024 ? 16 : x_bytes <= 64 * 1024 ? 64 : 120;
  if (x_bytes <= xkb * 1024 && (p.mt == 1 || !gated)) {
    p.xkb = xkb;
    auto groups = [&](int lg) { return (tiles + (kWaves >> lg) - 1) / (kWaves >> lg); };
    if (p.mt == 1) {
      p.lg = chunks <= 1 ? 0 : chunks <= 2 ? 1 : chunks <= 4 ? 2 : 3;
      // One workgroup a compute unit reads x once for it; two, where they fit, hide more of each other's waits, which pays from five tiles each.
      // us with 256 / 512 of them: 6144 x 4096, 8 rows, 7.8 / 8.7; 16384 x 1024, 1 row, 6.0 / 6.3; 32768 x 4096, 1 row, 17.4 / 15.5;
      // 151936 x 4096, 8 rows, 80 / 63; the gated block, 12288 x 4096, 1 row, 12.9 / 14.5, 65536 x 2048, 34.5 / 37.9
      p.workgroups = !gated && p.xkb <= 64 && groups(p.lg) > 1024 ? 512 : 256;
    } else {
      // as many waves to a tile as leave the longest workgroup the fewest chunks, one of them for the tile's end
      p.workgroups = 256 / p.row_tiles > 0 ? 256 / p.row_tiles : 1;
      int64_t best = -1;
      for (int lg = 3; lg >= 0; --lg) {
        const int64_t per_wave = (chunks + (1 << lg) - 1) >> lg, cost = (groups(lg) + p.workgroups - 1) / p.workgroups * (per_wave + 1);
        if (best < 0 || cost < best) best = cost, p.lg = lg;
      }
    }
    if (p.workgroups > groups(p.lg)) p.workgroups = groups(p.lg);
    return p;
  }
  // Tiles of up to 64 rows, as even as they can be.  us, 48 rows as one tile of three times 16 / of four: gated 12288 x 4096 24.8 / 28.9;
  // 76 rows as two of three / of four: 7159 x 9344 31.8 / 37.0.
  const int64_t even = (rows + 63) / 64;
  p.mt = (int)(((rows + even - 1) / even + 15) / 16);
  p.row_tiles = (rows + 16 * p.mt - 1) / (16 * p.mt);
  const int64_t groups = (gated ? (w4_tiles(n) + 3) / 4 : (w4_tiles(n) + 7) / 8) * p.row_tiles;
  // Columns are split where the tiles leave compute units idle and there are more than four rounds, into runs of at least two rounds.  us, runs of at
  // least four rounds and at most 8 of them / these: 1077 x 1824, 43 rows 19.7 / 14.5; 374 x 12480, 44 rows 17.4 / 13.5; 4096 x 12288, 64 rows 22.5 both.
  int64_t s = chunks > 8 ? 256 / groups : 1, most = chunks / 4;
  if (s > most) s = most;
  if (s > kMaxSplits) s = kMaxSplits;
  if (s < 1) s = 1;
  p.per_split = (int)(((chunks + s - 1) / s + 1) / 2 * 2);
  p.splits = (int)((chunks + p.per_split - 1) / p.per_split);
  return p;
}
size_t w4_ws_floats(const W4Plan &p, int64_t rows, int64_t n, bool gated) { return p.splits == 1 ? 0 : (size_t)p.splits * (gated ? 2 : 1) * rows * n; }

template <bool GATED>
int w4_launch(const void *x, int64_t x_stride, int64_t rows, W4Matrix a, W4Matrix b, int64_t n, int64_t k, int group, const void *bias,
              void *y, int out_f32, void *ws, size_t ws_bytes, hipStream_t s) {
  const W4Plan p = w4_plan(rows, n, k, GATED);
  const int64_t tiles = w4_tiles(n), chunks = w4_chunks(k);
  PKV_REQUIRE(p.row_tiles <= 65535, "pkv_w4: too many rows (%lld)", (long long)rows);
  const size_t need = w4_ws_floats(p, rows, n, GATED) * sizeof(float);
  if (need && (!ws || ws_bytes < need || !pkv_aligned(ws, 16))) {
    pkv_set_error("pkv_w4: workspace of %zu bytes required, got %zu", need, ws ? ws_bytes : (size_t)0);
    return PKV_ENOMEM;
  }
  const W4Out out = {(const uint16_t *)bias, y, out_f32};
  const dim3 block(kWaves * PKV_WAVE);
  if (p.xkb) {
    const int64_t groups = (tiles + (kWaves >> p.lg) - 1) / (kWaves >> p.lg);
    const dim3 grid((unsigned)p.workgroups, (unsigned)p.row_tiles);
    const int row_vecs = (int)chunks * (kTileCols / 8), by_row_vecs = ((1 << 24) + row_vecs - 1) / row_vecs;  // v / row_vecs = v by_row_vecs >> 24, v <= 512
#define PKV_W4_X(MT, G, XKB)                                                                                                       \
  hipLaunchKernelGGL((pkv_w4_resident_kernel<MT, G, GATED, XKB, (GATED && G == 32) ? 2 : 4>), grid, block, 0, s, (const uint16_t *)x, \
                     x_stride, rows, a, b, n, (int)k, (int)chunks, by_row_vecs, p.lg, (int)(groups / grid.x), (int)(groups % grid.x), out)
#define PKV_W4_G(G)                                        \
  do {                                                     \
    if (p.mt == 4) PKV_W4_X(GATED ? 1 : 4, G, 120);        \
    else if (p.mt == 2) PKV_W4_X(GATED ? 1 : 2, G, 120);   \
    else if (p.xkb == 16) PKV_W4_X(1, G, 16);              \
    else if (p.xkb == 64) PKV_W4_X(1, G, 64);              \
    else PKV_W4_X(1, G, 120);                              \
  } while (0)
    if (group == 32) PKV_W4_G(32);
    else if (group == 64) PKV_W4_G(64);
    else PKV_W4_G(128);
#undef PKV_W4_G
#undef PKV_W4_X
    PKV_LAUNCH_CHECK("pkv_w4_resident_kernel");
    return PKV_OK;
  }
  const dim3 grid((unsigned)((tiles + (GATED ? 3 : 7)) / (GATED ? 4 : 8)), (unsigned)p.row_tiles, (unsigned)p.splits);
#define PKV_W4(MT, G)                                                                                                              \
  hipLaunchKernelGGL((pkv_w4_kernel<MT, G, GATED>), grid, block, 0, s, (const uint16_t *)x, x_stride, rows, a, b, n, k, (int)chunks, \
                     p.per_split, out, (float *)ws)
#define PKV_W4_G(MT)                    \
  do {                                  \
    if (group == 32) PKV_W4(MT, 32);    \
    else if (group == 64) PKV_W4(MT, 64); \
    else PKV_W4(MT, 128);               \
  } while (0)
  if (p.mt == 1) PKV_W4_G(1);
  else if (p.mt == 2) PKV_W4_G(2);
  else if (p.mt == 3) PKV_W4_G(3);
  else PKV_W4_G(4);
#undef PKV_W4_G
#undef PKV_W4
  PKV_LAUNCH_CHECK("pkv_w4_kernel");
  if (p.splits > 1) {
    const dim3 sum_grid((unsigned)((n + 255) / 256), (unsigned)rows);
#define PKV_W4_SUM(MOST) hipLaunchKernelGGL((pkv_w4_sum_kernel<GATED, MOST>), sum_grid, dim3(256), 0, s, (const float *)ws, p.splits, n, out)
    if (p.splits <= 2) PKV_W4_SUM(2);
    else if (p.splits <= 4) PKV_W4_SUM(4);
    else if (p.splits <= 8) PKV_W4_SUM(8);
    else PKV_W4_SUM(kMaxSplits);
#undef PKV_W4_SUM
    PKV_LAUNCH_CHECK("pkv_w4_sum_kernel");
  }
  return PKV_OK;
}

int w4_check_x(const void *x, int64_t x_stride, int64_t rows, int64_t n, int64_t k, const void *y) {
  PKV_REQUIRE(x && y, "pkv_w4: null pointer");
  PKV_REQUIRE(rows > 0 && rows < ((int64_t)1 << 22) && rows * n < ((int64_t)1 << 39), "pkv_w4: bad row count %lld", (long long)rows);
  PKV_REQUIRE(pkv_aligned(x, 16) && (rows == 1 || (x_stride % 8 == 0 && x_stride >= k)),
              "pkv_w4: rows of x must be 16-byte aligned and not overlap");
  return PKV_OK;
}

}  // namespace

extern "C" size_t pkv_w4_bytes(int64_t n, int64_t k, int group) {
  if (!w4_shape_ok(n, k, group)) return 0;
  return (size_t)(w4_tiles(n) * w4_chunks(k)) * (kTileBytes + kTileCols / group * kTileRows * 4);
}

extern "C" size_t pkv_w4_ws_bytes(int64_t rows, int64_t n, int64_t k, int group, int gated) {
  if (!w4_shape_ok(n, k, group) || rows <= 0 || rows >= ((int64_t)1 << 22)) return 0;
  return w4_ws_floats(w4_plan(rows, n, k, gated != 0), rows, n, gated != 0) * sizeof(float);
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
                             const void *bias, void *y, int out_dtype, void *ws, size_t ws_bytes, void *stream) {
  PKV_REQUIRE(packed && pkv_aligned(packed, 16), "pkv_w4_linear: 16-byte aligned weights required");
  PKV_REQUIRE(out_dtype == PKV_DTYPE_F32 || out_dtype == PKV_DTYPE_BF16, "unknown dtype %d", out_dtype);
  PKV_W4_SHAPE("pkv_w4_linear");
  const int rc = w4_check_x(x, x_stride, rows, n, k, y);
  if (rc) return rc;
  return w4_launch<false>(x, x_stride, rows, w4_matrix(packed, n, k), W4Matrix{}, n, k, group, bias, y, out_dtype == PKV_DTYPE_F32,
                          ws, ws_bytes, (hipStream_t)stream);
}

extern "C" int pkv_w4_silu_mul(const void *x, int64_t x_stride, int64_t rows, const void *gate, const void *up, int64_t n, int64_t k,
                               int group, void *y, void *ws, size_t ws_bytes, void *stream) {
  PKV_REQUIRE(gate && up && pkv_aligned(gate, 16) && pkv_aligned(up, 16), "pkv_w4_silu_mul: 16-byte aligned weights required");
  PKV_W4_SHAPE("pkv_w4_silu_mul");
  const int rc = w4_check_x(x, x_stride, rows, n, k, y);
  if (rc) return rc;
  return w4_launch<true>(x, x_stride, rows, w4_matrix(gate, n, k), w4_matrix(up, n, k), n, k, group, nullptr, y, 0, ws,
                         ws_bytes, (hipStream_t)stream);
}
