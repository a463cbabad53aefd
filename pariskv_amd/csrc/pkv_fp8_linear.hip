// Products of eight-bit rows with eight-bit matrices, a scale for each row of both: y[m][n] = sx[m] sw[n] sum_k xc[m][k] wc[n][k] + bias[n],
// codes e4m3.  (No counterpart in the reference, whose projections are bf16 GEMMs, model_hub/qwen.py:327-383.)
//
// Codes become bf16 numbers in registers, exactly (two to an instruction), and go to bf16 matrix instructions, whose products of them
// are exact and whose sums are fp32.  The instructions that take e4m3 codes themselves have twice the rate (4096 rows x (6144 x 4096) 100 us, 193 with bf16
// instructions), but add eight neighbouring products up with nothing below 2^-13 of the largest of them (2^16 + 4 is 2^16): where large products
// of eight cancel, what is left is lost.  They are not used.
// Which columns a lane has is free as long as both operands agree: lane (r, j) takes columns 16 j .. 16 j + 15 and 64 + 16 j .. of a chunk of 128,
// so that the rows of x are read 64 bytes side by side.  The matrix is laid out once in tiles of 16 rows x 128 columns in the order of the lanes.
#include "pkv_fp8.h"

namespace {

typedef __bf16 fp8_bf16x8 __attribute__((ext_vector_type(8)));
typedef float fp8_f32x4 __attribute__((ext_vector_type(4)));
typedef float fp8_f32x16 __attribute__((ext_vector_type(16)));

constexpr int kTileRows = 16, kTileCols = 128, kTileBytes = kTileRows * kTileCols;

struct Codes {  // 32 codes of a lane
  pkv_u32x4 half[2];
  // a quarter of them as bf16 numbers
  __device__ __forceinline__ pkv_u32x4 part(int p) const {
    const uint32_t a = half[p >> 1][2 * (p & 1)], b = half[p >> 1][2 * (p & 1) + 1];
    return pkv_u32x4{fp8_bf16x2<false>(a), fp8_bf16x2<true>(a), fp8_bf16x2<false>(b), fp8_bf16x2<true>(b)};
  }
};
__device__ __forceinline__ fp8_f32x4 fp8_mfma_part(pkv_u32x4 a, pkv_u32x4 b, fp8_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(fp8_bf16x8, a), __builtin_bit_cast(fp8_bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ fp8_f32x16 fp8_mfma32_part(pkv_u32x4 a, pkv_u32x4 b, fp8_f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(fp8_bf16x8, a), __builtin_bit_cast(fp8_bf16x8, b), c, 0, 0, 0);
}
// Until at most LEFT of this wave's loads are on their way, and none of its reads of LDS; the instructions before stay before.
template <int LEFT>
__device__ __forceinline__ void fp8_wait() {
  static_assert(LEFT >= 0 && LEFT < 64, "six bits");
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LEFT) : "memory");
}

// Order of the instructions since the last barrier: between the matrix instructions the reads of LDS first, then the loads, evenly.
template <int MFMA, int READS, int LOADS>
__device__ __forceinline__ void fp8_mix() {
  constexpr int kHalf = MFMA > 1 ? MFMA / 2 : 1, kReads = (READS + kHalf - 1) / kHalf, kLoads = (LOADS + kHalf - 1) / kHalf;
#pragma unroll
  for (int i = 0; i < MFMA; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if (i * kReads < READS) __builtin_amdgcn_sched_group_barrier(0x100, kReads, 0);
    else if (kLoads > 0) __builtin_amdgcn_sched_group_barrier(0x010, kLoads, 0);
  }
}

struct LinearArgs {
  const uint8_t *x;     // [m], rows x_stride bytes apart, chunks * 128 of them read
  int64_t x_stride;
  const float *sx;
  const uint8_t *tiles; // [row tile][chunk][half][lane] of 16 bytes
  const float *sw;      // [row tiles * 16]
  const uint16_t *bias; // or null
  void *y;
  int64_t m, n;
  int chunks, f32;
  float *part;         // splits > 1: sums of each split's columns, [split][m][part_n], part_n = n rounded up to 4
  int64_t part_n;
  int splits;
};

// Scales as m 2^e, |m| < 1: sums of codes are 0 or of 2^-18 to 2^38, so sum mx mw is far from fp32's ends whatever the scales are, and only the result
// itself can pass them.  (sum sx sw overflows on the way for sx = 2^107, sw = 2^-25.)
struct Scale {
  float m;
  int e;
  __device__ __forceinline__ explicit Scale(float s) : m(__builtin_amdgcn_frexp_mantf(s)), e(__builtin_amdgcn_frexp_expf(s)) {}
};
__device__ __forceinline__ float scaled(float sum, const Scale &x, const Scale &w) { return __builtin_ldexpf(sum * x.m * w.m, x.e + w.e); }

// Columns col .. col + 3 of a row of y, col a multiple of four.  WHOLE: rows of y are whole vectors.  The flags are chosen once for all of a
// workgroup's results: asked for at each of the 64 a lane may have, they take longer than eight chunks of columns (20 us of 256 x 256).
template <bool F32, bool BIAS, bool WHOLE>
__device__ __forceinline__ void put4(const LinearArgs &a, int64_t row, int64_t col, fp8_f32x4 sum, float sx) {
  if (row >= a.m || col >= a.n) return;
  const fp8_f32x4 sw = *(const fp8_f32x4 *)(a.sw + col);  // there are scales up to the next multiple of 16
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = scaled(sum[i], Scale(sx), Scale(sw[i]));
  if constexpr (BIAS) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += pkv_bf16_bits_to_f32(a.bias[WHOLE || col + i < a.n ? col + i : col]);
  }
  const int64_t at = row * a.n + col;
  if (WHOLE || col + 4 <= a.n) {
    struct __attribute__((packed)) Four {
      uint32_t w[F32 ? 4 : 2];
    } o;
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) o.w[i] = __float_as_uint(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) o.w[i] = (uint32_t)pkv_f32_to_bf16_bits(v[2 * i]) | ((uint32_t)pkv_f32_to_bf16_bits(v[2 * i + 1]) << 16);
    }
    __builtin_memcpy((char *)a.y + at * (F32 ? 4 : 2), &o, sizeof o);  // the memory takes it at any alignment
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (col + i >= a.n) break;
      if constexpr (F32) ((float *)a.y)[at + i] = v[i];
      else ((uint16_t *)a.y)[at + i] = pkv_f32_to_bf16_bits(v[i]);
    }
  }
}
// f(put4 of this call)
template <typename F>
__device__ __forceinline__ void with_put4(const LinearArgs &a, F f) {
  const bool whole = (a.n & 3) == 0;
#define PKV_PUT(F32, BIAS, WHOLE) f([&](int64_t row, int64_t col, fp8_f32x4 sum, float sx) { put4<F32, BIAS, WHOLE>(a, row, col, sum, sx); })
  if (whole && !a.bias) {
    if (a.f32) PKV_PUT(true, false, true);
    else PKV_PUT(false, false, true);
  } else if (whole) {
    if (a.f32) PKV_PUT(true, true, true);
    else PKV_PUT(false, true, true);
  } else if (a.bias) {
    if (a.f32) PKV_PUT(true, true, false);
    else PKV_PUT(false, true, false);
  } else {
    if (a.f32) PKV_PUT(true, false, false);
    else PKV_PUT(false, false, false);
  }
#undef PKV_PUT
}

// Few rows: the matrix is read once and the bytes bound it.  A workgroup takes 16 RT rows of the matrix and 16 MT of x, its waves every
// kStreamWaves-th chunk of columns, straight from memory into the operands; they meet in LDS, in their order.
constexpr int kStreamWaves = 8;
template <int MT, int RT>
__global__ __launch_bounds__(kStreamWaves * PKV_WAVE) void pkv_fp8_stream_kernel(LinearArgs a) {
  constexpr int kAhead = MT + RT > 4 ? 1 : MT + RT > 3 ? 2 : 4;  // chunks under way
  __shared__ fp8_f32x4 s_part[kStreamWaves][RT][MT][PKV_WAVE];
  const int tid = threadIdx.x, lane = pkv_lane(), wave = tid / PKV_WAVE, n = lane & 15, j = lane >> 4;
  const int64_t tiles = (a.n + kTileRows - 1) / kTileRows, m0 = (int64_t)blockIdx.y * 16 * MT, t0 = (int64_t)blockIdx.x * RT;
  const uint8_t *w_at[RT], *x_at[MT];
#pragma unroll
  for (int r = 0; r < RT; ++r) w_at[r] = a.tiles + (t0 + r < tiles ? t0 + r : tiles - 1) * a.chunks * kTileBytes + lane * 16;
#pragma unroll
  for (int t = 0; t < MT; ++t) x_at[t] = a.x + (m0 + 16 * t + n < a.m ? m0 + 16 * t + n : a.m - 1) * a.x_stride + 16 * j;
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
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const pkv_u32x4 wo = w[u][r].part(p);
#pragma unroll
          for (int t = 0; t < MT; ++t) acc[r][t] = fp8_mfma_part(wo, x[u][t].part(p), acc[r][t]);
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < MT; ++t) s_part[wave][r][t][lane] = acc[r][t];
  __syncthreads();
  with_put4(a, [&](auto put) {
    for (int e = tid; e < RT * MT * PKV_WAVE; e += kStreamWaves * PKV_WAVE) {  // a lane's four columns of a tile at a time
      const int r = e / (MT * PKV_WAVE), t = e / PKV_WAVE % MT, l = e % PKV_WAVE;
      fp8_f32x4 sum = s_part[0][r][t][l];
#pragma unroll
      for (int w = 1; w < kStreamWaves; ++w) sum += s_part[w][r][t][l];
      const int64_t row = m0 + 16 * t + (l & 15);
      put(row, (t0 + r) * 16 + 4 * (l >> 4), sum, a.sx[row < a.m ? row : a.m - 1]);
    }
  });
}

// Many rows: 64 TM rows of x by 64 TN of the matrix a workgroup, a quarter of them a wave, a chunk of columns at a time (of its split's), straight from memory to
// LDS.  Of x a load takes 8 rows x 128 columns, whole lines: 64 bytes of each of 16 rows, all in the same half of their lines, come at half the rate
// (16 KB 0.7 us a compute unit; 0.4).  Vector v of row r lies at v ^ (r mod 8) of the row, so that rows of an operand are on different banks.
typedef const __attribute__((address_space(1))) void *fp8_global;
typedef __attribute__((address_space(3))) void *fp8_lds;
// A wave's results, rows m0 .., columns n0 .. of y, past the caches, 32 rows at a time through a part of LDS of its own and out as whole rows of it: 16 bytes of each of
// 32 rows, as they lie in the registers, would take 20 us of 256 x 256 where rows of y are a multiple of 4096 bytes.
// RAW: as sums, to a split's part.
template <int TM, int TN, bool F32, bool RAW>
__device__ __forceinline__ void block_store(const LinearArgs &a, const fp8_f32x16 (&acc)[TN][TM], uint8_t *lds, int64_t m0, int64_t n0) {
  constexpr int kEs = F32 ? 4 : 2, kRow = 32 * TN * kEs, kStep = kRow + 16, kVecs = kRow / 16, kRows = PKV_WAVE / kVecs;
  static_assert(4 * 32 * kStep <= 2 * 4 * (TM + TN) * kTileBytes, "room for it");
  const int lane = pkv_lane(), wave = threadIdx.x / PKV_WAVE, row = lane & 31;
  uint8_t *const mine = lds + wave * (32 * kStep);
  static_assert(F32 || !RAW, "sums are fp32");
  const int64_t n = RAW ? a.part_n : a.n, left = n - n0;  // RAW: past the matrix's last row its last tile has zeros
  const bool whole = n % (16 / kEs) == 0;
  char *const y = RAW ? (char *)(a.part + blockIdx.y * a.m * n) : (char *)a.y;
  const int vec = lane % kVecs, col = vec * (16 / kEs);
#pragma unroll
  for (int t = 0; t < TM; ++t) {
    const Scale sx(a.sx[m0 + 32 * t + row < a.m ? m0 + 32 * t + row : a.m - 1]);
#pragma unroll
    for (int r = 0; r < TN; ++r)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = 32 * r + 8 * q + 4 * (lane >> 5);
        const bool in = c < left;
        const fp8_f32x4 sw = *(const fp8_f32x4 *)(a.sw + (in ? n0 + c : 0));  // there are scales up to the next multiple of 16
        fp8_f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = RAW ? acc[r][t][4 * q + i] : scaled(acc[r][t][4 * q + i], sx, Scale(sw[i]));
        if (!RAW && a.bias) {
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] += pkv_bf16_bits_to_f32(a.bias[c + i < left ? n0 + c + i : 0]);
        }
        if constexpr (F32) *(fp8_f32x4 *)(mine + row * kStep + c * 4) = v;
        else
          *(pkv_u32x2 *)(mine + row * kStep + c * 2) = pkv_u32x2{(uint32_t)pkv_f32_to_bf16_bits(v[0]) | ((uint32_t)pkv_f32_to_bf16_bits(v[1]) << 16),
                                                                 (uint32_t)pkv_f32_to_bf16_bits(v[2]) | ((uint32_t)pkv_f32_to_bf16_bits(v[3]) << 16)};
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    for (int r0 = lane / kVecs; r0 < 32; r0 += kRows) {
      const int64_t at = m0 + 32 * t + r0;
      const pkv_u32x4 v = *(const pkv_u32x4 *)(mine + r0 * kStep + vec * 16);
      if (at >= a.m || col >= left) continue;
      char *const to = y + (at * n + n0 + col) * kEs;
      if (RAW) *(pkv_u32x4 *)to = v;  // read again by the second launch
      else if (whole) __builtin_nontemporal_store(v, (pkv_u32x4 *)to);
      else if (col + 16 / kEs <= left) __builtin_memcpy(to, &v, 16);  // the memory takes it at any alignment
      else
#pragma unroll
        for (int i = 0; i < 16 / kEs; ++i) {
          if (col + i >= left) break;
          if constexpr (F32) ((uint32_t *)to)[i] = v[i];
          else ((uint16_t *)to)[i] = (uint16_t)(v[i >> 1] >> (16 * (i & 1)));
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

template <int TM, int TN, int DEPTH>
__global__ __launch_bounds__(256, TM * TN > 4 ? 1 : 2) void pkv_fp8_block_kernel(LinearArgs a, int m_blocks, int n_blocks) {
  constexpr int kEach = TM + TN, kX = 4 * TM * kTileBytes, kBuffer = kX + 4 * TN * kTileBytes;  // pieces of 1 KB that a wave brings in, of x and of the matrix
  extern __shared__ uint8_t lds[];
  const int lane = pkv_lane(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / PKV_WAVE);
  // Workgroups go to the eight dies in turn: each die takes a run of blocks that share rows.
  const int blocks = m_blocks * n_blocks, per = (blocks + 7) / 8, id = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || id >= blocks) return;  // the whole workgroup
  constexpr int kGroup = 4;  // blocks of x rows side by side
  const int group = id / (kGroup * n_blocks), in = id - group * kGroup * n_blocks, here = m_blocks - group * kGroup < kGroup ? m_blocks - group * kGroup : kGroup;
  const int mb = group * kGroup + in % here, nb = in / here;
  const int64_t tiles = (a.n + kTileRows - 1) / kTileRows, m0 = (int64_t)mb * (64 * TM), t0 = (int64_t)nb * (4 * TN);
  const int wm = wave & 1, wn = wave >> 1, c0 = (int)blockIdx.y * a.chunks / a.splits, last = ((int)blockIdx.y + 1) * a.chunks / a.splits - c0 - 1;
  // what this wave brings in: 8 rows each of x, half tiles of the matrix
  const uint8_t *x_from[2 * TM], *w_from[TN];
#pragma unroll
  for (int u = 0; u < 2 * TM; ++u) {
    const int64_t row = m0 + (wave * 2 * TM + u) * 8 + (lane >> 3);
    x_from[u] = a.x + (row < a.m ? row : a.m - 1) * a.x_stride + c0 * kTileCols + 16 * ((lane & 7) ^ (lane >> 3));
  }
#pragma unroll
  for (int u = 0; u < TN; ++u) {
    const int64_t tile = t0 + wave * TN + u;
    w_from[u] = a.tiles + ((tile < tiles ? tile : tiles - 1) * a.chunks + c0) * kTileBytes + lane * 16;
  }
  auto fetch = [&](int c, int buffer) {
    uint8_t *const to = lds + buffer * kBuffer;
#pragma unroll
    for (int u = 0; u < 2 * TM; ++u)
      __builtin_amdgcn_global_load_lds((fp8_global)(x_from[u] + c * kTileCols), (fp8_lds)(to + (wave * 2 * TM + u) * 1024), 16, 0, 0);
#pragma unroll
    for (int u = 0; u < TN; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        __builtin_amdgcn_global_load_lds((fp8_global)(w_from[u] + (int64_t)c * kTileBytes + h * 1024), (fp8_lds)(to + kX + (wave * TN + u) * kTileBytes + h * 1024),
                                         16, 0, 0);
  };
  // operands: row lane mod 32 of a pair of tiles, vectors 4 half + 2 (lane / 32) + e of its chunk
  const int row = lane & 31, x_row = wm * TM * 4096 + (row >> 3) * 1024 + (row & 7) * 128, w_row = kX + wn * TN * 4096 + (row >> 4) * 2048 + (row & 15) * 16;
  int x_vec[2][2];
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int e = 0; e < 2; ++e) x_vec[half][e] = x_row + 16 * ((4 * half + 2 * (lane >> 5) + e) ^ (row & 7));
  const int w_vec = w_row + (lane >> 5) * 512;
  auto read = [&](int buffer, int half, Codes (&x)[TM], Codes (&w)[TN]) {
    const uint8_t *const p = lds + buffer * kBuffer;
#pragma unroll
    for (int t = 0; t < TM; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) x[t].half[e] = *(const pkv_u32x4 *)(p + x_vec[half][e] + t * 4096);
#pragma unroll
    for (int r = 0; r < TN; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) w[r].half[e] = *(const pkv_u32x4 *)(p + w_vec + half * 1024 + e * 256 + r * 4096);
  };
  fp8_f32x16 acc[TN][TM];
#pragma unroll
  for (int r = 0; r < TN; ++r)
#pragma unroll
    for (int t = 0; t < TM; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[r][t][i] = 0.f;
  auto product = [&](const Codes (&x)[TM], const Codes (&w)[TN]) {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      pkv_u32x4 xo[TM];
#pragma unroll
      for (int t = 0; t < TM; ++t) xo[t] = x[t].part(p);
#pragma unroll
      for (int r = 0; r < TN; ++r) {
        const pkv_u32x4 wo = w[r].part(p);
#pragma unroll
        for (int t = 0; t < TM; ++t) acc[r][t] = fp8_mfma32_part(wo, xo[t], acc[r][t]);
      }
    }
  };
  // Operands of the next half chunk are read while this one's are multiplied; a chunk is asked for when the one DEPTH before it has been
  // read, half a chunk before its end.
  Codes x[2][TM], w[2][TN];
#pragma unroll
  for (int c = 0; c < DEPTH; ++c) fetch(c < last ? c : last, c);  // past the last: read again, not used
  fp8_wait<(DEPTH - 1) * 2 * kEach>();
  __builtin_amdgcn_s_barrier();
  read(0, 0, x[0], w[0]);
  int now = 0;
  for (int c = 0; c <= last; ++c) {
    const int next = now + 1 == DEPTH ? 0 : now + 1;
    read(now, 1, x[1], w[1]);
    product(x[0], w[0]);
    fp8_mix<4 * TM * TN, 2 * (TM + TN), 0>();
    fp8_wait<(DEPTH - 2) * 2 * kEach>();  // chunk c + 1 is there, for this wave, and its reads of chunk c are done
    __builtin_amdgcn_s_barrier();         // ... for all
    fetch(c + DEPTH < last ? c + DEPTH : last, now);
    read(next, 0, x[0], w[0]);
    product(x[1], w[1]);
    fp8_mix<4 * TM * TN, 2 * (TM + TN), 2 * kEach>();
    __builtin_amdgcn_sched_barrier(0);
    now = next;
  }
  fp8_wait<0>();  // nothing may be on its way to LDS that another workgroup gets
  __builtin_amdgcn_s_barrier();
  if (a.splits > 1) block_store<TM, TN, true, true>(a, acc, lds, m0 + TM * wm * 32, t0 * 16 + TN * wn * 32);
  else if (a.f32) block_store<TM, TN, true, false>(a, acc, lds, m0 + TM * wm * 32, t0 * 16 + TN * wn * 32);
  else block_store<TM, TN, false, false>(a, acc, lds, m0 + TM * wm * 32, t0 * 16 + TN * wn * 32);
}

// The splits' sums, in their order: four columns a thread.
__global__ __launch_bounds__(256) void pkv_fp8_sum_kernel(LinearArgs a) {
  const uint32_t at = blockIdx.x * 256 + threadIdx.x, across = (uint32_t)a.part_n / 4, row = at / across, col = 4 * (at - row * across);
  if (row >= a.m) return;
  const float *const from = a.part + (int64_t)row * a.part_n + col;
  fp8_f32x4 sum = *(const fp8_f32x4 *)from;
#pragma unroll 4
  for (int i = 1; i < a.splits; ++i) sum += *(const fp8_f32x4 *)(from + i * a.m * a.part_n);
  with_put4(a, [&](auto put) { put(row, col, sum, a.sx[row]); });
}

template <int MT, int RT>
void launch_stream(const LinearArgs &a, hipStream_t s) {
  const unsigned tiles = (unsigned)((a.n + kTileRows - 1) / kTileRows);
  hipLaunchKernelGGL((pkv_fp8_stream_kernel<MT, RT>), dim3((tiles + RT - 1) / RT, (unsigned)((a.m + 16 * MT - 1) / (16 * MT))), dim3(kStreamWaves * PKV_WAVE), 0, s, a);
}

template <int TM, int TN, int DEPTH>
int launch_block(const LinearArgs &a, hipStream_t s) {
  const int mb = (int)((a.m + 64 * TM - 1) / (64 * TM)), nb = (int)((a.n + 64 * TN - 1) / (64 * TN));
  const int lds = DEPTH * 4 * (TM + TN) * kTileBytes;
  PKV_HIP(hipFuncSetAttribute((const void *)pkv_fp8_block_kernel<TM, TN, DEPTH>, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
  hipLaunchKernelGGL((pkv_fp8_block_kernel<TM, TN, DEPTH>), dim3((unsigned)((mb * (int64_t)nb + 7) / 8 * 8), (unsigned)a.splits), dim3(256), lds, s, a, mb, nb);
  PKV_LAUNCH_CHECK("pkv_fp8_block_kernel");
  if (a.splits > 1) {
    hipLaunchKernelGGL(pkv_fp8_sum_kernel, dim3((unsigned)((a.m * (a.part_n / 4) + 255) / 256)), dim3(256), 0, s, a);
    PKV_LAUNCH_CHECK("pkv_fp8_sum_kernel");
  }
  return PKV_OK;
}

int64_t row_tiles(int64_t n) { return (n + kTileRows - 1) / kTileRows; }
int chunks_of(int64_t k) { return (int)((k + kTileCols - 1) / kTileCols); }
size_t tile_bytes(int64_t n, int64_t k) { return (size_t)row_tiles(n) * chunks_of(k) * kTileBytes; }

// What a workgroup takes: 16 MT rows of x by 16 RT of the matrix (stream), 64 TM by 64 TN (block).
enum Shape { kStream11, kStream12, kStream14, kStream22, kStream24, kBlock11, kBlock12, kBlock21, kBlock22, kBlock22Two };

struct Plan {
  Shape shape;
  int splits;
};
struct Kind {
  int bm, bn, at_once;
  double start, each, rate;  // KB a us of a compute unit
};
const Kind kKinds[] = {{16, 16, 1, 2.4, 0.85, 43}, {16, 32, 1, 2.4, 0.85, 43}, {16, 64, 1, 2.4, 0.85, 43},   {32, 32, 1, 2.4, 0.85, 43}, {32, 64, 1, 2.4, 0.85, 43},
                       {64, 64, 1, 4.5, 2.5, 58},  {64, 128, 1, 4.5, 3.5, 57},  {128, 64, 1, 4.5, 3.5, 53},  {128, 128, 1, 4.5, 5.0, 36}, {128, 128, 2, 4.5, 5.0, 44}};
static_assert(sizeof kKinds / sizeof kKinds[0] == kBlock22Two + 1, "a row a shape");

// The shape and number of splits of the least estimate, in us: a start, and for each round of workgroups (one to a compute unit; of kBlock22Two two)
// another one and what they read at what a compute unit takes in with that shape, or the matrix at what memory gives, whichever is longer and a tenth of the other; splits write their sums, read again by a
// second launch.  Over 180 products of 1 .. 4096 rows with matrices of 64 .. 150 000 rows and 100 .. 16 384 columns, half of them with bf16 results, its choice takes 3 % more
// than the best of all shapes and splits (up to 16, of four chunks at least), 1.3 times at the worst.  us, bf16 results: 1 x (4096 x 4096), 16x16 / 16x64 stream 5.3 / 8.8;
// 22 x (9637 x 4096) 18.7 / 19.0, 32x64 11.1; 294 x (1840 x 4096), 32x64 stream 22.3, 64x64 block 15.9, 16.8 in two splits; 256 x (28672 x 4096) 155 and 86, 64x128 69;
// 145 x (955 x 12288), 64x64 block in 1 / 4 / 5 / 8 splits 35.8 / 16.1 / 14.8 / 15.9; 128x128 blocks, one to a compute unit with four buffers / two with two:
// 4096 x (6144 x 4096) 206 / 176-190, 1024 x (4096 x 4096) 36.9 / 35.6.
Plan linear_plan(int64_t m, int64_t n, int64_t k) {
  const int chunks = chunks_of(k);
  Plan best = {kStream11, 1};
  double least = 0;
  // up to 16 rows, streams only: 16 x (3208 x 12288) 13.0 us, the best split block 16.1; 3 x (363 x 12288) 7.2 and 10.3
  for (int i = 0; i <= (m <= 16 ? kStream24 : kBlock22Two); ++i) {
    const Kind &q = kKinds[i];
    const int64_t groups = (m + q.bm - 1) / q.bm * ((n + q.bn - 1) / q.bn);
    if (q.at_once > 1 && groups <= 256) continue;
    const int most = i < kBlock11 || q.at_once > 1 || chunks < 8 ? 1 : chunks < 64 ? chunks / 4 : 16;
    for (int s = 1; s <= most && (s == 1 || groups * s <= 512); ++s) {
      const int64_t round = 256 * q.at_once, whole = (groups * s + round - 1) / round;
      // workgroups that the vector instructions bound, which make bf16 numbers of codes, end less in step
      const double rounds = whole == 1 ? 1.0 : 0.6 * (double)whole + 0.4 * (double)(groups * s) / (double)round;
      const double reads = 0.128 * ((chunks + s - 1) / s) * ((m < q.bm ? m : q.bm) + q.bn) * q.at_once;
      const double units = rounds * (reads / q.rate + q.each), memory = (double)n * (double)k / 6e6;
      const double us = q.start + (units > memory ? units + 0.1 * memory : memory + 0.1 * units) + (s > 1 ? 1.25e-6 * s * (double)m * (double)n : 0.0);
      if ((i == 0 && s == 1) || us < least) best = {(Shape)i, s}, least = us;
    }
  }
  return best;
}

// Codes [n][k] into tiles, one 16-byte vector of a tile a thread at a time, and back, element by element.  A launch has fewer than 2^32 threads.
constexpr int64_t kMostBlocks = (int64_t)1 << 23;
__global__ __launch_bounds__(256) void pkv_fp8_pack_kernel(const uint8_t *__restrict__ codes, const float *__restrict__ scales, int64_t n, int64_t k,
                                                           int64_t stride, int chunks, int64_t vecs, uint8_t *__restrict__ tiles, float *__restrict__ sw) {
  const int64_t rows = (n + kTileRows - 1) / kTileRows * kTileRows;
  for (int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x; v < vecs; v += kMostBlocks * 256) {
    if (v < rows) sw[v] = v < n ? scales[v] : 0.f;  // there are more vectors than rows
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
}

__global__ __launch_bounds__(256) void pkv_fp8_unpack_kernel(const uint8_t *__restrict__ tiles, const float *__restrict__ sw, int64_t n, int64_t k,
                                                             int chunks, float *__restrict__ w) {
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n * k; e += kMostBlocks * 256) {
    const int64_t row = e / k, col = e - row * k;
    const int in = (int)(col & 127);
    const uint8_t code = tiles[((row >> 4) * chunks + (col >> 7)) * kTileBytes + (in >> 6) * 1024 + (((in & 63) >> 4) * 16 + (row & 15)) * 16 + (in & 15)];
    w[e] = __builtin_amdgcn_cvt_pk_f32_fp8((int)code, false)[0] * sw[row];
  }
}

bool matrix_ok(int64_t n, int64_t k) { return n > 0 && n < ((int64_t)1 << 31) - 16 && k > 0 && k <= ((int64_t)1 << 20); }
bool rows_ok(int64_t rows, int64_t n, int64_t k) { return matrix_ok(n, k) && rows > 0 && rows <= ((int64_t)1 << 22) && rows * n <= ((int64_t)1 << 40); }

}  // namespace

extern "C" size_t pkv_fp8_bytes(int64_t n, int64_t k) {
  if (!matrix_ok(n, k)) return 0;
  return tile_bytes(n, k) + (size_t)row_tiles(n) * kTileRows * sizeof(float);
}

extern "C" int pkv_fp8_pack(const uint8_t *codes, int64_t row_stride, const float *scales, int64_t n, int64_t k, void *packed, void *stream) {
  PKV_REQUIRE(codes && scales && packed, "pkv_fp8_pack: null pointer");
  PKV_REQUIRE(matrix_ok(n, k) && row_stride >= k, "pkv_fp8_pack: bad matrix %lld x %lld", (long long)n, (long long)k);
  PKV_REQUIRE(pkv_aligned(packed, 16) && pkv_aligned(scales, 4), "pkv_fp8_pack: 16-byte aligned buffers required");
  const int64_t vecs = (int64_t)(tile_bytes(n, k) / 16), blocks = (vecs + 255) / 256;
  hipLaunchKernelGGL(pkv_fp8_pack_kernel, dim3((unsigned)(blocks < kMostBlocks ? blocks : kMostBlocks)), dim3(256), 0, (hipStream_t)stream, codes, scales, n, k, row_stride,
                     chunks_of(k), vecs, (uint8_t *)packed, (float *)((uint8_t *)packed + tile_bytes(n, k)));
  PKV_LAUNCH_CHECK("pkv_fp8_pack_kernel");
  return PKV_OK;
}

extern "C" int pkv_fp8_unpack(const void *packed, int64_t n, int64_t k, float *w, void *stream) {
  PKV_REQUIRE(packed && w, "pkv_fp8_unpack: null pointer");
  PKV_REQUIRE(matrix_ok(n, k) && pkv_aligned(packed, 16), "pkv_fp8_unpack: bad matrix %lld x %lld", (long long)n, (long long)k);
  const int64_t blocks = (n * k + 255) / 256;
  hipLaunchKernelGGL(pkv_fp8_unpack_kernel, dim3((unsigned)(blocks < kMostBlocks ? blocks : kMostBlocks)), dim3(256), 0, (hipStream_t)stream, (const uint8_t *)packed,
                     (const float *)((const uint8_t *)packed + tile_bytes(n, k)), n, k, chunks_of(k), w);
  PKV_LAUNCH_CHECK("pkv_fp8_unpack_kernel");
  return PKV_OK;
}

extern "C" size_t pkv_fp8_linear_ws_bytes(int64_t rows, int64_t n, int64_t k, int /*out_dtype: the same for all*/) {
  if (!rows_ok(rows, n, k)) return 0;
  const int splits = linear_plan(rows, n, k).splits;
  return splits == 1 ? 0 : (size_t)splits * rows * ((n + 3) / 4 * 4) * sizeof(float);
}

extern "C" int pkv_fp8_linear_plan(int64_t rows, int64_t n, int64_t k, int *plan) {
  PKV_REQUIRE(plan, "pkv_fp8_linear_plan: null pointer");
  PKV_REQUIRE(rows_ok(rows, n, k), "pkv_fp8_linear_plan: bad shape %lld rows, %lld x %lld", (long long)rows, (long long)n, (long long)k);
  const Plan p = linear_plan(rows, n, k);
  const Kind &q = kKinds[p.shape];
  plan[0] = q.bm, plan[1] = q.bn, plan[2] = p.splits, plan[3] = q.at_once;
  return PKV_OK;
}

extern "C" int pkv_fp8_linear(const uint8_t *x, int64_t x_stride, const float *x_scales, int64_t rows, const void *packed, int64_t n, int64_t k, const void *bias,
                              void *y, int out_dtype, void *ws, size_t ws_bytes, void *stream) {
  PKV_REQUIRE(x && x_scales && packed && y, "pkv_fp8_linear: null pointer");
  PKV_REQUIRE(out_dtype == PKV_DTYPE_F32 || out_dtype == PKV_DTYPE_BF16, "unknown dtype %d", out_dtype);
  PKV_REQUIRE(rows_ok(rows, n, k), "pkv_fp8_linear: bad shape %lld rows, %lld x %lld", (long long)rows, (long long)n, (long long)k);
  PKV_REQUIRE(x_stride % 16 == 0 && x_stride >= (int64_t)chunks_of(k) * kTileCols, "pkv_fp8_linear: rows of x must be 16-byte multiples apart and hold whole chunks of 128");
  PKV_REQUIRE(pkv_aligned(x, 16) && pkv_aligned(packed, 16) && pkv_aligned(x_scales, 4) && pkv_aligned(bias, 2) && pkv_aligned(y, 16), "pkv_fp8_linear: 16-byte aligned operands required");
  LinearArgs a;
  a.x = x, a.x_stride = x_stride, a.sx = x_scales, a.tiles = (const uint8_t *)packed, a.sw = (const float *)((const uint8_t *)packed + tile_bytes(n, k));
  a.bias = (const uint16_t *)bias, a.y = y, a.m = rows, a.n = n, a.chunks = chunks_of(k), a.f32 = out_dtype == PKV_DTYPE_F32;
  hipStream_t s = (hipStream_t)stream;
  const Plan plan = linear_plan(rows, n, k);
  a.splits = plan.splits, a.part_n = (n + 3) / 4 * 4, a.part = (float *)ws;
  const size_t need = a.splits == 1 ? 0 : (size_t)a.splits * rows * a.part_n * sizeof(float);
  if (need && (!ws || ws_bytes < need || !pkv_aligned(ws, 16))) {
    pkv_set_error("pkv_fp8_linear: workspace of %zu bytes required, got %zu", need, ws ? ws_bytes : (size_t)0);
    return PKV_ENOMEM;
  }
  switch (plan.shape) {
    case kStream11: launch_stream<1, 1>(a, s); break;
    case kStream12: launch_stream<1, 2>(a, s); break;
    case kStream14: launch_stream<1, 4>(a, s); break;
    case kStream22: launch_stream<2, 2>(a, s); break;
    case kStream24: launch_stream<2, 4>(a, s); break;
    case kBlock11: return launch_block<1, 1, 4>(a, s);
    case kBlock12: return launch_block<1, 2, 3>(a, s);
    case kBlock21: return launch_block<2, 1, 3>(a, s);
    case kBlock22: return launch_block<2, 2, 4>(a, s);
    default: return launch_block<2, 2, 2>(a, s);
  }
  PKV_LAUNCH_CHECK("pkv_fp8_linear");
  return PKV_OK;
}
