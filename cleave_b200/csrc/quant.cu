// Block quantization to 8 bits, its inverse, and the derivative form of an activation that was kept in 8 bits.
//
// One kernel does all the writing.  A CTA takes a 128 x 128 tile, one block of every form, holds it in registers (32 values a
// thread, all its loads issued before the first use) and makes each form that is asked for from that one read: a warp owns 8
// whole rows of the tile, so a 1 x 128 block's maximum is one warp reduction, and a 128 x 1 block's is a maximum over the
// warp's 8 rows in a register and over the 16 warps in shared memory.  HBM bound: 4 bytes read (5 with a checkpoint) and one
// byte written per element and form.
//
// Scale of a block: s = 2^e with e = ceil(log2(amax / 448)), the smallest power of two that brings the block's largest
// magnitude to at most 448 = 1.75 * 2^8.  With amax = m * 2^E (1 <= m < 2) that is e = E - 8, or E - 7 where m > 1.75: an
// integer addition that carries into the exponent field exactly when the mantissa is above 1.75's.  A power of two costs
// no precision (e4m3 is a floating-point format: only values 2^14 below the block's maximum reach its subnormals) and makes
// x / s, q * s and a later sum of products scaled by s exact.  e is clamped to [-126, 120]; amax = 0 gives -126.
//
// Non-finite values: they do not count for the maximum and are stored as NaN, so one infinity shows up as one NaN, and in
// the sums it takes part in, instead of flushing its block to zero or passing as 448.
#include <cmath>

#include "common.cuh"
#include "quant.cuh"

namespace cleave {

constexpr int kQThreads = 512;
constexpr int kQWarps = kQThreads / 32;
constexpr int kQRows = kQBlock / kQWarps;   // rows of the tile per warp
// Column sums are finished in the kernel up to so many column blocks (counters) and row blocks (the last CTA's walk over them),
// beyond that by colsum_launch.  In the kernel / by a second one, us: 128 row blocks (16384 x 1024) 28.7 / 29.3, 256 49.5 / 47.4,
// 512 99.7 / 88.4, 8192 (1048576 x 128) 398 / 161.
constexpr int kQMaxColBlocks = 4096;
constexpr int kQMaxRowBlocks = 128;

struct TileArgs {
  int rows, cols;
  int row_blocks, col_blocks;   // q_blocks of them: tile_kernel, short of registers, spills less when it need not work them out
                                // (4096 x 4096, tanh, two forms and sums: 28.7 us against 34.6)
  int vec;                // x (and dz) are 16-byte aligned and cols is a multiple of 4
  const float* x;         // [rows, cols]: the values, or the upstream gradient
  const uint8_t* y_q;     // checkpoint of the activation's output (null: plain quantization)
  const float* y_s;
  int y_blocks, act;
  float* dz;              // outputs, each may be null
  uint8_t *q_rows, *q_cols, *q_tiles;
  float *s_rows, *s_cols, *s_tiles;
  float* db_part;         // [row blocks][cols]: column sums of each row block
  float* db;              // their sum, written by the last CTA of each column block (null: left to a second kernel)
};

// Arrivals of a column block's CTAs; each count wraps to zero with the last arrival.  Launches of this library are ordered on
// one stream, so no two of them count at once.
static __device__ unsigned int g_db_arrivals[kQMaxColBlocks];

// Exponent field of a block's largest magnitude after the carry described above, held at 9 or more (a scale of 2^-126);
// scale and 1 / scale follow by one subtraction each.
__device__ __forceinline__ uint32_t amax_exponent(uint32_t amax_bits) {
  const uint32_t e = (amax_bits + 0x1fffffu) & 0x7f800000u;
  return e < (9u << 23) ? 9u << 23 : e;
}
__device__ __forceinline__ float scale_of(uint32_t e) { return __uint_as_float(e - (8u << 23)); }
__device__ __forceinline__ float inverse_scale_of(uint32_t e) { return __uint_as_float((262u << 23) - e); }

// v with an infinity turned into NaN (v * 0 is a zero of v's sign, or NaN), which maxima then skip and conversions keep.
__device__ __forceinline__ float finite_or_nan(float v) { return __fmaf_rn(v, 0.0f, v); }

// Two values to two e4m3 bytes (lo in the low byte), round to nearest even; NaN to 0x7F.
__device__ __forceinline__ uint32_t e4m3x2(float hi, float lo) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t quantize4(const float (&v)[4], const float (&inv)[4]) {
  return e4m3x2(__fmul_rn(v[1], inv[1]), __fmul_rn(v[0], inv[0])) |
         (e4m3x2(__fmul_rn(v[3], inv[3]), __fmul_rn(v[2], inv[2])) << 16);
}
// Four e4m3 bytes to f32 (exact).
__device__ __forceinline__ void unpack4(uint32_t w, float (&v)[4]) {
  uint32_t a, b;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(a) : "h"((uint16_t)(w & 0xffffu)));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(b) : "h"((uint16_t)(w >> 16)));
  asm("{.reg .b16 l, h; mov.b32 {l, h}, %2; cvt.f32.f16 %0, l; cvt.f32.f16 %1, h;}" : "=f"(v[0]), "=f"(v[1]) : "r"(a));
  asm("{.reg .b16 l, h; mov.b32 {l, h}, %2; cvt.f32.f16 %0, l; cvt.f32.f16 %1, h;}" : "=f"(v[2]), "=f"(v[3]) : "r"(b));
}

// act'(y) * g with every step rounded as the f32 derivative forms round it (elementwise.cu).
template <int ACT>
__device__ __forceinline__ float act_grad(float y, float g) {
  if (ACT == CLEAVE_ACT_TANH) return __fmul_rn(__fsub_rn(1.0f, __fmul_rn(y, y)), g);
  if (ACT == CLEAVE_ACT_SIGMOID) return __fmul_rn(__fmul_rn(y, __fsub_rn(1.0f, y)), g);
  if (ACT == CLEAVE_ACT_RELU) return y > 0.0f ? g : 0.0f;
  return g;
}

// What a tile's CTA shares: the columns' maxima (bits of magnitudes, ordered as integers), the column sums of each warp's rows,
// a word for the last-CTA test.  The maxima meet in shared-memory atomics: a maximum does not depend on the order, and every
// warp reading the 16 warps' own ones took a sixth of the kernel's shared-memory cycles.
struct TileShared {
  uint32_t max[kQBlock];
  float sum[kQWarps][kQBlock];
  bool last;
};

// Column sums of a tile from its warps' (sh.sum, complete for the CTA), then, by the last CTA of the column block to get here, of
// the row blocks in ascending order, four runs of them side by side: the order of the additions is a function of the shape alone.
__device__ __forceinline__ void finish_sums(const TileArgs& a, TileShared& sh, int rb, int cb, int row_blocks) {
  const int tc = threadIdx.x & (kQBlock - 1), part = threadIdx.x / kQBlock;   // column, one of four
  const int c = cb * kQBlock + tc;
  if (part == 0 && c < a.cols) {
    float t = sh.sum[0][tc];
#pragma unroll
    for (int w = 1; w < kQWarps; ++w) t = __fadd_rn(t, sh.sum[w][tc]);
    a.db_part[(int64_t)rb * a.cols + c] = t;
  }
  if (a.db == nullptr) return;
  __syncthreads();
  if (threadIdx.x == 0) {   // releases what the CTA stored before the barrier, acquires what the others released
    unsigned int before;
    asm volatile("atom.acq_rel.gpu.global.inc.u32 %0, [%1], %2;"
                 : "=r"(before) : "l"(&g_db_arrivals[cb]), "r"((unsigned int)(row_blocks - 1)) : "memory");
    sh.last = before == (unsigned int)(row_blocks - 1);
  }
  __syncthreads();
  if (!sh.last) return;
  const int per = (row_blocks + 3) / 4, first = part * per;
  float t = 0.0f;
  if (c < a.cols)
    for (int r = first; r < first + per && r < row_blocks; ++r) t = __fadd_rn(t, __ldcg(a.db_part + (int64_t)r * a.cols + c));
  sh.sum[part][tc] = t;
  __syncthreads();
  if (part == 0 && c < a.cols)
    a.db[c] = __fadd_rn(__fadd_rn(sh.sum[0][tc], sh.sum[1][tc]), __fadd_rn(sh.sum[2][tc], sh.sum[3][tc]));
}

constexpr int kNoAct = -1;   // plain quantization

// One tile.  FULL: it lies inside the matrix and x can be read as 16-byte words, so that nothing is tested per row.
template <int ACT, bool FULL>
__device__ __forceinline__ void tile_pass(const TileArgs& a, TileShared& sh) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col_blocks = a.col_blocks;
  const int rb = blockIdx.x / col_blocks, cb = blockIdx.x - rb * col_blocks;
  const int r0 = rb * kQBlock + warp * kQRows, c0 = cb * kQBlock + lane * 4;
  const int64_t pitch = ((int64_t)a.cols + 15) / 16 * 16;
  const int rows_here = FULL ? kQRows : a.rows - r0 < kQRows ? a.rows - r0 : kQRows;   // may be negative
  const bool in_pitch = FULL || c0 < pitch;   // the padding behind the last column gets zeros

  const bool whole_tile = a.q_cols != nullptr || a.q_tiles != nullptr;
  if (whole_tile && threadIdx.x < kQBlock) sh.max[threadIdx.x] = 0u;

  // ---- every load of the thread
  float v[kQRows][4];
  const float* src = a.x + (int64_t)r0 * a.cols + c0;
  if (FULL || a.vec) {
#pragma unroll
    for (int i = 0; i < kQRows; ++i) {
      float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (FULL || (i < rows_here && c0 < a.cols)) t = __ldcs(reinterpret_cast<const float4*>(src));
      src += a.cols;
      v[i][0] = t.x; v[i][1] = t.y; v[i][2] = t.z; v[i][3] = t.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kQRows; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = i < rows_here && c0 + j < a.cols ? __ldg(src + (int64_t)i * a.cols + j) : 0.0f;
  }
  if constexpr (ACT != kNoAct) {
    uint32_t w[kQRows];
    const uint8_t* ysrc = a.y_q + r0 * pitch + c0;
#pragma unroll
    for (int i = 0; i < kQRows; ++i) {
      w[i] = FULL || (i < rows_here && c0 < a.cols) ? __ldcs(reinterpret_cast<const uint32_t*>(ysrc)) : 0u;
      ysrc += pitch;
    }
    float sc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    float row_scale = 0.0f;   // ROWS: lane i holds row i's
    if (a.y_blocks == CLEAVE_BLOCKS_COLS) {
#pragma unroll
      for (int j = 0; j < 4; ++j) sc[j] = FULL || c0 + j < a.cols ? __ldg(a.y_s + (int64_t)rb * a.cols + c0 + j) : 0.0f;
    } else if (a.y_blocks == CLEAVE_BLOCKS_TILES) {
      sc[0] = sc[1] = sc[2] = sc[3] = __ldg(a.y_s + (int64_t)rb * col_blocks + cb);
    } else {
      if (lane < rows_here) row_scale = __ldg(a.y_s + (int64_t)cb * a.rows + r0 + lane);
    }
#pragma unroll
    for (int i = 0; i < kQRows; ++i) {
      float y[4];
      unpack4(w[i], y);
      if (a.y_blocks == CLEAVE_BLOCKS_ROWS) sc[0] = sc[1] = sc[2] = sc[3] = __shfl_sync(0xffffffffu, row_scale, i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[i][j] = act_grad<ACT>(__fmul_rn(y[j], sc[j]), v[i][j]);
        if (!FULL && !(i < rows_here && c0 + j < a.cols)) v[i][j] = 0.0f;   // padding bytes may be anything
      }
    }
    if (a.dz != nullptr) {
      float* dst = a.dz + (int64_t)r0 * a.cols + c0;
#pragma unroll
      for (int i = 0; i < kQRows; ++i) {
        if (!FULL && i >= rows_here) break;
        if (FULL || a.vec) {
          if (FULL || c0 < a.cols)
            __stcs(reinterpret_cast<float4*>(dst + (int64_t)i * a.cols), make_float4(v[i][0], v[i][1], v[i][2], v[i][3]));
        } else {
          // rows that 16-byte words do not fit pass through the warp's shared row, so that a store covers whole lines: four
          // 4-byte stores a stride of 16 bytes apart write every sector four times
          float* row = sh.sum[warp];
          __syncwarp();
          *reinterpret_cast<float4*>(row + lane * 4) = make_float4(v[i][0], v[i][1], v[i][2], v[i][3]);
          __syncwarp();
          float* out = a.dz + (int64_t)(r0 + i) * a.cols + cb * kQBlock + lane;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (cb * kQBlock + lane + 32 * j < a.cols) __stcs(out + 32 * j, row[lane + 32 * j]);
        }
      }
      __syncwarp();
    }
    if (a.db_part != nullptr) {
      float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < kQRows; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] = __fadd_rn(sum[j], v[i][j]);
      *reinterpret_cast<float4*>(&sh.sum[warp][lane * 4]) = make_float4(sum[0], sum[1], sum[2], sum[3]);
    }
  }
#pragma unroll
  for (int i = 0; i < kQRows; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) v[i][j] = finite_or_nan(v[i][j]);

  // ---- column maxima to shared memory
  if (whole_tile) {
    __syncthreads();   // they start at zero
    float m[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[j] = 0.0f;
#pragma unroll
      for (int i = 0; i < kQRows; ++i) m[j] = fmaxf(m[j], fabsf(v[i][j]));
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) atomicMax(&sh.max[lane * 4 + j], __float_as_uint(m[j]));
  }
  // ---- 1 x 128 blocks: a row of the tile is one warp's.  Lane i works out row i's scale for all.
  if (a.q_rows != nullptr) {
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < kQRows; ++i) {
      // the leading 0 also replaces a NaN met first
      const float m = fmaxf(fmaxf(fmaxf(0.0f, fabsf(v[i][0])), fabsf(v[i][1])), fmaxf(fmaxf(0.0f, fabsf(v[i][2])), fabsf(v[i][3])));
      const uint32_t row_max = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
      mine = lane == i ? row_max : mine;
    }
    const uint32_t e = amax_exponent(mine);
    if (lane < kQRows && lane < rows_here) a.s_rows[(int64_t)cb * a.rows + r0 + lane] = scale_of(e);
    const float my_inv = inverse_scale_of(e);
    uint8_t* dst = a.q_rows + r0 * pitch + c0;
#pragma unroll
    for (int i = 0; i < kQRows; ++i) {
      const float inv = __shfl_sync(0xffffffffu, my_inv, i);
      const float inv4[4] = {inv, inv, inv, inv};
      if (FULL || (i < rows_here && in_pitch)) *reinterpret_cast<uint32_t*>(dst) = quantize4(v[i], inv4);
      dst += pitch;
    }
  }
  const bool sums = ACT != kNoAct && a.db_part != nullptr;
  if (!whole_tile && !sums) return;
  __syncthreads();
  if (whole_tile) {
    const uint4 m4 = *reinterpret_cast<const uint4*>(&sh.max[lane * 4]);
    const uint32_t m[4] = {m4.x, m4.y, m4.z, m4.w};
    if (a.q_cols != nullptr) {
      float inv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t e = amax_exponent(m[j]);
        inv[j] = inverse_scale_of(e);
        if (warp == 0 && (FULL || c0 + j < a.cols)) a.s_cols[(int64_t)rb * a.cols + c0 + j] = scale_of(e);
      }
      uint8_t* dst = a.q_cols + r0 * pitch + c0;
#pragma unroll
      for (int i = 0; i < kQRows; ++i) {
        if (FULL || (i < rows_here && in_pitch)) *reinterpret_cast<uint32_t*>(dst) = quantize4(v[i], inv);
        dst += pitch;
      }
    }
    if (a.q_tiles != nullptr) {
      const uint32_t e = amax_exponent(__reduce_max_sync(0xffffffffu, max(max(m[0], m[1]), max(m[2], m[3]))));
      const float inv = inverse_scale_of(e);
      const float inv4[4] = {inv, inv, inv, inv};
      if (threadIdx.x == 0) a.s_tiles[(int64_t)rb * col_blocks + cb] = scale_of(e);
      uint8_t* dst = a.q_tiles + r0 * pitch + c0;
#pragma unroll
      for (int i = 0; i < kQRows; ++i) {
        if (FULL || (i < rows_here && in_pitch)) *reinterpret_cast<uint32_t*>(dst) = quantize4(v[i], inv4);
        dst += pitch;
      }
    }
  }
  if (sums) finish_sums(a, sh, rb, cb, a.row_blocks);
}

// f32 output and column sums only: nothing has to be neighbours for packing, so a lane's columns are 32 apart and every load and
// store of a warp covers whole lines whatever the alignment, four rows of a warp in flight at a time.  For rows that 16-byte
// words do not fit: 6007 x 1283 24.6 us, 28.7 with tile_pass, whose 4-byte loads 16 bytes apart keep L1 70 % busy; where they fit,
// tile_pass is the faster (4096 x 4096: 27.8 us against 39.7).
template <int ACT>
__global__ void __launch_bounds__(kQThreads, 2) act_bwd_kernel(const TileArgs a) {
  __shared__ __align__(16) TileShared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col_blocks = q_blocks(a.cols);
  const int rb = blockIdx.x / col_blocks, cb = blockIdx.x - rb * col_blocks;
  const int r0 = rb * kQBlock + warp * kQRows, c0 = cb * kQBlock + lane;
  const int64_t pitch = ((int64_t)a.cols + 15) / 16 * 16;
  float sc[4], sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  bool col_ok[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    col_ok[j] = c0 + 32 * j < a.cols;
    sc[j] = a.y_blocks == CLEAVE_BLOCKS_TILES ? __ldg(a.y_s + (int64_t)rb * col_blocks + cb)
            : a.y_blocks == CLEAVE_BLOCKS_COLS && col_ok[j] ? __ldg(a.y_s + (int64_t)rb * a.cols + c0 + 32 * j) : 0.0f;
  }
  constexpr int kBatch = 4;
#pragma unroll
  for (int i0 = 0; i0 < kQRows; i0 += kBatch) {
    float g[kBatch][4];
    uint32_t q[kBatch][4];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const bool row_ok = r0 + i0 + i < a.rows;
      const float* x = a.x + (int64_t)(r0 + i0 + i) * a.cols + c0;
      const uint8_t* y = a.y_q + (r0 + i0 + i) * pitch + c0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        g[i][j] = row_ok && col_ok[j] ? __ldcs(x + 32 * j) : 0.0f;
        q[i][j] = row_ok && col_ok[j] ? __ldcs(y + 32 * j) : 0u;
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const bool row_ok = r0 + i0 + i < a.rows;
      if (a.y_blocks == CLEAVE_BLOCKS_ROWS) sc[0] = sc[1] = sc[2] = sc[3] = row_ok ? __ldg(a.y_s + (int64_t)cb * a.rows + r0 + i0 + i) : 0.0f;
      float y[4];
      unpack4(q[i][0] | (q[i][1] << 8) | (q[i][2] << 16) | (q[i][3] << 24), y);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!(row_ok && col_ok[j])) continue;
        const float d = act_grad<ACT>(__fmul_rn(y[j], sc[j]), g[i][j]);
        sum[j] = __fadd_rn(sum[j], d);
        if (a.dz != nullptr) __stcs(a.dz + (int64_t)(r0 + i0 + i) * a.cols + c0 + 32 * j, d);
      }
    }
  }
  if (a.db_part == nullptr) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) sh.sum[warp][lane + 32 * j] = sum[j];
  __syncthreads();
  finish_sums(a, sh, rb, cb, q_blocks(a.rows));
}

template <int ACT>
__global__ void __launch_bounds__(kQThreads, 2) tile_kernel(const TileArgs a) {
  __shared__ __align__(16) TileShared sh;
  const int col_blocks = a.col_blocks;
  const int rb = blockIdx.x / col_blocks, cb = blockIdx.x - rb * col_blocks;
  if (a.vec && rb < a.rows / kQBlock && cb < a.cols / kQBlock) tile_pass<ACT, true>(a, sh);
  else tile_pass<ACT, false>(a, sh);
}

// out[r, c] = q * scale: one thread per four columns of a row.
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t* __restrict__ q, const float* __restrict__ s,
                                                         float* __restrict__ out, int rows, int cols, int blocks, int vec) {
  const int64_t pitch = ((int64_t)cols + 15) / 16 * 16;
  const int col_blocks = q_blocks(cols);
  const int groups = (cols - 1) / 4 + 1;
  const int64_t total = (int64_t)rows * groups;
  for (int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; t < total; t += (int64_t)gridDim.x * blockDim.x) {
    const int r = (int)(t / groups), c = (int)(t - (int64_t)r * groups) * 4;
    float v[4];
    unpack4(__ldg(reinterpret_cast<const uint32_t*>(q + r * pitch + c)), v);
    float sc[4];
    if (blocks == CLEAVE_BLOCKS_COLS) {
#pragma unroll
      for (int j = 0; j < 4; ++j) sc[j] = c + j < cols ? __ldg(s + (int64_t)(r / kQBlock) * cols + c + j) : 0.0f;
    } else {
      sc[0] = blocks == CLEAVE_BLOCKS_ROWS ? __ldg(s + (int64_t)(c / kQBlock) * rows + r)
                                           : __ldg(s + (int64_t)(r / kQBlock) * col_blocks + c / kQBlock);
      sc[1] = sc[2] = sc[3] = sc[0];
    }
    float* dst = out + (int64_t)r * cols + c;
    if (vec) {
      *reinterpret_cast<float4*>(dst) = make_float4(__fmul_rn(v[0], sc[0]), __fmul_rn(v[1], sc[1]), __fmul_rn(v[2], sc[2]),
                                                    __fmul_rn(v[3], sc[3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < cols) dst[j] = __fmul_rn(v[j], sc[j]);
    }
  }
}

bool q_operand(cleave_buf q, cleave_buf s, int rows, int cols, int blocks, const char* what, QOperand* out) {
  if (rows <= 0 || cols <= 0) {
    set_error(CLEAVE_CUDA_ERR_ARG, "%s: rows and cols must be positive (got %d, %d)", what, rows, cols);
    return false;
  }
  blocks &= ~CLEAVE_SCALES_ANY;
  if (blocks < CLEAVE_BLOCKS_ROWS || blocks > CLEAVE_BLOCKS_TILES) {
    set_error(CLEAVE_CUDA_ERR_ARG, "%s: unknown block form %d", what, blocks);
    return false;
  }
  Buf* Q = as_buf(q, what, DT_E4M3);
  if (!Q) return false;
  Buf* S = as_buf(s, what);
  if (!S) return false;
  if (Q->len != q_bytes(rows, cols) || S->len != q_scales(rows, cols, blocks)) {
    set_error(CLEAVE_CUDA_ERR_SHAPE, "%s: %lld bytes and %lld scales given, a %d x %d tensor has %lld and %lld", what,
              (long long)Q->len, (long long)S->len, rows, cols, (long long)q_bytes(rows, cols),
              (long long)q_scales(rows, cols, blocks));
    return false;
  }
  if (!aligned16(Q->ptr)) {
    set_error(CLEAVE_CUDA_ERR_ARG, "%s: the bytes of an 8-bit tensor must be 16-byte aligned", what);
    return false;
  }
  out->q = (uint8_t*)Q->ptr;
  out->s = S->ptr;
  return true;
}

static bool overlaps(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  return a && b && (const char*)a < (const char*)b + b_bytes && (const char*)b < (const char*)a + a_bytes;
}

bool ranges_distinct(const MemRange* out, int n_out, const MemRange* in, int n_in, const char* what) {
  for (int i = 0; i < n_out; ++i) {
    for (int j = i + 1; j < n_out; ++j)
      if (overlaps(out[i].p, out[i].bytes, out[j].p, out[j].bytes)) {
        set_error(CLEAVE_CUDA_ERR_ARG, "%s: two outputs share memory", what);
        return false;
      }
    for (int j = 0; j < n_in; ++j)
      if (overlaps(out[i].p, out[i].bytes, in[j].p, in[j].bytes)) {
        set_error(CLEAVE_CUDA_ERR_ARG, "%s: an output shares memory with an input", what);
        return false;
      }
  }
  return true;
}

template <int ACT>
static void launch_act_bwd(const TileArgs& a, int tiles) {
  if (a.q_rows || a.q_cols || a.vec) tile_kernel<ACT><<<tiles, kQThreads, 0, ctx().stream>>>(a);
  else act_bwd_kernel<ACT><<<tiles, kQThreads, 0, ctx().stream>>>(a);
}

static bool launch_tiles(const TileArgs& a, const char* what) {
  const int64_t tiles = (int64_t)a.row_blocks * a.col_blocks;
  if (tiles > 0x7fffffffll) {
    set_error(CLEAVE_CUDA_ERR_UNSUPPORTED, "%s: %d x %d has more than 2^31 - 1 blocks", what, a.rows, a.cols);
    return false;
  }
  if (!a.y_q) tile_kernel<kNoAct><<<(int)tiles, kQThreads, 0, ctx().stream>>>(a);
  else if (a.act == CLEAVE_ACT_TANH) launch_act_bwd<CLEAVE_ACT_TANH>(a, (int)tiles);
  else if (a.act == CLEAVE_ACT_SIGMOID) launch_act_bwd<CLEAVE_ACT_SIGMOID>(a, (int)tiles);
  else if (a.act == CLEAVE_ACT_RELU) launch_act_bwd<CLEAVE_ACT_RELU>(a, (int)tiles);
  else launch_act_bwd<CLEAVE_ACT_IDENTITY>(a, (int)tiles);
  count_launch();
  return cuda_ok(cudaGetLastError(), "quantize kernel launch");
}

}  // namespace cleave

using namespace cleave;

extern "C" {

int64_t cleave_cuda_e4m3_bytes(int32_t rows, int32_t cols) { return rows > 0 && cols > 0 ? q_bytes(rows, cols) : 0; }

int64_t cleave_cuda_e4m3_scales(int32_t rows, int32_t cols, int32_t blocks) {
  return rows > 0 && cols > 0 ? q_scales(rows, cols, blocks & ~CLEAVE_SCALES_ANY) : 0;
}

cleave_buf cleave_cuda_alloc_e4m3(int64_t bytes) {
  ApiLock lock;
  return (cleave_buf)new_buf(bytes, DT_E4M3);
}

cleave_buf cleave_cuda_wrap_e4m3(void* device_ptr, int64_t bytes) {
  ApiLock lock;
  if (!device_ptr || bytes <= 0 || !aligned16(device_ptr)) {
    set_error(CLEAVE_CUDA_ERR_ARG, "wrap_e4m3: need a 16-byte aligned device pointer and a positive length");
    return nullptr;
  }
  return (cleave_buf)new_view(device_ptr, bytes, DT_E4M3);
}

cleave_buf cleave_cuda_upload_e4m3(const uint8_t* host, int64_t bytes) {
  ApiLock lock;
  if (!host) {
    set_error(CLEAVE_CUDA_ERR_ARG, "upload_e4m3: NULL host pointer");
    return nullptr;
  }
  Buf* b = new_buf(bytes, DT_E4M3);
  if (!b) return nullptr;
  if (!cuda_ok(cudaMemcpyAsync(b->ptr, host, (size_t)bytes, cudaMemcpyHostToDevice, ctx().stream), "cudaMemcpyAsync(H2D)") ||
      !cuda_ok(cudaStreamSynchronize(ctx().stream), "cudaStreamSynchronize")) {
    release_buf(b);
    return nullptr;
  }
  return (cleave_buf)b;
}

int64_t cleave_cuda_download_e4m3(cleave_buf t, uint8_t* host, int64_t bytes) {
  ApiLock lock;
  Buf* b = as_buf(t, "download_e4m3", DT_E4M3);
  if (!b) return -cleave_cuda_last_error();
  if (!host || bytes != b->len)
    return -set_error(CLEAVE_CUDA_ERR_SHAPE, "download_e4m3: room for %lld bytes, tensor has %lld", (long long)bytes,
                      (long long)b->len);
  if (!cuda_ok(cudaMemcpyAsync(host, b->ptr, (size_t)bytes, cudaMemcpyDeviceToHost, ctx().stream), "cudaMemcpyAsync(D2H)") ||
      !cuda_ok(cudaStreamSynchronize(ctx().stream), "cudaStreamSynchronize") || check_device_status() != CLEAVE_CUDA_OK)
    return -cleave_cuda_last_error();
  return bytes;
}

int32_t cleave_cuda_quantize_e4m3(cleave_buf x, int32_t rows, int32_t cols, cleave_buf q_rows, cleave_buf s_rows,
                                  cleave_buf q_cols, cleave_buf s_cols, cleave_buf q_tiles, cleave_buf s_tiles) {
  ApiLock lock;
  if (!ensure_init()) return -cleave_cuda_last_error();   // also makes the library's device this thread's
  Buf* X = as_buf(x, "quantize");
  if (!X) return -cleave_cuda_last_error();
  if (rows <= 0 || cols <= 0 || X->len != (int64_t)rows * cols)
    return -set_error(CLEAVE_CUDA_ERR_SHAPE, "quantize: tensor has %lld elements, not %d x %d", (long long)X->len, rows, cols);
  QOperand o[3];
  const cleave_buf given[3][2] = {{q_rows, s_rows}, {q_cols, s_cols}, {q_tiles, s_tiles}};
  MemRange out[6];
  int n_out = 0;
  for (int f = 0; f < 3; ++f)
    if (given[f][0] || given[f][1]) {
      const int blocks = CLEAVE_BLOCKS_ROWS + f;
      if (!q_operand(given[f][0], given[f][1], rows, cols, blocks, "quantize", &o[f])) return -cleave_cuda_last_error();
      out[n_out++] = {o[f].q, q_bytes(rows, cols)};
      out[n_out++] = {o[f].s, q_scales(rows, cols, blocks) * 4};
    }
  if (n_out == 0) return -set_error(CLEAVE_CUDA_ERR_ARG, "quantize: no output given");
  const MemRange in[1] = {{X->ptr, X->len * 4}};
  if (!ranges_distinct(out, n_out, in, 1, "quantize")) return -cleave_cuda_last_error();
  Trace tr("quantize", "rows=%d cols=%d", rows, cols);
  TileArgs a{};
  a.rows = rows;
  a.cols = cols;
  a.row_blocks = q_blocks(rows);
  a.col_blocks = q_blocks(cols);
  a.vec = aligned16(X->ptr) && cols % 4 == 0;
  a.x = X->ptr;
  a.q_rows = o[0].q; a.s_rows = o[0].s;
  a.q_cols = o[1].q; a.s_cols = o[1].s;
  a.q_tiles = o[2].q; a.s_tiles = o[2].s;
  return launch_tiles(a, "quantize") ? CLEAVE_CUDA_OK : -cleave_cuda_last_error();
}

int32_t cleave_cuda_dequantize_e4m3(cleave_buf out, cleave_buf q, cleave_buf s, int32_t rows, int32_t cols, int32_t blocks) {
  ApiLock lock;
  if (!ensure_init()) return -cleave_cuda_last_error();   // also makes the library's device this thread's
  Buf* O = as_buf(out, "dequantize");
  if (!O) return -cleave_cuda_last_error();
  QOperand in;
  if (!q_operand(q, s, rows, cols, blocks, "dequantize", &in)) return -cleave_cuda_last_error();
  blocks &= ~CLEAVE_SCALES_ANY;
  if (O->len != (int64_t)rows * cols)
    return -set_error(CLEAVE_CUDA_ERR_SHAPE, "dequantize: output has %lld elements, not %d x %d", (long long)O->len, rows, cols);
  const MemRange outs[1] = {{O->ptr, O->len * 4}};
  const MemRange ins[2] = {{in.q, q_bytes(rows, cols)}, {in.s, q_scales(rows, cols, blocks) * 4}};
  if (!ranges_distinct(outs, 1, ins, 2, "dequantize")) return -cleave_cuda_last_error();
  Trace tr("dequantize", "rows=%d cols=%d blocks=%d", rows, cols, blocks);
  dequantize_kernel<<<stream_grid((int64_t)rows * ((cols - 1) / 4 + 1), 256, 8), 256, 0, ctx().stream>>>(
      in.q, in.s, O->ptr, rows, cols, blocks, aligned16(O->ptr) && cols % 4 == 0);
  count_launch();
  return cuda_ok(cudaGetLastError(), "dequantize kernel launch") ? CLEAVE_CUDA_OK : -cleave_cuda_last_error();
}

int32_t cleave_cuda_act_bwd_e4m3(cleave_buf y, cleave_buf y_scale, int32_t y_blocks, cleave_buf g, int32_t rows, int32_t cols,
                                 int32_t act, cleave_buf dz, cleave_buf q_rows, cleave_buf s_rows, cleave_buf q_cols,
                                 cleave_buf s_cols, cleave_buf db) {
  ApiLock lock;
  if (!ensure_init()) return -cleave_cuda_last_error();   // also makes the library's device this thread's
  QOperand Y;
  if (!q_operand(y, y_scale, rows, cols, y_blocks, "act_bwd", &Y)) return -cleave_cuda_last_error();
  y_blocks &= ~CLEAVE_SCALES_ANY;
  Buf* G = as_buf(g, "act_bwd");
  if (!G) return -cleave_cuda_last_error();
  const int64_t n = (int64_t)rows * cols;
  if (G->len != n)
    return -set_error(CLEAVE_CUDA_ERR_SHAPE, "act_bwd: gradient has %lld elements, not %d x %d", (long long)G->len, rows, cols);
  if (act < CLEAVE_ACT_IDENTITY || act > CLEAVE_ACT_TANH)
    return -set_error(CLEAVE_CUDA_ERR_ARG, "act_bwd: unknown activation code %d", act);
  MemRange out[6];
  int n_out = 0;
  Buf *DZ = nullptr, *DB = nullptr;
  if (dz) {
    DZ = as_buf(dz, "act_bwd");
    if (!DZ) return -cleave_cuda_last_error();
    if (DZ->len != n)
      return -set_error(CLEAVE_CUDA_ERR_SHAPE, "act_bwd: dz has %lld elements, not %d x %d", (long long)DZ->len, rows, cols);
    out[n_out++] = {DZ->ptr, n * 4};
  }
  if (db) {
    DB = as_buf(db, "act_bwd");
    if (!DB) return -cleave_cuda_last_error();
    if (DB->len != cols)
      return -set_error(CLEAVE_CUDA_ERR_SHAPE, "act_bwd: db has %lld elements for %d columns", (long long)DB->len, cols);
    out[n_out++] = {DB->ptr, (int64_t)cols * 4};
  }
  QOperand o[2];
  const cleave_buf given[2][2] = {{q_rows, s_rows}, {q_cols, s_cols}};
  for (int f = 0; f < 2; ++f)
    if (given[f][0] || given[f][1]) {
      const int blocks = CLEAVE_BLOCKS_ROWS + f;
      if (!q_operand(given[f][0], given[f][1], rows, cols, blocks, "act_bwd", &o[f])) return -cleave_cuda_last_error();
      out[n_out++] = {o[f].q, q_bytes(rows, cols)};
      out[n_out++] = {o[f].s, q_scales(rows, cols, blocks) * 4};
    }
  if (n_out == 0) return -set_error(CLEAVE_CUDA_ERR_ARG, "act_bwd: no output given");
  const MemRange in[3] = {{G->ptr, n * 4}, {Y.q, q_bytes(rows, cols)}, {Y.s, q_scales(rows, cols, y_blocks) * 4}};
  if (!ranges_distinct(out, n_out, in, 3, "act_bwd")) return -cleave_cuda_last_error();
  Trace tr("act_bwd_e4m3", "rows=%d cols=%d act=%d", rows, cols, act);
  TileArgs a{};
  a.rows = rows;
  a.cols = cols;
  a.row_blocks = q_blocks(rows);
  a.col_blocks = q_blocks(cols);
  a.vec = aligned16(G->ptr) && (!DZ || aligned16(DZ->ptr)) && cols % 4 == 0;
  a.x = G->ptr;
  a.y_q = Y.q;
  a.y_s = Y.s;
  a.y_blocks = y_blocks;
  a.act = act;
  a.dz = DZ ? DZ->ptr : nullptr;
  a.q_rows = o[0].q; a.s_rows = o[0].s;
  a.q_cols = o[1].q; a.s_cols = o[1].s;
  // Column sums: every tile leaves the sums of its 128 rows; the kernel adds the row blocks itself, or a second one does.
  const int row_blocks = q_blocks(rows);
  const bool in_kernel = q_blocks(cols) <= kQMaxColBlocks && row_blocks <= kQMaxRowBlocks;
  float* part = nullptr;
  if (DB) {
    part = row_blocks == 1 ? DB->ptr : scratch_alloc((int64_t)row_blocks * cols * (int64_t)sizeof(float));
    if (!part) return -cleave_cuda_last_error();
    a.db_part = part;
    a.db = row_blocks > 1 && in_kernel ? DB->ptr : nullptr;
  }
  bool ok = launch_tiles(a, "act_bwd");
  if (DB && row_blocks > 1) {
    if (!in_kernel) ok = ok && colsum_launch(part, DB->ptr, row_blocks, cols, ctx().stream);
    scratch_free(part);
  }
  return ok ? CLEAVE_CUDA_OK : -cleave_cuda_last_error();
}

}  // extern "C"
