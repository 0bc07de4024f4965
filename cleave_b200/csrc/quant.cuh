// Block-scaled 8-bit tensors: the stored form shared by quant.cu and gemm_q.cu.
//
// A matrix [rows, cols] is kept as e4m3 bytes (4 exponent bits, 3 mantissa bits, largest value 448, no infinity), row-major
// with a row pitch of cols rounded up to 16 bytes (what a TMA tensor map asks of a stride), and one f32 scale per block:
//   rows   1 x 128     scales [ceil(cols/128)][rows]
//   cols   128 x 1     scales [ceil(rows/128)][cols]
//   tiles  128 x 128   scales [ceil(rows/128)][ceil(cols/128)]
// The value of an element is q * scale.  The quantizer's scales are powers of two, so that value is exact in f32, dividing by
// a scale loses nothing, and the tensor pipe can apply a scale by its exponent; CLEAVE_SCALES_ANY marks a tensor with others.
#pragma once
#include <stdint.h>

#include "common.cuh"

namespace cleave {

constexpr int kQBlock = 128;

// Blocks along a side of n >= 1 elements; n + 127 would pass 2^31 for the longest sides.
__host__ __device__ constexpr int q_blocks(int n) { return (n - 1) / kQBlock + 1; }
inline int64_t q_pitch(int cols) { return ((int64_t)cols + 15) / 16 * 16; }
inline int64_t q_bytes(int rows, int cols) { return (int64_t)rows * q_pitch(cols); }
inline int64_t q_scales(int rows, int cols, int blocks) {
  const int64_t rb = q_blocks(rows), cb = q_blocks(cols);
  switch (blocks) {
    case CLEAVE_BLOCKS_ROWS: return cb * rows;
    case CLEAVE_BLOCKS_COLS: return rb * cols;
    case CLEAVE_BLOCKS_TILES: return rb * cb;
    default: return 0;
  }
}

// One 8-bit operand of an entry point: both handles resolved and checked against the shape.
struct QOperand {
  uint8_t* q = nullptr;
  float* s = nullptr;
};
// false + error (naming `what`) when a handle is not live, has the wrong element type or length, the bytes are not 16-byte
// aligned, or `blocks` is no CLEAVE_BLOCKS_* value.
bool q_operand(cleave_buf q, cleave_buf s, int rows, int cols, int blocks, const char* what, QOperand* out);

// Memory ranges of one call: outputs may meet neither each other nor an input (one CTA still reads while another writes).
// false + error naming `what` otherwise.  Null pointers meet nothing.
struct MemRange {
  const void* p;
  int64_t bytes;
};
bool ranges_distinct(const MemRange* out, int n_out, const MemRange* in, int n_in, const char* what);

}  // namespace cleave
