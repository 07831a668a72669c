// step_ops.h -- launch interface of the operators around a serving step's
// layers: norms that hand on 8 bits, products of 4-bit weights with group
// scales, and the rules on logits (host side: step_ops.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/hale_moe.h"

namespace hale {

// ---- norms ---------------------------------------------------------------------

struct NormQ8Args {
  const void *x, *delta;  // [rows][n], a stride of so many elements per row; delta may be null
  const float* w;
  void *sum, *y;          // may be null
  int8_t* q;              // [rows][n]
  float* scales;          // [rows][n / block]
  size_t x_stride, delta_stride, sum_stride, y_stride;
  unsigned n, block;      // block 0: one a row
  float eps;
  bool vec;               // all rows (and w) start at multiples of 16 bytes, codes of 8
};
constexpr size_t STEP_ROWS = 1u << 22;  // a grid has less than 2^32 threads, a work-group up to 1024
constexpr size_t NORM_Q8_MAX = 16384;  // numbers per row
hipError_t launch_norm_q8(int dtype, const NormQ8Args& a, size_t rows, hipStream_t st);

// ---- 4-bit weights with group scales ---------------------------------------------
//
// Tiles of 16 rows, along them chunks of 128 numbers.  In a tile, from a multiple of 128 bytes
// on, first the codes of all chunks, then their scales, then their zeros:
//   codes   16 rows x 128 numbers, lane 16 g + i of a wave 16 bytes: row i,
//           word j holds numbers 32 j + 8 g .. + 7, number b in the four bits from
//           4 (b / 2) + 16 (b % 2) on;
//   scales  [4][128 / group][4 rows], 16 bits;
//   zeros   [4][128 / group][4 rows], a byte, plus 16; only where the matrix has them.
// Numbers and rows that pad the last chunk and tile are code 8 (zero 8), scale 0.
// The matrix instructions take operands of 16 rows x 32 numbers whose lane 16 g + i holds
// row i, numbers 8 g .. 8 g + 7: a word of codes; the results' lane 16 g + i holds rows 4 g ..
// 4 g + 3 of token i, whose scales and zeros lie side by side.
constexpr unsigned Q4G_CHUNK = 128, Q4G_ROWS = 16, Q4G_OFFSET = 16;

struct Q4gGeom {
  uint8_t* data;
  size_t rows, cols;
  unsigned group, chunks;       // chunks of 128 numbers per row
  unsigned per;                 // groups per chunk
  size_t tile_bytes, scales_at;  // scales_at: of a tile's first chunk
  bool zeros, bf16;             // bf16: type of the scales (else f16)
  // where the first tile's zeros are read, and how far apart chunks' and tiles' are: in the data,
  // or, for a matrix without zeros, 64 bytes of 16 + 8 for all (no branch, and no bytes from
  // memory)
  const uint8_t* zero_data;
  unsigned zero_chunk;
  size_t zero_tile;
  // sums of tiles whose rows are divided over work-groups, [split][tile][64][4], and how many
  // of a tile's work-groups are done (0 between calls)
  float* parts;
  unsigned* done;
};
// Most work-groups that a tile's row is divided over, and that the divided rows of a launch come to.
constexpr unsigned Q4G_SPLITS = 8, Q4G_GROUPS = 256;
// Over how many work-groups a launch of `tiles` tiles for `slices` times 16 tokens divides rows of which
// `most` parts are worth it.
inline unsigned q4g_splits(size_t tiles, size_t slices, unsigned most) {
  size_t n = Q4G_GROUPS / (tiles * slices);
  n = n > most ? most : n;
  n = n > Q4G_SPLITS / slices ? Q4G_SPLITS / slices : n;
  return n < 1 ? 1 : (unsigned)n;
}
// The partial sums of tiles that a launch can need room for: a matrix of more tiles is never divided.
inline size_t q4g_part_tiles(size_t tiles) {
  if (2 * tiles > Q4G_GROUPS) return 0;
  return tiles * Q4G_SPLITS < Q4G_GROUPS ? tiles * Q4G_SPLITS : Q4G_GROUPS;
}

hipError_t launch_q4g_pack(const Q4gGeom& g, const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros,
                           hipStream_t st);
hipError_t launch_q4g_unpack(const Q4gGeom& g, uint8_t* codes, uint16_t* scales, uint8_t* zeros, hipStream_t st);

struct Q4gArgs {
  Q4gGeom g;
  const void* x;             // [ntok][cols] of a float type with a stride, or codes
  const float* x_scales;     // [ntok][x_per] of codes
  size_t x_stride;           // elements
  unsigned x_shift, x_per;   // numbers per scale of codes, as a power of two (31: one a token), and a token's scales
  size_t ntok;
  int out_dtype;
  void* out;                 // [ntok][rows]
  size_t out_stride;
  bool out_vec;              // out: all rows start at multiples of four numbers
};
enum Q4gInput : int { Q4G_F32 = 0, Q4G_F16 = 1, Q4G_BF16 = 2, Q4G_I8 = 3 };
hipError_t launch_q4g(Q4gInput in, const Q4gArgs& a, hipStream_t st);

// ---- logits ------------------------------------------------------------------------

struct LogitsArgs {
  const void* in;
  void* out;
  size_t in_stride, out_stride;
  size_t vocab;
  hale_logits_rules r;
  bool vec;                  // rows of in and out start at multiples of 16 bytes
};
hipError_t launch_logits(int dtype, const LogitsArgs& a, size_t rows, hipStream_t st);

}  // namespace hale
