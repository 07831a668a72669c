// kv.h -- the paged 8-bit key/value cache: its layout in HBM and the launch
// interface between the host runtime (kv.hip) and the kernels
// (kernels_kv.hip, kernels_kv_attn.hip).
//
// A page holds 64 positions of every layer and head, page after page in one
// pool: [page][layer][head][keys | values | scales].  Codes are bytes, the
// whole number -127 .. 127 plus 128; a block of 16 positions of one head has
// one f32 scale for its keys and one for its values.
//
// Within a head's region both tiles are laid out as the matrix instructions
// take them (16 x 16 x 32 f16, A operand: lane l holds 8 numbers of row l %
// 16 from column 8 * (l / 16) on), so that a wave reads 1 KiB of consecutive
// bytes, 16 per lane, and every lane finds its own operands in them:
//   keys    position t = 16 m + i, number d = 64 c + 16 g + b (g < 4, b < 16):
//           byte ((c * 4 + m) * 64 + 16 g + i) * 16 + b; lane 16 g + i.  A
//           last half chunk of 32 numbers d = 64 c + 8 g + b (b < 8):
//           c * 4096 + (m * 64 + 16 g + i) * 8 + b.
//   values  number d = 16 n + i, position t = 16 m + 4 g + r (r < 4):
//           byte (n * 64 + 16 g + i) * 16 + 4 m + r; lane 16 g + i.
// The scores leave the matrix instruction with lane 16 g + i holding positions
// 16 m + 4 g + r of query row i: exactly the values' order, so they become
// the second product's operand without leaving the lane.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "kv_pages.h"

namespace hale {

// The padded head dimensions the kernels are built for, in units of 32: head
// dimensions between are padded (keys only) to the next.
inline int kv_chunks(size_t head_dim) {
  for (int c : {2, 3, 4, 6, 8})
    if (head_dim <= (size_t)c * 32) return c;
  return 0;
}

struct KvGeom {
  uint8_t* pool;
  size_t page_bytes;   // of all layers
  size_t layer_bytes;
  unsigned head_bytes, v_off, s_off;  // of one head's region: values, scales
  int chunks;          // keys: numbers per position / 32, padded
  int hd, kv_heads, group;
  const uint32_t* table;  // [max_seqs][max_pages] page of each 64 positions
  unsigned max_pages;
};

__host__ __device__ inline unsigned kv_key_byte(int chunks, unsigned t, unsigned d) {
  const unsigned m = t / 16, i = t % 16, c = d / 64;
  if (c < (unsigned)chunks / 2) return ((c * 4 + m) * 64 + d % 64 / 16 * 16 + i) * 16 + d % 16;
  return c * 4096 + (m * 64 + d % 64 / 8 * 16 + i) * 8 + d % 8;
}
__host__ __device__ inline unsigned kv_value_byte(unsigned t, unsigned d) {
  return (d / 16 * 64 + t % 16 / 4 * 16 + d % 16) * 16 + t / 16 * 4 + t % 4;
}

// What the device reads from host memory: the plan's pieces in src, one behind
// the other (16-byte aligned, multiples of four words), each to its own place;
// npairs changes (index, value) of the page table; and ncopies pages to copy, none of
// them written that is read.
struct KvUploadArgs {
  const uint32_t* src;
  int pieces;
  uint32_t* dst[KV_MAX_PIECES];
  unsigned words[KV_MAX_PIECES];
  const uint32_t* pairs;
  unsigned npairs;
  uint32_t* table;
  const KvCopy* copies;
  unsigned ncopies;
  uint8_t* pool;
  size_t page_bytes;
  uint32_t* done;   // host memory: receives `number`, the last upload before this one
  uint32_t number;
};
hipError_t launch_kv_upload(const KvUploadArgs& a, hipStream_t st);

struct KvAppendArgs {
  KvGeom g;
  size_t layer;
  const KvBlock* blocks;
  const uint32_t* count;  // blocks of the step, on the device (captured calls), or null
  unsigned nblocks;       // the same
  const void *k, *v;  // [tokens][kv_heads][hd], a stride of so many elements per token
  size_t k_stride, v_stride;
  bool vec;               // all rows start at multiples of 16 bytes
};
// grid: blocks launched for at least (they loop over the step's)
hipError_t launch_kv_append(int dtype, const KvAppendArgs& a, unsigned grid, hipStream_t st);

// Positions first .. first + count - 1 of the sequence in page table row
// `row`: k and v [count][kv_heads][hd] f32.
hipError_t launch_kv_read(const KvGeom& g, size_t layer, uint32_t row, size_t first, size_t count, float* k, float* v,
                          hipStream_t st);

struct KvAttnArgs {
  KvGeom g;
  size_t layer;
  int dtype;                   // of q and out
  const void* q;               // [tokens][heads][hd], q_stride elements per token
  void* out;
  size_t q_stride, out_stride;
  float scale;                 // times log2(e)
  int window;                  // 0: none
  const KvItem* items;         // of one kind
  const KvJoin* joins;
  const KvShareJoin* share_joins;  // of kind 2
  const uint32_t* counts;      // {few, many, joins of few (or all, of kind 2), of many} of the plan, on the device
  unsigned nitems, njoins;     // the same, or 0xffffffff: read counts (captured calls)
  int kind;                    // 0: items and joins of few rows, 1: of many; 2: joins of shared pages
  bool alone;                  // kind 2: each join has one series, its row's own pages
  float* part_o;               // [row][hd], times a power of two that follows from the sum
  float2* part_ml;             // [row] running maximum (base 2) and sum
  bool vec;                    // q and out rows start at multiples of four elements
};
// Sequences of few rows: cols groups of 16 per work-group.  grid: work-groups
// launched (they loop over the plan).
hipError_t launch_kv_attend_few(const KvAttnArgs& a, int cols, unsigned grid, hipStream_t st);
// Of many rows: kv_many_rows per work-group.
hipError_t launch_kv_attend_many(const KvAttnArgs& a, unsigned grid, hipStream_t st);
// Joins of one kind, of at most `rows` rows each; parts: of a row, at most (but for joins
// of several series).
hipError_t launch_kv_join(const KvAttnArgs& a, unsigned grid, unsigned rows, unsigned parts, hipStream_t st);

// ---- rotary positions --------------------------------------------------------

struct RopeArgs {
  const int32_t* pos;      // [rows]
  const double* turns;     // [rotary / 2] turns per position
  size_t rows;
  int hd, half, interleaved;  // head dimension, rotary / 2, pairs (2i, 2i + 1)
  float factor;            // on cos and sin
  const void* src[2];      // queries, keys
  void* dst[2];
  size_t src_stride[2], dst_stride[2];  // elements per row
  int heads[2];
};
hipError_t launch_rope(int dtype, const RopeArgs& a, hipStream_t st);

}  // namespace hale
