// kernels_kv.hip -- rotary positions, and storing to, reading from and moving
// the pages of the 8-bit key/value cache (layout: kv.h).
#include <hip/hip_runtime.h>

#include "hale_device.h"
#include "kernels.h"
#include "kv.h"
#include "kv_device.h"

namespace hale {

// ---------------------------------------------------------------------------
// rotary positions
// ---------------------------------------------------------------------------
//
// Pair i of a row at position t turns by the angle t * f_i: (a, b) becomes
// (a cos - b sin, b cos + a sin), both times `factor`.  The angle is formed in
// turns in f64 (t * f_i / 2 pi), of which the whole turns are dropped, so that
// the f32 argument of sin and cos is exact to 2^-24 of a turn's fraction at any
// position an int32 holds; in f32 the angle of position 10^6 would be off by
// 0.03.
template <typename T>
__global__ __launch_bounds__(256) void k_rope(RopeArgs a) {
  // a thread per pair or untouched number of one head, its rows apart
  const int per = a.hd - a.half;  // pairs, then the numbers behind them
  const size_t total = a.rows * (size_t)(a.heads[0] + a.heads[1]) * per;
  for (size_t id = (size_t)blockIdx.x * 256 + threadIdx.x; id < total; id += (size_t)gridDim.x * 256) {
    const int e = (int)(id % per);
    const size_t rest = id / per;
    int h = (int)(rest % (a.heads[0] + a.heads[1]));
    const size_t row = rest / (a.heads[0] + a.heads[1]);
    const int which = h >= a.heads[0];
    if (which) h -= a.heads[0];
    const T* x = (const T*)a.src[which] + row * a.src_stride[which] + (size_t)h * a.hd;
    T* y = (T*)a.dst[which] + row * a.dst_stride[which] + (size_t)h * a.hd;
    if (e >= a.half) {  // behind the rotary numbers: copied
      const int d = e + a.half;
      y[d] = x[d];
      continue;
    }
    float c, s;
    rope_angle(a.pos[row], a.turns[e], a.factor, &c, &s);
    const int d0 = a.interleaved ? 2 * e : e, d1 = a.interleaved ? 2 * e + 1 : e + a.half;
    const float u = to_f32(x[d0]), v = to_f32(x[d1]);
    y[d0] = from_f32<T>(u * c - v * s);
    y[d1] = from_f32<T>(v * c + u * s);
  }
}

hipError_t launch_rope(int dtype, const RopeArgs& a, hipStream_t st) {
  const size_t total = a.rows * (size_t)(a.heads[0] + a.heads[1]) * (a.hd - a.half);
  if (total == 0) return hipSuccess;
  const unsigned grid = (unsigned)std::min<size_t>((total + 255) / 256, 1u << 20);
  switch (dtype) {
    case F32: return launch(k_rope<float>, grid, 256, 0, st, a);
    case F16: return launch(k_rope<_Float16>, grid, 256, 0, st, a);
    case BF16: return launch(k_rope<Bf16>, grid, 256, 0, st, a);
    default: return hipErrorInvalidValue;
  }
}

// ---------------------------------------------------------------------------
// plan upload, page copies
// ---------------------------------------------------------------------------

__global__ __launch_bounds__(256) void k_kv_upload(KvUploadArgs a) {
  const unsigned id = blockIdx.x * 256 + threadIdx.x, step = gridDim.x * 256;
  const u32x4* src = (const u32x4*)a.src;
  for (int p = 0; p < a.pieces; p++) {
    const unsigned n = a.words[p] / 4;
    u32x4* dst = (u32x4*)a.dst[p];
    for (unsigned i = id; i < n; i += step) dst[i] = src[i];
    src += n;
  }
  for (unsigned i = id; i < a.npairs; i += step) a.table[a.pairs[2 * i]] = a.pairs[2 * i + 1];
}

hipError_t launch_kv_upload(const KvUploadArgs& a, hipStream_t st) {
  size_t most = a.npairs;
  for (int p = 0; p < a.pieces; p++) most = std::max<size_t>(most, a.words[p] / 4);
  if (most == 0) return hipSuccess;
  return launch(k_kv_upload, (unsigned)std::min<size_t>((most + 255) / 256, 64), 256, 0, st, a);
}

constexpr unsigned COPY_BYTES = 16384;  // per work-group: four 16-byte pieces a thread

__global__ __launch_bounds__(256) void k_kv_copy_pages(uint8_t* pool, size_t page_bytes, const KvCopy* list) {
  const KvCopy c = list[blockIdx.y];
  const size_t at = (size_t)blockIdx.x * COPY_BYTES;
  const u32x4* s = (const u32x4*)(pool + c.src * page_bytes + at);
  u32x4* d = (u32x4*)(pool + c.dst * page_bytes + at);
  const unsigned n = (unsigned)(page_bytes - at < COPY_BYTES ? page_bytes - at : COPY_BYTES) / 16;
  u32x4 x[4];
#pragma unroll
  for (int j = 0; j < 4; j++)
    if (threadIdx.x + 256 * j < n) x[j] = s[threadIdx.x + 256 * j];
#pragma unroll
  for (int j = 0; j < 4; j++)
    if (threadIdx.x + 256 * j < n) d[threadIdx.x + 256 * j] = x[j];
}

hipError_t launch_kv_copy_pages(uint8_t* pool, size_t page_bytes, const KvCopy* list, unsigned n, hipStream_t st) {
  const unsigned chunks = (unsigned)((page_bytes + COPY_BYTES - 1) / COPY_BYTES);
  for (unsigned at = 0; at < n; at += 32768) {  // the grid's second dimension ends at 65535
    const hipError_t e = launch(k_kv_copy_pages, dim3(chunks, std::min(n - at, 32768u)), 256, 0, st, pool, page_bytes,
                                list + at);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// ---------------------------------------------------------------------------
// storing
// ---------------------------------------------------------------------------
//
// One wave per block of 16 positions, head, and keys or values: the largest
// magnitude of the new numbers, the block's scale from it and the former one,
// the codes.  Quotients are rounded to whole numbers from their exact values:
// x / s is formed in f64, whose rounding cannot carry a quotient of two f32
// onto a half (they are at least 2^-25 of it apart from one, or on it).
template <typename T, int NI>
__device__ __forceinline__ void append_block(const KvAppendArgs& a, KvBlock blk) {
  const KvStepSeq sq = a.seqs[blk.seq];
  const int head = blockIdx.y, lane = threadIdx.x, values = threadIdx.y, hd = a.g.hd;
  const unsigned pos0 = blk.block * KV_BLOCK;
  const int old = sq.len0 > pos0 ? (int)(sq.len0 - pos0) : 0;  // positions held; < 16
  const int end = sq.len0 + sq.ntok - pos0 < KV_BLOCK ? (int)(sq.len0 + sq.ntok - pos0) : (int)KV_BLOCK;
  const size_t stride = values ? a.v_stride : a.k_stride;
  // the token of the block's position 0 (it may lie before the step's first)
  const long long tok = (long long)sq.tok0 + pos0 - sq.len0;
  const T* src = (const T*)(values ? a.v : a.k) + (size_t)head * hd;
  const uint32_t page = a.g.table[(size_t)sq.row * a.g.max_pages + pos0 / KV_PAGE];
  uint8_t* region = a.g.pool + page * a.g.page_bytes + a.layer * a.g.layer_bytes + (size_t)head * a.g.head_bytes;
  const unsigned t0 = pos0 % KV_PAGE;
  float* scale = (float*)(region + a.g.s_off) + values * 4 + t0 / KV_BLOCK;

  float x[NI][KV_BLOCK], top = 0.0f;
#pragma unroll
  for (int n = 0; n < NI; n++) {
    const int d = lane + 64 * n;
#pragma unroll
    for (int t = 0; t < (int)KV_BLOCK; t++) {
      float v = 0.0f;
      if (t >= old && t < end && d < hd) v = to_f32(src[(size_t)(tok + t) * stride + d]);
      v = __builtin_isfinite(v) ? v : 0.0f;  // what is not finite is stored as 0 and raises no scale
      x[n][t] = v;
      top = fmaxf(top, fabsf(v));
    }
  }
  top = wave_max_f32(top);
  const float had = old ? *scale : 0.0f;
  const float s = fmaxf(had, top / 127.0f);
  const bool grown = old && s > had;
  const double wide = (double)s;
#pragma unroll
  for (int n = 0; n < NI; n++) {
    const int d = lane + 64 * n;
    if (d >= hd) break;
#pragma unroll
    for (int t = 0; t < (int)KV_BLOCK; t++) {
      uint8_t* at = region + (values ? a.g.v_off + kv_value_byte(t0 + t, d) : kv_key_byte(a.g.chunks, t0 + t, d));
      if (t < old) {
        if (grown) *at = (uint8_t)((int)rint((double)((int)*at - 128) * had / wide) + 128);
      } else if (t < end) {
        const double q = s > 0.0f ? rint((double)x[n][t] / wide) : 0.0;
        *at = (uint8_t)((int)fmin(fmax(q, -127.0), 127.0) + 128);
      }
    }
  }
  if (lane == 0) *scale = s;
}

template <typename T, int NI>
__global__ __launch_bounds__(128) void k_kv_append(KvAppendArgs a) {
  const unsigned nblocks = a.count ? *a.count : a.nblocks;
  for (unsigned b = blockIdx.x; b < nblocks; b += gridDim.x) append_block<T, NI>(a, a.blocks[b]);
}

template <typename T>
static hipError_t append_typed(const KvAppendArgs& a, unsigned n, hipStream_t st) {
  const dim3 grid(std::min(n, 1u << 20), (unsigned)a.g.kv_heads), block(64, 2);
  if (a.g.hd <= 64) return launch(k_kv_append<T, 1>, grid, block, 0, st, a);
  if (a.g.hd <= 128) return launch(k_kv_append<T, 2>, grid, block, 0, st, a);
  return launch(k_kv_append<T, 4>, grid, block, 0, st, a);
}

hipError_t launch_kv_append(int dtype, const KvAppendArgs& a, unsigned grid, hipStream_t st) {
  if (grid == 0) return hipSuccess;
  switch (dtype) {
    case F32: return append_typed<float>(a, grid, st);
    case F16: return append_typed<_Float16>(a, grid, st);
    case BF16: return append_typed<Bf16>(a, grid, st);
    default: return hipErrorInvalidValue;
  }
}

// ---------------------------------------------------------------------------
// reading back
// ---------------------------------------------------------------------------

__global__ __launch_bounds__(256) void k_kv_read(KvGeom g, size_t layer, uint32_t row, size_t first, size_t count,
                                                 float* k, float* v) {
  const size_t total = count * g.kv_heads * g.hd;
  for (size_t id = (size_t)blockIdx.x * 256 + threadIdx.x; id < total; id += (size_t)gridDim.x * 256) {
    const unsigned d = (unsigned)(id % g.hd);
    const size_t rest = id / g.hd;
    const unsigned head = (unsigned)(rest % g.kv_heads);
    const size_t pos = first + rest / g.kv_heads;
    const uint32_t page = g.table[(size_t)row * g.max_pages + pos / KV_PAGE];
    const uint8_t* region = g.pool + page * g.page_bytes + layer * g.layer_bytes + (size_t)head * g.head_bytes;
    const unsigned t = (unsigned)(pos % KV_PAGE);
    const float* scale = (const float*)(region + g.s_off) + t / KV_BLOCK;
    k[id] = (float)((int)region[kv_key_byte(g.chunks, t, d)] - 128) * scale[0];
    v[id] = (float)((int)region[g.v_off + kv_value_byte(t, d)] - 128) * scale[4];
  }
}

hipError_t launch_kv_read(const KvGeom& g, size_t layer, uint32_t row, size_t first, size_t count, float* k, float* v,
                          hipStream_t st) {
  const size_t total = count * g.kv_heads * g.hd;
  if (total == 0) return hipSuccess;
  return launch(k_kv_read, (unsigned)std::min<size_t>((total + 255) / 256, 1u << 20), 256, 0, st, g, layer, row, first,
                count, k, v);
}

}  // namespace hale
