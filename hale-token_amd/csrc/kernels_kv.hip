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
// Rows of 16-byte pieces: a work-group per row (blockIdx.y: its share of the
// heads) finds the row's cosines and sines once, a thread then turns eight pairs of
// a head at a time, or copies eight numbers behind them.
template <typename T, bool INTERLEAVED>
__global__ __launch_bounds__(256) void k_rope_vec(RopeArgs a) {
  __shared__ float2 cs[512];
  const size_t row = blockIdx.x;
  const int pos = a.pos[row], turned = a.half / 8, rest = (a.hd - 2 * a.half) / 8, per = turned + rest;
  const int units = (a.heads[0] + a.heads[1]) * per;
  for (int e = threadIdx.x; e < a.half; e += 256) rope_angle(pos, a.turns[e], a.factor, &cs[e].x, &cs[e].y);
  __syncthreads();
  union Piece {
    u32x4 u[sizeof(T) / 2];
    T v[8];
  };
  auto load = [](Piece& p, const T* x) {
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) / 2; j++) p.u[j] = ((const u32x4*)x)[j];
  };
  auto store = [](const Piece& p, T* x) {
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) / 2; j++) ((u32x4*)x)[j] = p.u[j];
  };
#pragma unroll 2
  for (int u = blockIdx.y * 256 + threadIdx.x; u < units; u += 256 * gridDim.y) {
    int h = u / per;
    const int j = u % per, which = h >= a.heads[0];
    if (which) h -= a.heads[0];
    const T* x = (const T*)a.src[which] + row * a.src_stride[which] + (size_t)h * a.hd;
    T* y = (T*)a.dst[which] + row * a.dst_stride[which] + (size_t)h * a.hd;
    Piece p, q;
    if (j >= turned) {
      const int d = 2 * a.half + (j - turned) * 8;
      if (x == y) continue;
      load(p, x + d);
      store(p, y + d);
      continue;
    }
    const int d0 = INTERLEAVED ? 16 * j : 8 * j, d1 = INTERLEAVED ? 16 * j + 8 : 8 * j + a.half;
    load(p, x + d0);
    load(q, x + d1);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float2 t = cs[8 * j + e];
      T& s0 = INTERLEAVED ? (e < 4 ? p.v[2 * (e & 3)] : q.v[2 * (e & 3)]) : p.v[e];
      T& s1 = INTERLEAVED ? (e < 4 ? p.v[2 * (e & 3) + 1] : q.v[2 * (e & 3) + 1]) : q.v[e];
      const float f = to_f32(s0), g = to_f32(s1);
      s0 = from_f32<T>(f * t.x - g * t.y);
      s1 = from_f32<T>(g * t.x + f * t.y);
    }
    store(p, y + d0);
    store(q, y + d1);
  }
}

// Any strides, alignments and dimensions: a thread per pair or copied number.
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

constexpr size_t ROPE_VEC_PAIRS = 65536;

template <typename T>
static hipError_t rope_typed(const RopeArgs& a, hipStream_t st) {
  size_t bits = 0;
  for (int i = 0; i < 2; i++)
    if (a.heads[i]) bits |= (uintptr_t)a.src[i] | (uintptr_t)a.dst[i] | (a.src_stride[i] | a.dst_stride[i]) * sizeof(T);
  // few rows are a matter of latency, where a thread per pair is the shorter way
  const size_t pairs = a.rows * (size_t)(a.heads[0] + a.heads[1]) * a.half;
  if (pairs >= ROPE_VEC_PAIRS && bits % 16 == 0 && a.hd % 8 == 0 && a.half % 8 == 0) {
    const int units = (a.heads[0] + a.heads[1]) * (a.half / 8 + (a.hd - 2 * a.half) / 8);
    // few rows: their heads spread over more work-groups
    const unsigned split = a.rows >= 512 ? 1 : (unsigned)(units + 255) / 256;
    const dim3 grid((unsigned)a.rows, split);
    return a.interleaved ? launch(k_rope_vec<T, true>, grid, 256, 0, st, a) : launch(k_rope_vec<T, false>, grid, 256, 0, st, a);
  }
  const size_t total = a.rows * (size_t)(a.heads[0] + a.heads[1]) * (a.hd - a.half);
  if (total == 0) return hipSuccess;
  const unsigned grid = (unsigned)std::min<size_t>((total + 255) / 256, 1u << 20);
  return launch(k_rope<T>, grid, 256, 0, st, a);
}

hipError_t launch_rope(int dtype, const RopeArgs& a, hipStream_t st) {
  switch (dtype) {
    case F32: return rope_typed<float>(a, st);
    case F16: return rope_typed<_Float16>(a, st);
    case BF16: return rope_typed<Bf16>(a, st);
    default: return hipErrorInvalidValue;
  }
}

// ---------------------------------------------------------------------------
// plan upload, page copies
// ---------------------------------------------------------------------------

// A thread per 16 bytes, all of them read at once: the host's memory is a
// microsecond away, once.
__global__ __launch_bounds__(256) void k_kv_upload(KvUploadArgs a, unsigned n4) {
  const unsigned id = blockIdx.x * 256 + threadIdx.x;
  // that this kernel runs says that the one before it has ended
  if (id == 0) __hip_atomic_store(a.done, a.number, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
  if (id < n4) {
    const u32x4 x = ((const u32x4*)a.src)[id];
    unsigned at = id;
    for (int p = 0; p < a.pieces; p++) {
      const unsigned n = a.words[p] / 4;
      if (at < n) {
        ((u32x4*)a.dst[p])[at] = x;
        break;
      }
      at -= n;
    }
  } else if (id - n4 < a.npairs) {
    const unsigned i = id - n4;
    a.table[a.pairs[2 * i]] = a.pairs[2 * i + 1];
  }
}

hipError_t launch_kv_upload(const KvUploadArgs& a, hipStream_t st) {
  unsigned n4 = 0;
  for (int p = 0; p < a.pieces; p++) n4 += a.words[p] / 4;
  if (n4 + a.npairs == 0) return hipSuccess;
  return launch(k_kv_upload, (n4 + a.npairs + 255) / 256, 256, 0, st, a, n4);
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
// One work-group per block of 16 positions, head, and keys or values: the new
// rows go to LDS as f32 on the way to the largest magnitude; the block's scale
// from it and the former one; then the codes, each thread those of the bytes it writes:
// 8 consecutive numbers of one position of the keys, four positions of one number
// of the values, so that no thread's bytes depend on another's.  A decode step's
// call is a chain of latencies (the block, its page, scale and codes, the
// rounding of held codes where the scale grew, about 20 dependent instructions
// each): four waves share a block, 8 codes a thread at head dimension 128.

// The whole number nearest to (p + e) / s, ties to even, where |p / s| < 200, e is
// the rest of a product rounded to p (or 0), and inv is within 2^-21 of 1 / s
// relative.  p inv is off by less than 2^-13, so its nearest whole number c is
// the quotient's or the one beside it; p - c s, of at most half of s and a little,
// is a multiple of the smaller of both ulps and so exact, as is 2 |p - c s| - s
// where it is near 0; the sign of that with e decides.
__device__ __forceinline__ unsigned nearest_code(float p, float e, float s, float inv) {
  float c = rintf(p * inv);
  const float r = __builtin_fmaf(-c, s, p);
  const float over = (2.0f * fabsf(r) - s) + 2.0f * (r < 0.0f ? -e : e);
  const bool odd = ((int)c & 1) != 0;
  c += over > 0.0f || (over == 0.0f && odd) ? (r > 0.0f ? 1.0f : -1.0f) : 0.0f;
  return (unsigned)((int)fminf(fmaxf(c, -127.0f), 127.0f) + 128);
}

// A lane's number n of the keys, n a multiple of 8: which of the dimension
// it is (lane group g), and where its code and the next seven go.
__device__ __forceinline__ int key_dim(int kc, int n, int g) {
  return n / 16 < kc / 2 ? 64 * (n / 16) + 16 * g + n % 16 : 64 * (kc / 2) + 8 * g;
}
__device__ __forceinline__ unsigned key_at(int kc, int n, int block, int lane) {
  return n / 16 < kc / 2 ? ((n / 16 * 4 + block) * 64 + lane) * 16 + n % 16 : kc / 2 * 4096 + (block * 64 + lane) * 8;
}

template <typename T>
__global__ __launch_bounds__(256) void k_kv_append(KvAppendArgs a) {
  extern __shared__ float x[];  // [16][hd + 4]
  __shared__ float red[4];
  const int tid = threadIdx.x, hd = a.g.hd, ldx = hd + 4;
  const bool values = blockIdx.z;
  const size_t stride = values ? a.v_stride : a.k_stride;
  const T* base = (const T*)(values ? a.v : a.k) + (size_t)blockIdx.y * hd;
  const KvBlock first = a.blocks[blockIdx.x];  // read beside the count: the plan has room for the whole grid
  const unsigned nblocks = a.count ? *a.count : a.nblocks;
  for (unsigned b = blockIdx.x; b < nblocks; b += gridDim.x) {
    const KvBlock blk = b == blockIdx.x ? first : a.blocks[b];
    const int old = blk.old, end = blk.end;
    const uint32_t page = a.g.table[blk.entry];
    const T* src = base + (long long)blk.tok * (long long)stride;
    uint8_t* region = a.g.pool + page * a.g.page_bytes + a.layer * a.g.layer_bytes + (size_t)blockIdx.y * a.g.head_bytes;
    float* scale = (float*)(region + a.g.s_off) + (values ? 4 : 0) + blk.block;
    const float had = old ? *scale : 0.0f;

    float top = 0.0f;
    auto keep = [&](int t, int d, float v) {
      v = __builtin_isfinite(v) ? v : 0.0f;  // what is not finite is stored as 0 and raises no scale
      top = fmaxf(top, fabsf(v));
      x[t * ldx + d] = v;
    };
    if (a.vec) {
      constexpr int PER = 16 / sizeof(T);
      const int row = hd / PER, n = (end - old) * row;  // 16-byte pieces
      for (int e = tid; e < n; e += 256) {
        const int t = old + e / row, d = e % row * PER;
        union {
          u32x4 u;
          T v[PER];
        } r;
        r.u = *(const u32x4*)(src + (size_t)t * stride + d);
#pragma unroll
        for (int j = 0; j < PER; j++) keep(t, d + j, to_f32(r.v[j]));
      }
    } else {
      const int n = (end - old) * hd;
#pragma unroll 4
      for (int e = tid; e < n; e += 256) {
        const int t = old + e / hd, d = e % hd;
        keep(t, d, to_f32(src[(size_t)t * stride + d]));
      }
    }
    top = wave_max_f32(top);
    if (tid % 64 == 0) red[tid / 64] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float s = fmaxf(had, top / 127.0f);
    const bool grown = old && s > had;
    // the reciprocal of a very small scale overflows: both sides times 2^64, exactly
    const float up = s < 0x1p-64f ? 0x1p64f : 1.0f, su = s * up, hu = had * up;
    const float inv = s > 0.0f ? 1.0f / su : 0.0f;  // scale 0: all numbers are 0, and so are their quotients
    auto code = [&](bool held, unsigned was, float v) {
      const float c = (float)((int)was - 128), m = c * hu;
      return nearest_code(held ? m : v * up, held ? __builtin_fmaf(c, hu, -m) : 0.0f, su, inv);
    };
    if (!values) {
      // thread: position i, numbers d .. d + 7 (lane and piece as in kv_key_byte)
      for (int e = tid; e < a.g.chunks * 64; e += 256) {
        const int lane = e % 64, i = lane % 16, n = e / 64 * 8;
        const int d = key_dim(a.g.chunks, n, lane / 16);
        const bool held = i < old;
        if (d >= hd || !(held ? grown : i < end)) continue;
        u32x2* at = (u32x2*)(region + key_at(a.g.chunks, n, blk.block, lane));
        u32x2 o = {0, 0}, w;
        f32x4 v[2] = {};
        if (held) {
          o = *at;
        } else {
          v[0] = *(const f32x4*)(x + i * ldx + d);
          v[1] = *(const f32x4*)(x + i * ldx + d + 4);
        }
#pragma unroll
        for (int j = 0; j < 2; j++) {
          w[j] = 0;
#pragma unroll
          for (int k = 0; k < 4; k++) w[j] |= code(held, o[j] >> (8 * k) & 255, v[j][k]) << (8 * k);
        }
        *at = w;
      }
    } else {
      // thread: number d = 16 n + i, positions 4 g .. 4 g + 3
#pragma unroll 2
      for (int e = tid; e < hd * 4; e += 256) {
        const int lane = e % 64, i = lane % 16, g = lane / 16, n = e / 64;
        if (4 * g >= end || !(grown || 4 * g + 3 >= old)) continue;
        unsigned* at = (unsigned*)(region + a.g.v_off + e * 16 + 4 * blk.block);
        const unsigned o = 4 * g < old ? *at : 0;
        unsigned w = 0;
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int t = 4 * g + r;
          const float v = t >= old && t < end ? x[t * ldx + 16 * n + i] : 0.0f;
          w |= code(t < old, o >> (8 * r) & 255, v) << (8 * r);
        }
        *at = w;
      }
    }
    if (tid == 0) *scale = s;
    __syncthreads();  // the next block's rows may overwrite these
  }
}

template <typename T>
static hipError_t append_typed(const KvAppendArgs& a, unsigned n, hipStream_t st) {
  const dim3 grid(std::min(n, 1u << 20), (unsigned)a.g.kv_heads, 2);
  return launch(k_kv_append<T>, grid, 256, (uint32_t)(KV_BLOCK * (a.g.hd + 4) * 4), st, a);
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

// A work-group per page, head, and keys or values; a lane reads 16 bytes as they
// lie: 16 numbers of one position of the keys (four 16-byte stores, 64 bytes of
// a row), 16 positions of one number of the values (16 stores, of which a wave's
// make 64-byte pieces of four rows).
__global__ __launch_bounds__(256) void k_kv_read(KvGeom g, size_t layer, uint32_t row, size_t first, size_t count,
                                                 float* k, float* v) {
  const size_t p = first / KV_PAGE + blockIdx.x;
  const int head = blockIdx.y, hd = g.hd;
  const uint8_t* region = g.pool + g.table[(size_t)row * g.max_pages + p] * g.page_bytes + layer * g.layer_bytes +
                          (size_t)head * g.head_bytes;
  const long long base = (long long)(p * KV_PAGE) - (long long)first;  // output row of the page's position 0
  const size_t stride = (size_t)g.kv_heads * hd;
  const f32x4 s = *(const f32x4*)(region + g.s_off + (blockIdx.z ? 16 : 0));
  auto row_of = [&](int t) { return base + t; };
  auto wanted = [&](long long r) { return r >= 0 && r < (long long)count; };
  if (blockIdx.z == 0) {
    float* out = k + (size_t)head * hd;
    const int whole = g.chunks / 2 * 256;
    for (int e = threadIdx.x; e < whole; e += 256) {
      const int lane = e % 64, mm = e / 64 % 4, d = e / 256 * 64 + lane / 16 * 16;
      const long long r = row_of(16 * mm + lane % 16);
      if (!wanted(r) || d >= hd) continue;
      const u32x4 w = *(const u32x4*)(region + e * 16);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        f32x4 x;
#pragma unroll
        for (int b = 0; b < 4; b++) x[b] = (float)((int)(w[j] >> (8 * b) & 255) - 128) * s[mm];
        *(f32x4u*)(out + r * stride + d + 4 * j) = x;
      }
    }
    if (g.chunks & 1) {
      const int lane = threadIdx.x % 64, mm = threadIdx.x / 64, d = g.chunks / 2 * 64 + lane / 16 * 8;
      const long long r = row_of(16 * mm + lane % 16);
      if (wanted(r) && d < hd) {
        const u32x2 w = *(const u32x2*)(region + whole * 16 + threadIdx.x * 8);
#pragma unroll
        for (int j = 0; j < 2; j++) {
          f32x4 x;
#pragma unroll
          for (int b = 0; b < 4; b++) x[b] = (float)((int)(w[j] >> (8 * b) & 255) - 128) * s[mm];
          *(f32x4u*)(out + r * stride + d + 4 * j) = x;
        }
      }
    }
  } else {
    for (int e = threadIdx.x; e < hd * 4; e += 256) {
      const int lane = e % 64, d = e / 64 * 16 + lane % 16;
      const u32x4 w = *(const u32x4*)(region + g.v_off + e * 16);
      float* out = v + (size_t)head * hd + d;
#pragma unroll
      for (int mm = 0; mm < 4; mm++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const long long r = row_of(16 * mm + lane / 16 * 4 + j);
          if (wanted(r)) out[r * stride] = (float)((int)(w[mm] >> (8 * j) & 255) - 128) * s[mm];
        }
    }
  }
}

hipError_t launch_kv_read(const KvGeom& g, size_t layer, uint32_t row, size_t first, size_t count, float* k, float* v,
                          hipStream_t st) {
  if (count == 0) return hipSuccess;
  const size_t pages = (first + count - 1) / KV_PAGE - first / KV_PAGE + 1;
  return launch(k_kv_read, dim3((unsigned)pages, (unsigned)g.kv_heads, 2), 256, 0, st, g, layer, row, first, count, k, v);
}

}  // namespace hale
