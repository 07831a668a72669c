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
// a head at a time, or copies eight numbers behind them.  Bound by memory: 2048 bf16 rows of
// 40 heads of 128, 42 MB, take 10 us (4.2 TB/s, where a large copy reaches 4.85).
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

// Any strides, alignments and dimensions: a thread per pair or copied number.  One
// row of 36 f32 heads of 128 takes 2.7 us, little more than an empty launch.
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

constexpr size_t ROPE_VEC_PAIRS = 1u << 18;
// Work-groups of 256 in a grid's dimension, whose threads are counted in 32 bits.
constexpr unsigned MAX_GROUPS = (1u << 24) - 1;

template <typename T>
static hipError_t rope_typed(const RopeArgs& a, hipStream_t st) {
  size_t bits = 0;
  for (int i = 0; i < 2; i++)
    if (a.heads[i]) bits |= (uintptr_t)a.src[i] | (uintptr_t)a.dst[i] | (a.src_stride[i] | a.dst_stride[i]) * sizeof(T);
  // few rows are a matter of latency, where a thread per pair is the shorter way (36
  // bf16 heads of 128, per pair / in pieces: 16 rows 2.7 / 3.2 us, 112 3.4 / 3.4, 224 4.5 / 3.6)
  const size_t pairs = a.rows * (size_t)(a.heads[0] + a.heads[1]) * a.half;
  if (pairs >= ROPE_VEC_PAIRS && bits % 16 == 0 && a.hd % 8 == 0 && a.half % 8 == 0) {
    const int units = (a.heads[0] + a.heads[1]) * (a.half / 8 + (a.hd - 2 * a.half) / 8);
    // few rows: their heads spread over more work-groups (bf16, 40 heads of 128, split / not:
    // 700 rows 4.7 / 5.6 us, 1024 5.8 / 6.8, 2048 9.8 / 9.2)
    const unsigned split = a.rows > 1024 ? 1 : (unsigned)(units + 255) / 256;
    RopeArgs b = a;
    for (size_t row = 0; row < a.rows; row += b.rows) {
      b.rows = std::min<size_t>(a.rows - row, MAX_GROUPS);
      b.pos = a.pos + row;
      for (int i = 0; i < 2; i++) {
        if (!a.heads[i]) continue;
        b.src[i] = (const T*)a.src[i] + row * a.src_stride[i];
        b.dst[i] = (T*)a.dst[i] + row * a.dst_stride[i];
      }
      const dim3 grid((unsigned)b.rows, split);
      const hipError_t e =
          a.interleaved ? launch(k_rope_vec<T, true>, grid, 256, 0, st, b) : launch(k_rope_vec<T, false>, grid, 256, 0, st, b);
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
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
// plan upload and page copies
// ---------------------------------------------------------------------------

// One launch for what a step or a page operation sends and moves: the first
// work-groups take a thread per 16 bytes of the plan, all of them read at once
// (the host's memory is a microsecond or two away, once), the others a piece of a
// page each, whose place they read from the same buffer.  A step of 16 sequences takes
// 4.6 us, a launch and the way to the host; 94 pages of 4 layers of 4 heads of 128 (50
// MB read and written) take 10 us, 5.0 TB/s.
constexpr unsigned COPY_BYTES = 16384;  // per work-group: four 16-byte pieces a thread

__global__ __launch_bounds__(256) void k_kv_upload(KvUploadArgs a, unsigned n4, unsigned uploads, unsigned chunks) {
  if (blockIdx.x >= uploads) {
    const unsigned w = blockIdx.x - uploads;
    const KvCopy c = a.copies[w / chunks];
    const size_t at = (size_t)(w % chunks) * COPY_BYTES;
    const u32x4* s = (const u32x4*)(a.pool + c.src * a.page_bytes + at);
    u32x4* d = (u32x4*)(a.pool + c.dst * a.page_bytes + at);
    const unsigned n = (unsigned)(a.page_bytes - at < COPY_BYTES ? a.page_bytes - at : COPY_BYTES) / 16;
    u32x4 x[4];
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (threadIdx.x + 256 * j < n) x[j] = s[threadIdx.x + 256 * j];
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (threadIdx.x + 256 * j < n) d[threadIdx.x + 256 * j] = x[j];
    return;
  }
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
  const unsigned uploads = (n4 + a.npairs + 255) / 256 + (n4 + a.npairs == 0);
  const size_t chunks = (a.page_bytes + COPY_BYTES - 1) / COPY_BYTES;
  const size_t most = (MAX_GROUPS - uploads) / chunks;
  KvUploadArgs b = a;
  for (bool first = true; first || b.ncopies; first = false) {
    const unsigned n = (unsigned)std::min<size_t>(b.ncopies, most);
    const hipError_t e = launch(k_kv_upload, uploads + n * (unsigned)chunks, 256, 0, st, b, n4, uploads, (unsigned)chunks);
    if (e != hipSuccess) return e;
    b.copies += n;
    b.ncopies -= n;
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

// The whole numbers nearest to (p + e) / s, ties to even, as four codes of a word,
// where |p / s| < 200, e is the rest of a product rounded to p (or 0), and inv is
// within 2^-21 of 1 / s relative.  p inv is off by less than 2^-13: where it is
// farther than that from a half, its nearest whole number c is the quotient's.  Else
// (one number in 2500) c or the one beside it is: p - c s, of at most half of s and a
// little, is a multiple of the smaller of both ulps and so exact, as is 2 |p - c s|
// - s where it is near 0; the sign of that with e decides.
__device__ __forceinline__ unsigned nearest_codes(const float (&p)[4], const float (&e)[4], float s, float inv) {
  float c[4];
  unsigned far = 0;  // magnitudes are ordered as their bits are
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const float t = p[k] * inv;
    c[k] = rintf(t);
    far = max(far, __float_as_uint(fabsf(t - c[k])));
  }
  if (__builtin_amdgcn_ballot_w64(far > __float_as_uint(0.4998f))) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const float r = __builtin_fmaf(-c[k], s, p[k]);
      const float over = (2.0f * fabsf(r) - s) + 2.0f * (r < 0.0f ? -e[k] : e[k]);
      const bool odd = ((int)c[k] & 1) != 0;
      c[k] += over > 0.0f || (over == 0.0f && odd) ? (r > 0.0f ? 1.0f : -1.0f) : 0.0f;
    }
  }
  unsigned w = 0;
#pragma unroll
  for (int k = 0; k < 4; k++) w = __builtin_amdgcn_cvt_pk_u8_f32(__builtin_amdgcn_fmed3f(c[k], -127.0f, 127.0f) + 128.0f, k, w);
  return w;
}

// A lane's number n of the keys, n a multiple of 8: which of the dimension
// it is (lane group g), and where its code and the next seven go.
__device__ __forceinline__ int key_dim(int kc, int n, int g) {
  return n / 16 < kc / 2 ? 64 * (n / 16) + 16 * g + n % 16 : 64 * (kc / 2) + 8 * g;
}
__device__ __forceinline__ unsigned key_at(int kc, int n, int block, int lane) {
  return n / 16 < kc / 2 ? ((n / 16 * 4 + block) * 64 + lane) * 16 + n % 16 : kc / 2 * 4096 + (block * 64 + lane) * 8;
}

//
// W: waves per block, 4 or 1.  Four where few blocks leave the chain to be shortened; one
// where there are many (bf16, 8 heads of 128, this kernel alone, four / one: 512 tokens
// 5.7 / 7.6 us, 1024 7.2 / 8.0, 2048 12.0 / 10.3, 4090 17.3 / 12.4).  A prompt of 4090
// reads 17 MB and writes 8 in 12.8 us: its 1024 work-groups all run at once, and so do
// their loads, maxima and roundings, one behind the other; by the counters the vector
// units work for 6 of them.
template <typename T, int W>
__global__ __launch_bounds__(256) void k_kv_append(KvAppendArgs a) {
  extern __shared__ float lds[];  // [4 / W][16][hd + 4]
  __shared__ float red[4];
  constexpr int N = 64 * W;  // threads of a block
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), mine = wave / W;
  const int tid = threadIdx.x % N, hd = a.g.hd, ldx = hd + 4;
  float* x = lds + mine * (int)KV_BLOCK * ldx;
  const bool values = blockIdx.z;
  const size_t stride = values ? a.v_stride : a.k_stride;
  const T* base = (const T*)(values ? a.v : a.k) + (size_t)blockIdx.y * hd;
  // read beside the count: the plan has room for the whole grid
  const unsigned b0 = blockIdx.x * (4 / W) + mine;
  KvBlock blk = a.blocks[b0];
  const unsigned nblocks = a.count ? *a.count : a.nblocks;
  for (unsigned b = b0; b < nblocks; b += gridDim.x * (4 / W)) {
    if (b != b0) blk = a.blocks[b];
    const int old = blk.old, end = blk.end;
    const uint32_t page = a.g.table[blk.entry];
    const T* src = base + (long long)blk.tok * (long long)stride;
    uint8_t* region = a.g.pool + page * a.g.page_bytes + a.layer * a.g.layer_bytes + (size_t)blockIdx.y * a.g.head_bytes;
    float* scale = (float*)(region + a.g.s_off) + (values ? 4 : 0) + blk.block;
    const float had = old ? *scale : 0.0f;

    unsigned bits = 0;  // of the largest magnitude
    auto keep = [&](int t, int d, float v) {
      // what is not finite is stored as 0 and raises no scale
      const unsigned u = __float_as_uint(v) & 0x7fffffffu, m = u < 0x7f800000u ? u : 0u;
      bits = max(bits, m);
      x[t * ldx + d] = u < 0x7f800000u ? v : 0.0f;
    };
    if (a.vec) {
      constexpr int PER = 16 / sizeof(T);
      const int row = hd / PER, n = (end - old) * row;  // 16-byte pieces
      const unsigned inv_row = (1u << 20) / row + 1;     // e / row exactly for e row < 2^20
#pragma unroll 4
      for (int e = tid; e < n; e += N) {
        const int q = (int)(e * inv_row >> 20), t = old + q, d = (e - q * row) * PER;
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
      for (int e = tid; e < n; e += N) {
        const int t = old + e / hd, d = e % hd;
        keep(t, d, to_f32(src[(size_t)t * stride + d]));
      }
    }
    float top = __uint_as_float(wave_max_u32(bits));
    if constexpr (W == 4) {
      if (tid % 64 == 0) red[wave] = top;
      __syncthreads();
      top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    } else {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave's rows, before other lanes read them
    }
    const float s = fmaxf(had, top / 127.0f);
    const bool grown = old && s > had;
    // the reciprocal of a very small scale overflows: both sides times 2^64, exactly
    const float up = s < 0x1p-64f ? 0x1p64f : 1.0f, su = s * up, hu = had * up;
    const float inv = s > 0.0f ? 1.0f / su : 0.0f;  // scale 0: all numbers are 0, and so are their quotients
    // four codes: of new numbers v, or where `held` says so of the codes `was`
    auto codes = [&](const bool (&held)[4], unsigned was, const float (&v)[4]) {
      float p[4], e[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        p[k] = v[k] * up;
        e[k] = 0.0f;
        if (old) {
          const float c = (float)((int)(was >> (8 * k) & 255) - 128), m = c * hu;
          e[k] = held[k] ? __builtin_fmaf(c, hu, -m) : 0.0f;
          p[k] = held[k] ? m : p[k];
        }
      }
      return nearest_codes(p, e, su, inv);
    };
    if (W == 1 && old == 0 && end == (int)KV_BLOCK) {
      // a whole new block, as most of a prompt are: the same without conditions
      const int lane = tid, i = lane % 16, g = lane / 16;
      const float none[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (!values) {
        const int full = hd / 64 * 16;  // numbers of a lane whose 16 consecutive ones all exist
#pragma unroll 2
        for (int n = 0; n < full; n += 8) {
          const float* v = x + i * ldx + key_dim(a.g.chunks, n, g);
          const f32x4 v0 = *(const f32x4*)v * up, v1 = *(const f32x4*)(v + 4) * up;
          *(u32x2*)(region + key_at(a.g.chunks, n, blk.block, lane)) =
              u32x2{nearest_codes({v0[0], v0[1], v0[2], v0[3]}, none, su, inv), nearest_codes({v1[0], v1[1], v1[2], v1[3]}, none, su, inv)};
        }
        for (int n = full; n < a.g.chunks * 8; n += 8) {
          const int d = key_dim(a.g.chunks, n, g);
          if (d >= hd) continue;
          const float* v = x + i * ldx + d;
          const f32x4 v0 = *(const f32x4*)v * up, v1 = *(const f32x4*)(v + 4) * up;
          *(u32x2*)(region + key_at(a.g.chunks, n, blk.block, lane)) =
              u32x2{nearest_codes({v0[0], v0[1], v0[2], v0[3]}, none, su, inv), nearest_codes({v1[0], v1[1], v1[2], v1[3]}, none, su, inv)};
        }
      } else {
        const float* v = x + 4 * g * ldx + i;
        unsigned* at = (unsigned*)(region + a.g.v_off + lane * 16 + 4 * blk.block);
#pragma unroll 4
        for (int n = 0; n < hd / 16; n++, v += 16, at += 256)
          *at = nearest_codes({v[0] * up, v[ldx] * up, v[2 * ldx] * up, v[3 * ldx] * up}, none, su, inv);
      }
    } else if (!values) {
      // thread: position i, numbers d .. d + 7 (lane and piece as in kv_key_byte)
      for (int e = tid; e < a.g.chunks * 64; e += N) {
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
        for (int j = 0; j < 2; j++) w[j] = codes({held, held, held, held}, o[j], {v[j][0], v[j][1], v[j][2], v[j][3]});
        *at = w;
      }
    } else {
      // thread: number d = 16 n + i, positions 4 g .. 4 g + 3
#pragma unroll 2
      for (int e = tid; e < hd * 4; e += N) {
        const int lane = e % 64, i = lane % 16, g = lane / 16, n = e / 64;
        if (4 * g >= end || !(grown || 4 * g + 3 >= old)) continue;
        unsigned* at = (unsigned*)(region + a.g.v_off + e * 16 + 4 * blk.block);
        const unsigned o = 4 * g < old ? *at : 0;
        float v[4];
        bool held[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int t = 4 * g + r;
          v[r] = t >= old && t < end ? x[t * ldx + 16 * n + i] : 0.0f;
          held[r] = t < old;
        }
        *at = codes(held, o, v);
      }
    }
    if (tid == 0) *scale = s;
    // the next block's rows overwrite these
    if constexpr (W == 4)
      __syncthreads();
    else
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// More than 64 KiB of LDS is asked for.
template <typename K>
static hipError_t allow_lds(K kernel, uint32_t lds) {
  if (lds <= 65536) return hipSuccess;
  return hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
}

template <typename T>
static hipError_t append_typed(const KvAppendArgs& a, unsigned n, hipStream_t st) {
  const uint32_t lds = (uint32_t)(KV_BLOCK * (a.g.hd + 4) * 4);
  const unsigned most = 1u << 20;
  if ((size_t)n * a.g.kv_heads * 2 <= 1024)
    return launch(k_kv_append<T, 4>, dim3(n, (unsigned)a.g.kv_heads, 2), 256, lds, st, a);
  const hipError_t e = allow_lds(k_kv_append<T, 1>, 4 * lds);
  if (e != hipSuccess) return e;
  return launch(k_kv_append<T, 1>, dim3(std::min((n + 3) / 4, most), (unsigned)a.g.kv_heads, 2), 256, 4 * lds, st, a);
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

// A work-group per page, head, and keys or values: 16 bytes a lane as they lie,
// through LDS into whole rows.  Bound by memory: 4090 positions of 8 heads of 128 take 8.8
// us, 8.4 MB read and 33.5 written (4.8 TB/s).
__global__ __launch_bounds__(256) void k_kv_read(KvGeom g, size_t layer, uint32_t row, size_t first, size_t count,
                                                 float* k, float* v) {
  extern __shared__ float x[];  // [64][hd + 4]
  const size_t p = first / KV_PAGE + blockIdx.x;
  const int head = blockIdx.y, hd = g.hd, ldx = hd + 4, tid = threadIdx.x;
  const uint8_t* region = g.pool + g.table[(size_t)row * g.max_pages + p] * g.page_bytes + layer * g.layer_bytes +
                          (size_t)head * g.head_bytes;
  const f32x4 s = *(const f32x4*)(region + g.s_off + (blockIdx.z ? 16 : 0));
  auto value = [](unsigned w, int b, float scale) { return (float)((int)(w >> (8 * b) & 255) - 128) * scale; };
  if (blockIdx.z == 0) {
    const int whole = g.chunks / 2 * 256;
    for (int e = tid; e < whole; e += 256) {
      const int lane = e % 64, mm = e / 64 % 4, d = e / 256 * 64 + lane / 16 * 16;
      if (d >= hd) continue;
      const u32x4 w = *(const u32x4*)(region + e * 16);
      float* at = x + (16 * mm + lane % 16) * ldx + d;
#pragma unroll
      for (int j = 0; j < 4; j++)
        *(f32x4*)(at + 4 * j) = f32x4{value(w[j], 0, s[mm]), value(w[j], 1, s[mm]), value(w[j], 2, s[mm]), value(w[j], 3, s[mm])};
    }
    if (g.chunks & 1) {
      const int lane = tid % 64, mm = tid / 64, d = g.chunks / 2 * 64 + lane / 16 * 8;
      if (d < hd) {
        const u32x2 w = *(const u32x2*)(region + whole * 16 + tid * 8);
        float* at = x + (16 * mm + lane % 16) * ldx + d;
#pragma unroll
        for (int j = 0; j < 2; j++)
          *(f32x4*)(at + 4 * j) = f32x4{value(w[j], 0, s[mm]), value(w[j], 1, s[mm]), value(w[j], 2, s[mm]), value(w[j], 3, s[mm])};
      }
    }
  } else {
    for (int e = tid; e < hd * 4; e += 256) {
      const int lane = e % 64;
      const u32x4 w = *(const u32x4*)(region + g.v_off + e * 16);
      float* at = x + lane / 16 * 4 * ldx + e / 64 * 16 + lane % 16;
#pragma unroll
      for (int mm = 0; mm < 4; mm++)
#pragma unroll
        for (int j = 0; j < 4; j++) at[(16 * mm + j) * ldx] = value(w[mm], j, s[mm]);
    }
  }
  __syncthreads();
  // the page's positions that are asked for
  const size_t pos0 = p * KV_PAGE;
  const int t0 = first > pos0 ? (int)(first - pos0) : 0;
  const int t1 = first + count - pos0 < KV_PAGE ? (int)(first + count - pos0) : (int)KV_PAGE;
  float* out = (blockIdx.z ? v : k) + (size_t)head * hd;
  const size_t stride = (size_t)g.kv_heads * hd;
  const int quads = hd / 4, n = (t1 - t0) * quads;
  for (int e = tid; e < n; e += 256) {
    const int t = t0 + e / quads, d = e % quads * 4;
    *(f32x4u*)(out + (pos0 + t - first) * stride + d) = *(const f32x4*)(x + t * ldx + d);
  }
}

hipError_t launch_kv_read(const KvGeom& g, size_t layer, uint32_t row, size_t first, size_t count, float* k, float* v,
                          hipStream_t st) {
  if (count == 0) return hipSuccess;
  const size_t pages = (first + count - 1) / KV_PAGE - first / KV_PAGE + 1;
  const uint32_t lds = (uint32_t)(KV_PAGE * (g.hd + 4) * 4);
  const hipError_t e = allow_lds(k_kv_read, lds);
  if (e != hipSuccess) return e;
  return launch(k_kv_read, dim3((unsigned)pages, (unsigned)g.kv_heads, 2), 256, lds, st, g, layer, row, first, count, k, v);
}

}  // namespace hale
