// kernels_q4g.hip -- products of 4-bit weights with group scales and one to
// many tokens.
//
// out[t][r] = sum over groups of scale[r][group] (sum_k q[r][k] x[t][k] - zero[r][group]
// sum_k x[t][k]).  Within a group both sums are matrix products of whole numbers (16 + q, and
// ones; the 16 goes with the zero) with x: of f16 and bf16 exactly, of f32 as three
// bf16 parts that add up to it, of 8-bit codes in whole numbers.  Their accumulators and
// the sum over groups are f32 (i32 within a unit of 8-bit codes), rounded at the size of sums of 16 + q, some
// five times that of q - zero: for f16 and bf16 far below a result's own rounding, for f32 what
// products() and the streaming kernel's sums keep to few roundings.  Layout of the weights:
// step_ops.h.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "hale_device.h"
#include "kernels.h"
#include "kv_device.h"
#include "step_ops.h"

namespace hale {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// ---- laying out and back ---------------------------------------------------------

// The word of codes at `word` of a tile's chunk holds numbers k0 .. k0 + 7 of row i,
// number b in bits code_bit(b) ..
__device__ __forceinline__ void q4g_word(unsigned word, unsigned* i, unsigned* k0) {
  const unsigned lane = word / 4, j = word % 4;
  *i = lane % 16;
  *k0 = 32 * j + 8 * (lane / 16);
}
__device__ __forceinline__ constexpr int code_bit(int b) { return 4 * (b / 2) + 16 * (b % 2); }

__global__ __launch_bounds__(256) void k_q4g_pack(Q4gGeom g, const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros) {
  const size_t tile = blockIdx.x;
  for (unsigned c = blockIdx.y; c < g.chunks; c += gridDim.y) {
    uint8_t* to = g.data + tile * g.tile_bytes + (size_t)c * 1024;
    unsigned i, k0;
    q4g_word(threadIdx.x, &i, &k0);
    const size_t row = tile * Q4G_ROWS + i, k = (size_t)c * Q4G_CHUNK + k0;
    unsigned w = 0x88888888u;
    if (row < g.rows && k < g.cols) {
      const uint8_t* p = codes + row * (g.cols / 2) + k / 2;
      w = 0;
#pragma unroll
      for (int b = 0; b < 8; b++) w |= (unsigned)(p[b / 2] >> (4 * (b % 2)) & 15) << code_bit(b);
    }
    ((uint32_t*)to)[threadIdx.x] = w;
    if (threadIdx.x < 16 * g.per) {
      const unsigned r = threadIdx.x % 4 + threadIdx.x / (4 * g.per) * 4, s = threadIdx.x / 4 % g.per;
      const size_t at = tile * Q4G_ROWS + r, group = (size_t)c * g.per + s;
      const bool in = at < g.rows && group * g.group < g.cols;
      const size_t from = at * (g.cols / g.group) + group;
      ((uint16_t*)(g.data + tile * g.tile_bytes + g.scales_at))[c * 16 * g.per + threadIdx.x] = in ? scales[from] : 0;
      if (g.zeros)
        (const_cast<uint8_t*>(g.zero_data) + tile * g.zero_tile)[c * g.zero_chunk + threadIdx.x] = Q4G_OFFSET + (in ? zeros[from] & 15 : 8);
    }
  }
}

__global__ __launch_bounds__(256) void k_q4g_unpack(Q4gGeom g, uint8_t* codes, uint16_t* scales, uint8_t* zeros) {
  const size_t tile = blockIdx.x;
  for (unsigned c = blockIdx.y; c < g.chunks; c += gridDim.y) {
    const uint8_t* from = g.data + tile * g.tile_bytes + (size_t)c * 1024;
    unsigned i, k0;
    q4g_word(threadIdx.x, &i, &k0);
    const size_t row = tile * Q4G_ROWS + i, k = (size_t)c * Q4G_CHUNK + k0;
    const unsigned w = ((const uint32_t*)from)[threadIdx.x];
    if (row < g.rows && k < g.cols) {
      uint8_t* p = codes + row * (g.cols / 2) + k / 2;
#pragma unroll
      for (int b = 0; b < 8; b += 2) p[b / 2] = (uint8_t)((w >> code_bit(b) & 15) | (w >> code_bit(b + 1) & 15) << 4);
    }
    if (threadIdx.x < 16 * g.per) {
      const unsigned r = threadIdx.x % 4 + threadIdx.x / (4 * g.per) * 4, s = threadIdx.x / 4 % g.per;
      const size_t at = tile * Q4G_ROWS + r, group = (size_t)c * g.per + s;
      if (at < g.rows && group * g.group < g.cols) {
        const size_t to = at * (g.cols / g.group) + group;
        scales[to] = ((const uint16_t*)(g.data + tile * g.tile_bytes + g.scales_at))[c * 16 * g.per + threadIdx.x];
        if (zeros) zeros[to] = g.zeros ? (g.zero_data + tile * g.zero_tile)[c * g.zero_chunk + threadIdx.x] - Q4G_OFFSET : 8;
      }
    }
  }
}

// ---- operands ----------------------------------------------------------------------

// Input types: what a lane holds of eight numbers of a token, and of the weights.
template <int IN> struct Q4gType {  // Q4G_F32, Q4G_BF16
  static constexpr int PARTS = IN == Q4G_F32 ? 3 : 1, SIZE = IN == Q4G_F32 ? 4 : 2;
  typedef bf16x8 Frag;
  typedef f32x4 Acc;
  typedef float Sum;
};
template <> struct Q4gType<Q4G_F16> {
  static constexpr int PARTS = 1, SIZE = 2;
  typedef f16x8 Frag;
  typedef f32x4 Acc;
  typedef float Sum;
};
template <> struct Q4gType<Q4G_I8> {
  static constexpr int PARTS = 1, SIZE = 1;
  typedef u32x2 Frag;
  typedef i32x4 Acc;
  typedef int Sum;
};

// A word's eight codes, each 16 + q.  16 .. 31 are consecutive steps of a float's mantissa:
// the four bits of a code go into it below the pattern of 16, one instruction for a pair
// (conversions to floats are one for each number and another to join a pair).
template <int IN> __device__ __forceinline__ typename Q4gType<IN>::Frag codes8(unsigned w) {
  if constexpr (IN == Q4G_I8) {
    return u32x2{(w & 0x0f0f0f0fu) | 0x10101010u, (w >> 4 & 0x0f0f0f0fu) | 0x10101010u};
  } else {
    constexpr int AT = IN == Q4G_F16 ? 6 : 3;  // of a code in the mantissa
    unsigned base = IN == Q4G_F16 ? 0x4c004c00u : 0x41804180u, mask = 0x000f000fu << AT;
    asm("" : "+v"(base), "+s"(mask));  // in registers, as the instruction of both operations takes them
    union {
      unsigned u[4];
      typename Q4gType<IN>::Frag v;
    } r;
#pragma unroll
    for (int p = 0; p < 4; p++) {
      const unsigned m = 4 * p <= AT ? w << (AT - 4 * p) : w >> (4 * p - AT);
      r.u[p] = (m & mask) | base;
    }
    return r.v;
  }
}
template <int IN> __device__ __forceinline__ typename Q4gType<IN>::Frag ones8() {
  if constexpr (IN == Q4G_I8) {
    return u32x2{0x01010101u, 0x01010101u};
  } else {
    typename Q4gType<IN>::Frag v;
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = 1.0f;
    return v;
  }
}

// One unit's products: STEPS operands of 32 numbers.
template <int IN, int STEPS>
__device__ __forceinline__ typename Q4gType<IN>::Acc products(const typename Q4gType<IN>::Frag (&w)[STEPS],
                                                              const typename Q4gType<IN>::Frag (*x)[Q4gType<IN>::PARTS]) {
  typename Q4gType<IN>::Acc acc = {0, 0, 0, 0};
  if constexpr (IN == Q4G_I8) {
    if constexpr (STEPS == 1) {
      acc = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, w[0]), __builtin_bit_cast(long, x[0][0]), acc, 0, 0, 0);
    } else {
#pragma unroll
      for (int k = 0; k < STEPS; k += 2) {
        const u32x4 a = {w[k][0], w[k][1], w[k + 1][0], w[k + 1][1]}, b = {x[k][0][0], x[k][0][1], x[k + 1][0][0], x[k + 1][0][1]};
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), acc, 0, 0, 0);
      }
    }
  } else {
    // the least parts of f32 numbers first: sums of them round far below the number's, and only STEPS
    // additions at its size
#pragma unroll
    for (int p = Q4gType<IN>::PARTS - 1; p >= 0; p--)
#pragma unroll
      for (int k = 0; k < STEPS; k++) {
        if constexpr (IN == Q4G_F16)
          acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[k], x[k][p], acc, 0, 0, 0);
        else
          acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[k], x[k][p], acc, 0, 0, 0);
      }
  }
  return acc;
}

typedef float f32x2u __attribute__((ext_vector_type(2), aligned(4)));
typedef unsigned u32x4a2 __attribute__((ext_vector_type(4), aligned(2)));  // at any 16-bit number's address

// Eight numbers of a token's row from 32 j + 8 g of a chunk on as operands.  Those behind the row's
// end are some of the row: their groups have scale 0.
template <int IN>
__device__ __forceinline__ void load_x(const Q4gArgs& a, const void* row, unsigned chunk, unsigned j, unsigned g,
                                       typename Q4gType<IN>::Frag (&x)[Q4gType<IN>::PARTS]) {
  const size_t from = (size_t)chunk * Q4G_CHUNK + 32 * j, k = (from < a.g.cols ? from : 0) + 8 * g;
  if constexpr (IN == Q4G_I8) {
    const u32x2 v = *(const u32x2*)((const int8_t*)row + k);
    // in the order of the codes' bytes: 0 4 1 5, 2 6 3 7 of a word's numbers lie at 0 1 2 3, 4 5 6 7
    x[0] = u32x2{__builtin_amdgcn_perm(v[1], v[0], 0x05010400u), __builtin_amdgcn_perm(v[1], v[0], 0x07030602u)};
  } else if constexpr (IN == Q4G_F32) {
    const float* p = (const float*)row + k;
    const f32x4 lo = *(const f32x4u*)p, hi = *(const f32x4u*)(p + 4);
    // the upper 8 bits of the mantissa, of what is left, and the rest: each a bf16, their sum
    // the number (a rest below bf16's range is lost: 2^-133)
    union {
      unsigned u[3][4];
      bf16x8 v[3];
    } r;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      unsigned part[3][2];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const float f = e < 4 ? lo[e + h] : hi[e + h - 4];
        const unsigned b0 = __float_as_uint(f) & 0xffff0000u;
        const float f1 = f - __uint_as_float(b0);
        const unsigned b1 = __float_as_uint(f1) & 0xffff0000u;
        const float f2 = f1 - __uint_as_float(b1);
        part[0][h] = b0, part[1][h] = b1, part[2][h] = __float_as_uint(f2);
      }
#pragma unroll
      for (int p3 = 0; p3 < 3; p3++) r.u[p3][e / 2] = __builtin_amdgcn_perm(part[p3][1], part[p3][0], 0x07060302u);
    }
#pragma unroll
    for (int p3 = 0; p3 < 3; p3++) x[p3] = r.v[p3];
  } else {
    x[0] = __builtin_bit_cast(typename Q4gType<IN>::Frag, (u32x4)(*(const u32x4a2*)((const uint16_t*)row + k)));
  }
}

// A chunk's M scales of a token's 8-bit codes, in one load.  Behind the row's end they are the last
// ones' (and the groups' scales are 0).
template <int M> __device__ __forceinline__ void load_x_scales(const Q4gArgs& a, const float* row, unsigned chunk, float (&s)[M]) {
  const unsigned at = a.x_per == 1 ? 0 : chunk * M;
  if constexpr (M == 1) {
    s[0] = row[at];
  } else if (at + M <= a.x_per) {
    if constexpr (M == 4) {
      const f32x4 v = *(const f32x4u*)(row + at);
      s[0] = v[0], s[1] = v[1], s[2] = v[2], s[3] = v[3];
    } else {
      const f32x2u v = *(const f32x2u*)(row + at);
      s[0] = v[0], s[1] = v[1];
    }
  } else {
#pragma unroll
    for (int m = 0; m < M; m++) s[m] = row[min(at + m, a.x_per - 1)];
  }
}

// Four scales of 16 bits.
template <bool BF> __device__ __forceinline__ f32x4 scales4(const float (&f)[2]) {
  if constexpr (BF) {
    const unsigned s[2] = {__float_as_uint(f[0]), __float_as_uint(f[1])};
    return f32x4{__uint_as_float(s[0] << 16), __uint_as_float(s[0] & 0xffff0000u), __uint_as_float(s[1] << 16),
                 __uint_as_float(s[1] & 0xffff0000u)};
  } else {
    const f16x2 a = __builtin_bit_cast(f16x2, f[0]), b = __builtin_bit_cast(f16x2, f[1]);
    return f32x4{(float)a[0], (float)a[1], (float)b[0], (float)b[1]};
  }
}

// Rows row .. row + 3 of a token's results, whose type is that of float tokens.
template <int IN> __device__ __forceinline__ void store_rows(const Q4gArgs& a, size_t token, unsigned row, f32x4 v) {
  const int type = IN == Q4G_F32 ? F32 : IN == Q4G_F16 ? F16 : IN == Q4G_BF16 ? BF16 : a.out_dtype;
  const size_t at = token * a.out_stride + row;
  const unsigned n = (unsigned)a.g.rows - row;  // (rows that pad the last tile: more than there are)
  if (row >= a.g.rows) return;
  if (type == F32) {
    float* p = (float*)a.out + at;
    if (a.out_vec && n >= 4) {
      *(f32x4*)p = v;
      return;
    }
#pragma unroll
    for (unsigned r = 0; r < 4; r++)
      if (r < n) p[r] = v[r];
    return;
  }
  union {
    uint16_t h[4];
    _Float16 f[4];
    u32x2 u;
  } h;
#pragma unroll
  for (int r = 0; r < 4; r++) {
    if (type == F16) h.f[r] = from_f32<_Float16>(v[r]);
    else h.h[r] = from_f32<Bf16>(v[r]).bits;
  }
  uint16_t* p = (uint16_t*)a.out + at;
  if (a.out_vec && n >= 4) {
    *(u32x2*)p = h.u;
    return;
  }
#pragma unroll
  for (unsigned r = 0; r < 4; r++)
    if (r < n) p[r] = h.h[r];
}

// What a lane holds of a tile's chunk: its word of codes of each operand, and of each
// group the scales and zeros of its four result rows.
template <int PER> struct Q4gChunk {
  u32x4 w;
  float s[PER][2];  // two of 16 bits each: as whole numbers the compiler takes them apart where they arrive,
  unsigned z[PER];  // which waits for loads that are meant to be ahead
  // What is computed of them is computed where they are used.
  __device__ __forceinline__ void arrive() {
#pragma unroll
    for (int u = 0; u < PER; u++) asm volatile("" : "+v"(s[u][0]), "+v"(s[u][1]), "+v"(z[u]));
  }
};

// A tile's chunks: places of a wave, and within them of a lane.  In as few loads as 16
// bytes each allow.
template <int PER> struct Q4gTile {
  const uint8_t *p, *ps, *pz;
  unsigned zstep, lw, ls, lz;
  __device__ __forceinline__ Q4gTile(const Q4gGeom& g, unsigned tile, unsigned lane)
      : p(g.data + (size_t)tile * g.tile_bytes),
        ps(p + g.scales_at),
        pz(g.zero_data + (size_t)tile * g.zero_tile),
        zstep(g.zero_chunk),
        lw(lane * 16),
        ls((lane >> 4) * 8 * PER),
        lz((lane >> 4) * 4 * PER) {}
  __device__ __forceinline__ void next(const Q4gGeom& g) {
    p += g.tile_bytes, ps += g.tile_bytes, pz += g.zero_tile;
  }
  __device__ __forceinline__ void load(unsigned chunk, Q4gChunk<PER>& c) const {
    const uint8_t *b = p + (size_t)chunk * 1024, *bs = ps + (size_t)chunk * 32 * PER, *bz = pz + (size_t)chunk * zstep;
    c.w = __builtin_nontemporal_load((const u32x4*)(b + lw));
    if constexpr (PER == 1) {
      const f32x2 v = *(const f32x2*)(bs + ls);
      c.s[0][0] = v[0], c.s[0][1] = v[1];
      c.z[0] = *(const unsigned*)(bz + lz);
    } else {
#pragma unroll
      for (int u = 0; u < PER; u += 2) {
        const f32x4 v = *(const f32x4*)(bs + ls + 8 * u);
        c.s[u][0] = v[0], c.s[u][1] = v[1], c.s[u + 1][0] = v[2], c.s[u + 1][1] = v[3];
      }
      if constexpr (PER == 2) {
        const u32x2 z = *(const u32x2*)(bz + lz);
        c.z[0] = z[0], c.z[1] = z[1];
      } else {
        const u32x4 z = *(const u32x4*)(bz + lz);
#pragma unroll
        for (int u = 0; u < 4; u++) c.z[u] = z[u];
      }
    }
  }
};

// Adds a unit's products to four rows' sums.  xs: the unit's scale of 8-bit codes.
template <int IN>
__device__ __forceinline__ f32x4 add_unit(f32x4 sum, typename Q4gType<IN>::Acc acc, typename Q4gType<IN>::Sum total, f32x4 s,
                                          unsigned z, float xs) {
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const unsigned zero = z >> (8 * e) & 255;
    if constexpr (IN == Q4G_I8)
      sum[e] = __builtin_fmaf((float)(acc[e] - __mul24((int)zero, total)), s[e] * xs, sum[e]);
    else
      sum[e] = __builtin_fmaf(__builtin_fmaf(-(float)zero, total, acc[e]), s[e], sum[e]);
  }
  return sum;
}

// ---- few tokens ----------------------------------------------------------------------

// Partial sums, written and read past the caches of one die, so that another die's
// work-group sees them without either cache being emptied (a fence there takes some 15 us).
__device__ __forceinline__ void put_part(float* p, f32x4 v) {
#pragma unroll
  for (int e = 0; e < 4; e++) __hip_atomic_store(p + e, v[e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f32x4 get_part(const float* p) {
  f32x4 v;
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = __hip_atomic_load(p + e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return v;
}

// What a wave's lanes have written to LDS, before others of them read it (they run in
// step, and LDS serves a wave in its order: nothing to wait for but the compiler).
__device__ __forceinline__ void lanes_exchange() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Tokens in LDS: a row per token and chunk of operands of eight numbers [part][16], in an
// order of the token's own that puts the same operand of 16 tokens, and 16 operands of one, into
// different banks (in their own order, with a gap between rows, two groups of lanes that LDS serves
// together met: 39 % of its cycles).
template <int IN> struct Q4gRow {
  typedef typename Q4gType<IN>::Frag Frag;
  static constexpr int P = Q4gType<IN>::PARTS;
  Frag f[16 * P];
  static __device__ __forceinline__ unsigned place(unsigned operand, unsigned token) { return operand ^ (token & 15); }
};

// A work-group of W waves computes a tile of 16 rows for 16 tokens (blockIdx.z); its waves take CH
// chunks of 128 numbers at a time, all of them on their way before the first is used,
// and join their sums in LDS, in the waves' order.  A token's numbers of a chunk are read by 16
// neighbouring lanes and change lanes through LDS (4096 x 4096, 16 tokens of 8 bits: 7.3 us, 11.0 where each
// lane read its operands itself; a launch alone 3.5).  Bound by latency: two turns of 4096 numbers.  Long rows of few tiles are divided over gridDim.y
// work-groups: the last of a tile's to finish adds their sums up in the splits' order.
// UNITS: units per chunk, within which the scales (PER of the weights, M of 8-bit codes) are the
// same.
template <int IN, int PER, int M, bool BF, int CH, int W>
__global__ __launch_bounds__(64 * W) void k_q4g_few(Q4gArgs a, unsigned per_split) {
  typedef Q4gType<IN> Ty;
  typedef typename Ty::Frag Frag;
  constexpr int UNITS = PER > M ? PER : M, STEPS = 4 / UNITS;  // operands of 32 numbers per unit
  extern __shared__ char lds[];  // [W][CH][ntok] rows; then [W][64] sums
  f32x4(*red)[64] = (f32x4(*)[64])lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned i = lane & 15, g = lane >> 4, tile = blockIdx.x, tok0 = 16 * blockIdx.z;
  const unsigned ntok = min((unsigned)a.ntok - tok0, 16u);
  const unsigned c0 = blockIdx.y * per_split, c1 = min(c0 + per_split, a.g.chunks);
  const unsigned t = min(i, ntok - 1);  // tokens that are missing are the last one
  const char* x0 = (const char*)a.x + tok0 * a.x_stride * Ty::SIZE;
  const float* xscale = IN == Q4G_I8 ? a.x_scales + (size_t)(tok0 + t) * a.x_per : nullptr;
  const Q4gTile<PER> weights(a.g, tile, lane);
  Q4gRow<IN>* rows = (Q4gRow<IN>*)lds + wave * CH * ntok;

  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  for (unsigned from = c0 + wave; from < c1; from += CH * W) {
    Frag in[CH][4][Ty::PARTS];
    float xs[CH][M];
    Q4gChunk<PER> q[CH];
#pragma unroll
    for (int k = 0; k < CH; k++)
      if (from + W * k < c1) weights.load(from + W * k, q[k]);
#pragma unroll
    for (int k = 0; k < CH; k++) {
      const unsigned c = from + W * k;
      if (c >= c1) continue;
#pragma unroll
      for (int n = 0; n < 4; n++) {  // four tokens at a time
        if (4 * n >= (int)ntok) break;
        load_x<IN>(a, x0 + min(4 * n + g, ntok - 1) * a.x_stride * Ty::SIZE, c, i / 4, i % 4, in[k][n]);
      }
      if constexpr (IN == Q4G_I8) load_x_scales<M>(a, xscale, c, xs[k]);
    }
#pragma unroll
    for (int k = 0; k < CH; k++) {
      if (from + W * k >= c1) continue;
#pragma unroll
      for (int n = 0; n < 4; n++) {
        if (4 * n >= (int)ntok) break;
        if (4 * n + g < ntok) {
#pragma unroll
          for (int p = 0; p < Ty::PARTS; p++) rows[k * ntok + 4 * n + g].f[16 * p + Q4gRow<IN>::place(i, 4 * n + g)] = in[k][n][p];
        }
      }
    }
    lanes_exchange();
#pragma unroll
    for (int k = 0; k < CH; k++) {
      if (from + W * k >= c1) continue;
      Frag x[4][Ty::PARTS];
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int p = 0; p < Ty::PARTS; p++) x[j][p] = rows[k * ntok + t].f[16 * p + Q4gRow<IN>::place(4 * j + g, t)];
      q[k].arrive();
#pragma unroll
      for (int u = 0; u < UNITS; u++) {
        Frag w[STEPS], ones[STEPS];
#pragma unroll
        for (int e = 0; e < STEPS; e++) w[e] = codes8<IN>(q[k].w[u * STEPS + e]), ones[e] = ones8<IN>();
        const typename Ty::Sum total = products<IN, STEPS>(ones, &x[u * STEPS])[0];
        sum = add_unit<IN>(sum, products<IN, STEPS>(w, &x[u * STEPS]), total, scales4<BF>(q[k].s[u * PER / UNITS]),
                           q[k].z[u * PER / UNITS], IN == Q4G_I8 ? xs[k][u * M / UNITS] : 0.0f);
      }
    }
    lanes_exchange();
  }
  __syncthreads();  // the rows are read
  red[wave][lane] = sum;
  __syncthreads();
  if (wave) return;
  f32x4 v = red[0][lane];
#pragma unroll
  for (int o = 1; o < W; o++) v = v + red[o][lane];
  if (gridDim.y > 1) {
    const size_t step = (size_t)gridDim.x * 256;
    float* part = a.g.parts + blockIdx.z * gridDim.y * step + ((size_t)tile * 64 + lane) * 4;
    unsigned* done = a.g.done + blockIdx.z * gridDim.x + tile;
    put_part(part + blockIdx.y * step, v);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the sums are where the others look before they are counted
    unsigned before = 0;
    if (lane == 0) before = atomicAdd(done, 1u);
    if (__builtin_amdgcn_readfirstlane(before) != gridDim.y - 1) return;
    v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (unsigned o = 0; o < gridDim.y; o++) v = v + get_part(part + o * step);
    if (lane == 0) *done = 0;
  }
  if (i < ntok) store_rows<IN>(a, tok0 + i, tile * Q4G_ROWS + 4 * g, v);
}

// The tokens in LDS: [chunk][token] operands [j][part][g] and then a gap that puts 16 tokens'
// equal operands into different banks, and [chunk][token][unit] sums and scales.
template <int IN, int UNITS> struct Q4gTokens {
  typedef typename Q4gType<IN>::Frag Frag;
  static constexpr unsigned ROW = 16 * Q4gType<IN>::PARTS + 1;  // operands
  static constexpr unsigned BYTES = ROW * sizeof(Frag) + 8 * UNITS;  // of a chunk and token
};

// Up to 16 tokens and many tiles.  The tokens' numbers are laid out in LDS as the operands
// lie, with their sums; then each wave streams through tiles of its own, one behind the
// other in memory, AHEAD chunks of weights on their way, and meets no other wave.  A vocabulary of
// 151936 x 2048, groups of 64 with zeros, a token of bf16, is 37.6 us: 4.5 TB/s where plain reads reach 6.25.
// The reads would take 27 us and the vector instructions (77 a chunk) 19; their loads come
// just in time, and the longest wave has 5 % more tiles than the mean.
template <int IN, int PER, int M, bool BF, int AHEAD>
__global__ __launch_bounds__(1024) void k_q4g_stream(Q4gArgs a) {
  typedef Q4gType<IN> Ty;
  typedef typename Ty::Frag Frag;
  constexpr int UNITS = PER > M ? PER : M, STEPS = 4 / UNITS, P = Ty::PARTS;
  typedef Q4gTokens<IN, UNITS> Tok;
  extern __shared__ char lds[];
  const unsigned ntok = (unsigned)a.ntok, chunks = a.g.chunks;
  Frag* xl = (Frag*)lds;
  typename Ty::Sum* totals = (typename Ty::Sum*)(xl + (size_t)chunks * ntok * Tok::ROW);
  float* xsl = (float*)(totals + chunks * ntok * UNITS);
  const unsigned lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned i = lane & 15, g = lane >> 4, tok = i < ntok ? i : ntok - 1;
  const unsigned tiles = (unsigned)((a.g.rows + Q4G_ROWS - 1) / Q4G_ROWS);
  const unsigned waves = blockDim.x / 64 * gridDim.x, me = blockIdx.x * (blockDim.x / 64) + wave;
  const unsigned first = (unsigned)((size_t)tiles * me / waves), end = (unsigned)((size_t)tiles * (me + 1) / waves);
  const unsigned n = (end - first) * chunks;  // chunks of the wave
  Q4gTile<PER> weights(a.g, first, lane);  // of the next chunk to be read
  unsigned ahead = 0, left = n;            // which chunk of its tile that is, and how many there are from it on
  Q4gChunk<PER> q[AHEAD];
  // (the last one again at the end: from a cache, without a branch around the loads)
  auto load_next = [&](Q4gChunk<PER>& to) {
    weights.load(ahead, to);
    if (left > 1) {
      left--;
      if (++ahead == chunks) ahead = 0, weights.next(a.g);
    }
  };
  if (n)
#pragma unroll
    for (int d = 0; d < AHEAD; d++) load_next(q[d]);

  const unsigned pieces = chunks * 16;
  for (unsigned k = threadIdx.x; k < pieces * ntok; k += blockDim.x) {  // along a token's row
    const unsigned part = k % pieces, t = k / pieces, c = part / 16, j = part / 4 % 4, gg = part % 4;
    Frag x[P];
    load_x<IN>(a, (const char*)a.x + t * a.x_stride * Ty::SIZE, c, j, gg, x);
#pragma unroll
    for (int p = 0; p < P; p++) xl[(c * ntok + t) * Tok::ROW + (j * P + p) * 4 + gg] = x[p];
  }
  __syncthreads();
  // f32 numbers, put together again, in 64 bits: what their sum is off by counts 16 + zero times
  for (unsigned k = threadIdx.x; k < chunks * ntok * UNITS; k += blockDim.x) {
    const unsigned u = k % UNITS, t = k / UNITS % ntok, c = k / UNITS / ntok;
    const Frag* from = xl + (c * ntok + t) * Tok::ROW + u * STEPS * P * 4;
    typename std::conditional<IN == Q4G_F32, double, typename Ty::Sum>::type sum = 0;
    for (int e = 0; e < STEPS * 4; e++) {
      const Frag* f = from + e / 4 * P * 4 + e % 4;
#pragma unroll
      for (int b = 0; b < 8; b++) {
        if constexpr (IN == Q4G_I8) sum += (int)(int8_t)(f[0][b / 4] >> (8 * (b % 4)));
        else if constexpr (IN == Q4G_F32) sum += (double)((float)f[0][b] + ((float)f[4][b] + (float)f[8][b]));
        else sum += (float)f[0][b];
      }
    }
    totals[k] = (typename Ty::Sum)sum;
    if constexpr (IN == Q4G_I8) {
      xsl[k] = a.x_scales[(size_t)t * a.x_per + (a.x_per == 1 ? 0 : min(c * M + u * M / UNITS, a.x_per - 1))];
    }
  }
  __syncthreads();

  if (n == 0) return;
  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  unsigned c = 0, tile = first;
  const Frag* px = xl + tok * Tok::ROW + g;
  unsigned pt = tok * UNITS;
  for (unsigned from = 0; from < n; from += AHEAD) {
#pragma unroll
    for (int d = 0; d < AHEAD; d++) {
      if (from + d >= n) return;
      Frag x[4][P];
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int p = 0; p < P; p++) x[j][p] = px[(j * P + p) * 4];
      q[d].arrive();
#pragma unroll
      for (int u = 0; u < UNITS; u++) {
        Frag w[STEPS];
#pragma unroll
        for (int e = 0; e < STEPS; e++) w[e] = codes8<IN>(q[d].w[u * STEPS + e]);
        sum = add_unit<IN>(sum, products<IN, STEPS>(w, &x[u * STEPS]), totals[pt + u], scales4<BF>(q[d].s[u * PER / UNITS]),
                           q[d].z[u * PER / UNITS], IN == Q4G_I8 ? xsl[pt + u] : 0.0f);
      }
      load_next(q[d]);
      px += ntok * Tok::ROW;
      pt += ntok * UNITS;
      if (++c == chunks) {
        if (i < ntok) store_rows<IN>(a, i, tile * Q4G_ROWS + 4 * g, sum);
        sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        c = 0;
        tile++;
        px = xl + tok * Tok::ROW + g;
        pt = tok * UNITS;
      }
    }
  }
}

// ---- many tokens -----------------------------------------------------------------------

template <int IN, int UNITS> struct Q4gStage {
  Q4gRow<IN> row[64];
  typename Q4gType<IN>::Sum total[UNITS][64];
  float xs[UNITS][64];
};

// A work-group computes 4 RT tiles of 16 rows for 64 tokens; its waves divide the rows, and
// (WK) the chunks of 128 numbers.  For each chunk the tokens' numbers go through LDS (wave k of
// four brings tokens 16 k .., each by 16 neighbouring lanes, and their sums); they are read
// from memory two chunks ahead, and the weights one, to registers: so two waves share a SIMD (with
// weights two ahead, one of them where groups are of 32: 512 tokens, 4096 x 4096, 69 us, 47 now).
// 512 tokens of f16, 4096 x 4096, groups of 128, take 29 us, 592 TFLOP/s; 2048 100, 688.  By the
// counters the vector units work for 43 % of the time, the matrix units for 30, and waves wait for 37: for
// 512 cycles of products of a chunk and wave there are 830 of vector instructions, laying codes out and
// scaling the groups' sums, and at its end a barrier that two waves a SIMD do not cover.  128 tokens for each reading
// of the weights leave room for one wave (120 us for 2048).
template <int IN, int PER, int M, bool BF, int RT, int WK>
__global__ __launch_bounds__(256 * WK, IN == Q4G_F32 ? 1 : 2) void k_q4g_many(Q4gArgs a, unsigned token_tiles) {
  typedef Q4gType<IN> Ty;
  typedef typename Ty::Frag Frag;
  constexpr int UNITS = PER > M ? PER : M, STEPS = 4 / UNITS, WR = 4, NT = 4, P = Ty::PARTS;
  typedef Q4gStage<IN, UNITS> Stage;
  extern __shared__ char lds[];  // [WK][2] stages; then the second half's sums
  const unsigned lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned wr = wave % WR, wk = wave / WR;
  Stage* stage = (Stage*)lds + 2 * wk;
  const unsigned i = lane & 15, g = lane >> 4;
  const unsigned tiles = (unsigned)((a.g.rows + Q4G_ROWS - 1) / Q4G_ROWS);
  // work-group b runs on die b % 8: all tokens of a row block on one, whose cache holds its weights
  const unsigned b = blockIdx.x, block = (b / 8 / token_tiles) * 8 + b % 8;
  const size_t tok0 = (size_t)(b / 8 % token_tiles) * (16 * NT);
  const unsigned tile0 = (block * WR + wr) * RT;
  if (block * WR * RT >= tiles) return;  // the whole work-group

  // the tokens that this lane brings numbers of, and one whose scales it does
  const char* row[4];
#pragma unroll
  for (int n = 0; n < 4; n++) row[n] = (const char*)a.x + min(tok0 + 16 * wr + 4 * n + g, a.ntok - 1) * a.x_stride * Ty::SIZE;
  const float* xscale = IN == Q4G_I8 ? a.x_scales + min(tok0 + 16 * wr + i, a.ntok - 1) * a.x_per : nullptr;

  struct Tokens {
    Frag x[4][P];
    float s[M];
  } in[2];
  Q4gChunk<PER> q[2][RT];
  // turn k of this half is chunk k WK + wk (the last again where there are no more)
  auto load_weights = [&](unsigned turn, Q4gChunk<PER> (&to)[RT]) {
    const unsigned c = min(turn * WK + wk, a.g.chunks - 1);
#pragma unroll
    for (int r = 0; r < RT; r++) Q4gTile<PER>(a.g, min(tile0 + r, tiles - 1), lane).load(c, to[r]);
  };
  auto load_tokens = [&](unsigned turn, Tokens& x) {
    const unsigned c = min(turn * WK + wk, a.g.chunks - 1);
#pragma unroll
    for (int n = 0; n < 4; n++) load_x<IN>(a, row[n], c, i / 4, i % 4, x.x[n]);
    if constexpr (IN == Q4G_I8) load_x_scales<M>(a, xscale, c, x.s);
  };
  auto bring = [&](Stage& s, const Tokens& x) {
#pragma unroll
    for (int n = 0; n < 4; n++)
#pragma unroll
      for (int p = 0; p < P; p++) s.row[16 * wr + 4 * n + g].f[16 * p + Q4gRow<IN>::place(i, 4 * n + g)] = x.x[n][p];
    lanes_exchange();
#pragma unroll
    for (int u = 0; u < UNITS; u++) {
      Frag ones[STEPS], mine[STEPS][P];  // of this wave's tokens, which it has just brought
#pragma unroll
      for (int e = 0; e < STEPS; e++) {
        ones[e] = ones8<IN>();
#pragma unroll
        for (int p = 0; p < P; p++) mine[e][p] = s.row[16 * wr + i].f[16 * p + Q4gRow<IN>::place(4 * (u * STEPS + e) + g, i)];
      }
      const typename Ty::Acc total = products<IN, STEPS>(ones, mine);
      if (g == 0) {
        s.total[u][16 * wr + i] = total[0];
        if constexpr (IN == Q4G_I8) s.xs[u][16 * wr + i] = x.s[u * M / UNITS];
      }
    }
  };

  f32x4 sum[RT][NT];
#pragma unroll
  for (int r = 0; r < RT; r++)
#pragma unroll
    for (int n = 0; n < NT; n++) sum[r][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  auto compute = [&](const Stage& s, Q4gChunk<PER> (&w)[RT]) {
#pragma unroll
    for (int r = 0; r < RT; r++) w[r].arrive();
#pragma unroll
    for (int u = 0; u < UNITS; u++) {
      Frag k8[RT][STEPS];
      f32x4 sc[RT];
#pragma unroll
      for (int r = 0; r < RT; r++) {
#pragma unroll
        for (int e = 0; e < STEPS; e++) k8[r][e] = codes8<IN>(w[r].w[u * STEPS + e]);
        sc[r] = scales4<BF>(w[r].s[u * PER / UNITS]);
      }
#pragma unroll
      for (int n = 0; n < NT; n++) {
        Frag x[STEPS][P];
#pragma unroll
        for (int e = 0; e < STEPS; e++)
#pragma unroll
          for (int p = 0; p < P; p++) x[e][p] = s.row[16 * n + i].f[16 * p + Q4gRow<IN>::place(4 * (u * STEPS + e) + g, i)];
        const typename Ty::Sum total = s.total[u][16 * n + i];
        const float xs = IN == Q4G_I8 ? s.xs[u][16 * n + i] : 0.0f;
#pragma unroll
        for (int r = 0; r < RT; r++) sum[r][n] = add_unit<IN>(sum[r][n], products<IN, STEPS>(k8[r], x), total, sc[r], w[r].z[u * PER / UNITS], xs);
      }
      __builtin_amdgcn_sched_barrier(0);  // the next unit's operands wait for this one's registers
    }
  };
  // the halves make as many turns; a chunk that is missing is not computed
  const unsigned turns = (a.g.chunks + WK - 1) / WK;
  load_weights(0, q[0]);
  load_tokens(0, in[0]);
  load_tokens(1, in[1]);
  bring(stage[0], in[0]);
  __syncthreads();
  for (unsigned from = 0; from < turns; from += 2) {
#pragma unroll
    for (int k = 0; k < 2; k++) {
      if (from + k >= turns) break;
      load_weights(from + k + 1, q[(k + 1) % 2]);
      load_tokens(from + k + 2, in[k]);
      __builtin_amdgcn_sched_barrier(0);  // on their way first
      if ((from + k) * WK + wk < a.g.chunks) compute(stage[k], q[k]);
      bring(stage[(k + 1) % 2], in[(k + 1) % 2]);
      __syncthreads();
    }
  }
  if constexpr (WK == 2) {  // the second half's sums to the first
    f32x4(*part)[RT][NT][64] = (f32x4(*)[RT][NT][64])lds;
    if (wk == 1) {
#pragma unroll
      for (int r = 0; r < RT; r++)
#pragma unroll
        for (int n = 0; n < NT; n++) part[wr][r][n][lane] = sum[r][n];
    }
    __syncthreads();
    if (wk == 1) return;
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
      for (int n = 0; n < NT; n++) sum[r][n] = sum[r][n] + part[wr][r][n][lane];
  }
#pragma unroll
  for (int r = 0; r < RT; r++)
#pragma unroll
    for (int n = 0; n < NT; n++) {
      const size_t token = tok0 + 16 * n + i;
      if (token < a.ntok) store_rows<IN>(a, token, (tile0 + r) * Q4G_ROWS + 4 * g, sum[r][n]);
    }
}

hipError_t launch_q4g_pack(const Q4gGeom& g, const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, hipStream_t st) {
  const unsigned tiles = (unsigned)((g.rows + Q4G_ROWS - 1) / Q4G_ROWS);
  return launch(k_q4g_pack, dim3(tiles, g.chunks < 1024 ? g.chunks : 1024), 256, 0, st, g, codes, scales, zeros);
}
hipError_t launch_q4g_unpack(const Q4gGeom& g, uint8_t* codes, uint16_t* scales, uint8_t* zeros, hipStream_t st) {
  const unsigned tiles = (unsigned)((g.rows + Q4G_ROWS - 1) / Q4G_ROWS);
  return launch(k_q4g_unpack, dim3(tiles, g.chunks < 1024 ? g.chunks : 1024), 256, 0, st, g, codes, scales, zeros);
}

constexpr uint32_t Q4G_LDS = 163840;  // of a compute unit

// More LDS than a kernel has unasked.  The limit is the process's, and calls of other contexts
// run beside: each asks for the same, all there is, whatever its own launch takes.
static hipError_t ask_lds(const void* kernel, uint32_t bytes) {
  return bytes <= 65536 ? hipSuccess : hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)Q4G_LDS);
}

template <int IN, int PER, int M, bool BF, int CH, int W>
static hipError_t q4g_few(const Q4gArgs& a, hipStream_t st) {
  const unsigned tiles = (unsigned)((a.g.rows + Q4G_ROWS - 1) / Q4G_ROWS);
  // As many work-groups as there are compute units, and twice all waves' chunks at least for each
  // of them: the join takes 1 us and 0.2 a split, as long as the chunks of two turns (1024 rows, a
  // token of bf16: of 4096 numbers 4.3 us whole, 6.0 in four; of 14336 8.4 whole, 6.9 in three).
  const unsigned slices = (unsigned)((a.ntok + 15) / 16);
  unsigned splits = q4g_splits(tiles, slices, a.g.chunks / (2 * W * CH));
  const unsigned per = (a.g.chunks + splits - 1) / splits;
  splits = (a.g.chunks + per - 1) / per;
  const uint32_t rows = W * CH * (uint32_t)(a.ntok < 16 ? a.ntok : 16) * sizeof(Q4gRow<IN>), lds = rows > W * 1024 ? rows : W * 1024;
  const hipError_t e = ask_lds((const void*)k_q4g_few<IN, PER, M, BF, CH, W>, lds);
  if (e != hipSuccess) return e;
  return launch(k_q4g_few<IN, PER, M, BF, CH, W>, dim3(tiles, splits, slices), 64 * W, lds, st, a, per);
}

template <int IN, int PER, int M, bool BF, int AHEAD>
static hipError_t q4g_stream(const Q4gArgs& a, uint32_t lds, hipStream_t st) {
  const unsigned tiles = (unsigned)((a.g.rows + Q4G_ROWS - 1) / Q4G_ROWS);
  const hipError_t e = ask_lds((const void*)k_q4g_stream<IN, PER, M, BF, AHEAD>, lds);
  if (e != hipSuccess) return e;
  // a work-group per compute unit, of so many waves that all of them have nearly as many tiles
  unsigned waves = 16, best = ~0u;
  for (unsigned w = 16; w >= 8; w--) {
    const unsigned longest = (tiles + 256 * w - 1) / (256 * w) * w;
    if (longest < best) best = longest, waves = w;
  }
  return launch(k_q4g_stream<IN, PER, M, BF, AHEAD>, 256, 64 * waves, lds, st, a);
}

template <int IN, int PER, int M, bool BF, int RT, int WK>
static hipError_t q4g_many(const Q4gArgs& a, hipStream_t st) {
  const unsigned tiles = (unsigned)((a.g.rows + Q4G_ROWS - 1) / Q4G_ROWS);
  const unsigned blocks = (tiles + 4 * RT - 1) / (4 * RT), token_tiles = (unsigned)((a.ntok + 63) / 64);
  constexpr uint32_t stage = sizeof(Q4gStage<IN, (PER > M ? PER : M)>);
  constexpr uint32_t sums = WK == 2 ? 4 * RT * 4 * 1024 : 0, lds = 2 * WK * stage > sums ? 2 * WK * stage : sums;
  static_assert(lds <= Q4G_LDS, "LDS of a compute unit");
  const hipError_t e = ask_lds((const void*)k_q4g_many<IN, PER, M, BF, RT, WK>, lds);
  if (e != hipSuccess) return e;
  const unsigned grid = (blocks + 7) / 8 * 8 * token_tiles;  // below 2^23 (2^35 results)
  return launch(k_q4g_many<IN, PER, M, BF, RT, WK>, grid, 256 * WK, lds, st, a, token_tiles);
}

// Which kernel: 4-bit rows of 4096, bf16 (f32), us:
//   rows     tokens   streaming      few            many
//   4096     1, 16                   4.3, 5.2 (5.6, 8.9)
//            32, 128                 6.9, 19 (14.8, 43)    28, 28 (76, 77)
//   14336    1, 16    14.3 (18)      9.4, 13 (19, 28)
//            32                      21 (43)               29 (76)
//   24576    1        14.9 (20.8)    15.8 (31.5)
//   151936   1, 16    60, 68 (81, 253 in slices)   87, 116 (185, 306)
// The streaming kernel gives each wave a tile or nearly so, and its tokens have to fit into LDS
// (Q4G_LDS), f32 ones in three slices at most, each with all weights: still faster than the other of
// few, whose time grows with the tokens.  Beyond 16 tokens the others work in slices of 16
// (the streaming kernel in as many launches), while that of many takes as long for 64 tokens as
// for one, and rounds of 256 work-groups: chunk by chunk a round of it is as long as some 2304 tiles
// (f32 3328) of few, and 3840 (f32 7680) of the streaming kernel.  Of 8-bit tokens with four groups or blocks to a
// chunk it is slower, the others hardly: 3840 and 4608 (groups of 32: 32768 rows of 2048, 32 tokens,
// streaming 29.8, many 35.1; 14336 rows of 4096, 64 tokens, few 57.8, many 64.7).
template <int IN, int PER, int M, bool BF>
static hipError_t q4g_sized(const Q4gArgs& a, hipStream_t st) {
  constexpr int UNITS = PER > M ? PER : M;
  constexpr bool WIDE = IN == Q4G_F32, FOUR8 = IN == Q4G_I8 && UNITS == 4;
  constexpr uint32_t BYTES = Q4gTokens<IN, UNITS>::BYTES;
  const size_t tiles = (a.g.rows + Q4G_ROWS - 1) / Q4G_ROWS, rounds = ((tiles + 7) / 8 * ((a.ntok + 63) / 64) + 255) / 256;
  size_t fit = a.g.chunks <= Q4G_LDS / BYTES ? Q4G_LDS / (a.g.chunks * BYTES) : 0;
  fit = fit > 16 ? 16 : fit;
  if (tiles >= (WIDE ? 1024 : 1536) && fit) {
    const size_t slices = (a.ntok + fit - 1) / fit;
    if (a.ntok <= 16 ? slices <= (WIDE ? 3 : 1) : slices * tiles <= (WIDE ? 7680 : FOUR8 ? 4608 : 3840) * rounds) {
      for (size_t k = 0, from = 0; k < slices; k++) {
        Q4gArgs slice = a;
        slice.ntok = (a.ntok - from) / (slices - k);
        slice.x = (const char*)a.x + from * a.x_stride * Q4gType<IN>::SIZE;
        if (IN == Q4G_I8) slice.x_scales = a.x_scales + from * a.x_per;
        slice.out = (char*)a.out + from * a.out_stride * (a.out_dtype == F32 ? 4 : 2);
        // chunks on their way: as many as registers hold
        constexpr int AHEAD = PER == 4 ? (WIDE ? 2 : 3) : UNITS == 4 || WIDE ? 4 : 6;
        const hipError_t e = q4g_stream<IN, PER, M, BF, AHEAD>(slice, a.g.chunks * BYTES * (unsigned)slice.ntok, st);
        if (e != hipSuccess) return e;
        from += slice.ntok;
      }
      return hipSuccess;
    }
  }
  const size_t slices = (a.ntok + 15) / 16;
  if (slices == 1 || (slices < 65536 && tiles * slices <= (FOUR8 ? 3840 : WIDE ? 3328 : 2304) * rounds)) {  // (a grid's third side)
    // work-groups of half as many waves, which follow each other more closely, where there are enough of them
    // (14336 rows of 4096, a token 9.4 and 10.7 us, 8192 7.2 and 6.0; f32, 16 tokens, 27.8 and 33.0, 4096 rows 11.9
    // and 8.9)
    if (tiles * slices >= (WIDE ? 384 : 640)) return q4g_few<IN, PER, M, BF, WIDE ? 1 : 2, 4>(a, st);
    return q4g_few<IN, PER, M, BF, WIDE ? 1 : 2, 8>(a, st);
  }
  // The chunks divided over two halves of a work-group where there would be few of them, f16, groups of
  // 128 (64): 512 tokens, 4096 x 4096, 29.0 us (35.4), undivided 32.8 (44.2); 2048 113 (141) and 100 (119).
  if constexpr (!WIDE) {
    if ((tiles + 7) / 8 * ((a.ntok + 63) / 64) < 512) return q4g_many<IN, PER, M, BF, 2, 2>(a, st);
  }
  return q4g_many<IN, PER, M, BF, 2, 1>(a, st);
}

template <int IN, int PER, bool BF>
static hipError_t q4g_scaled(const Q4gArgs& a, hipStream_t st) {
  if constexpr (IN == Q4G_I8) {
    if (a.x_shift == 5) return q4g_sized<IN, PER, 4, BF>(a, st);
    if (a.x_shift == 6) return q4g_sized<IN, PER, 2, BF>(a, st);
  }
  return q4g_sized<IN, PER, 1, BF>(a, st);
}

template <int IN, bool BF>
static hipError_t q4g_units(const Q4gArgs& a, hipStream_t st) {
  switch (a.g.per) {
    case 1: return q4g_scaled<IN, 1, BF>(a, st);
    case 2: return q4g_scaled<IN, 2, BF>(a, st);
    case 4: return q4g_scaled<IN, 4, BF>(a, st);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_q4g(Q4gInput in, const Q4gArgs& a, hipStream_t st) {
  if (a.ntok == 0 || a.g.rows == 0) return hipSuccess;
  switch (in) {
    case Q4G_F32: return a.g.bf16 ? q4g_units<Q4G_F32, true>(a, st) : q4g_units<Q4G_F32, false>(a, st);
    case Q4G_F16: return a.g.bf16 ? q4g_units<Q4G_F16, true>(a, st) : q4g_units<Q4G_F16, false>(a, st);
    case Q4G_BF16: return a.g.bf16 ? q4g_units<Q4G_BF16, true>(a, st) : q4g_units<Q4G_BF16, false>(a, st);
    case Q4G_I8: return a.g.bf16 ? q4g_units<Q4G_I8, true>(a, st) : q4g_units<Q4G_I8, false>(a, st);
  }
  return hipErrorInvalidValue;
}

}  // namespace hale
