// kernels_q4g.hip -- products of 4-bit weights with group scales and one to
// many tokens.
//
// out[t][r] = sum over groups of scale[r][group] (sum_k q[r][k] x[t][k] - zero[r][group]
// sum_k x[t][k]).  Within a group both sums are matrix products of whole numbers 0..15
// (and of ones) with x: of f16 and bf16 exactly, of f32 as three bf16 parts that add up
// to it, of 8-bit codes in whole numbers.  Their accumulators and the sum over
// groups are f32 (i32 within a unit of 8-bit codes).  Layout of the weights: step_ops.h.
#include <hip/hip_runtime.h>

#include "hale_device.h"
#include "kernels.h"
#include "kv_device.h"
#include "step_ops.h"

namespace hale {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// ---- laying out and back ---------------------------------------------------------

// The word of codes at `word` of a tile's chunk holds numbers k0 .. k0 + 7 of row i.
__device__ __forceinline__ void q4g_word(unsigned word, unsigned* i, unsigned* k0) {
  const unsigned lane = word / 4, j = word % 4;
  *i = lane % 16;
  *k0 = 32 * j + 8 * (lane / 16);
}

__global__ __launch_bounds__(256) void k_q4g_pack(Q4gGeom g, const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros) {
  const size_t tile = blockIdx.x;
  for (unsigned c = blockIdx.y; c < g.chunks; c += gridDim.y) {
    uint8_t* to = g.data + tile * g.tile_bytes + (size_t)c * g.chunk_bytes;
    unsigned i, k0;
    q4g_word(threadIdx.x, &i, &k0);
    const size_t row = tile * Q4G_ROWS + i, k = (size_t)c * Q4G_CHUNK + k0;
    unsigned w = 0x88888888u;
    if (row < g.rows && k < g.cols) {
      const uint8_t* p = codes + row * (g.cols / 2) + k / 2;
      w = 0;
#pragma unroll
      for (int b = 0; b < 8; b++) w |= (unsigned)(p[b / 2] >> (4 * (b % 2)) & 15) << (b < 4 ? 8 * b : 8 * (b - 4) + 4);
    }
    ((uint32_t*)to)[threadIdx.x] = w;
    if (threadIdx.x < 16 * g.per) {
      const unsigned r = threadIdx.x % 16, s = threadIdx.x / 16;
      const size_t at = tile * Q4G_ROWS + r, group = (size_t)c * g.per + s;
      const bool in = at < g.rows && group * g.group < g.cols;
      const size_t from = at * (g.cols / g.group) + group;
      ((uint16_t*)(to + 1024))[threadIdx.x] = in ? scales[from] : 0;
      if (g.zeros) (to + 1024 + 32 * g.per)[threadIdx.x] = in ? zeros[from] & 15 : 8;
    }
  }
}

__global__ __launch_bounds__(256) void k_q4g_unpack(Q4gGeom g, uint8_t* codes, uint16_t* scales, uint8_t* zeros) {
  const size_t tile = blockIdx.x;
  for (unsigned c = blockIdx.y; c < g.chunks; c += gridDim.y) {
    const uint8_t* from = g.data + tile * g.tile_bytes + (size_t)c * g.chunk_bytes;
    unsigned i, k0;
    q4g_word(threadIdx.x, &i, &k0);
    const size_t row = tile * Q4G_ROWS + i, k = (size_t)c * Q4G_CHUNK + k0;
    const unsigned w = ((const uint32_t*)from)[threadIdx.x];
    if (row < g.rows && k < g.cols) {
      uint8_t* p = codes + row * (g.cols / 2) + k / 2;
#pragma unroll
      for (int b = 0; b < 8; b += 2) {
        const unsigned lo = w >> (b < 4 ? 8 * b : 8 * (b - 4) + 4) & 15, hi = w >> (b < 4 ? 8 * b + 8 : 8 * (b - 4) + 12) & 15;
        p[b / 2] = (uint8_t)(lo | hi << 4);
      }
    }
    if (threadIdx.x < 16 * g.per) {
      const unsigned r = threadIdx.x % 16, s = threadIdx.x / 16;
      const size_t at = tile * Q4G_ROWS + r, group = (size_t)c * g.per + s;
      if (at < g.rows && group * g.group < g.cols) {
        const size_t to = at * (g.cols / g.group) + group;
        scales[to] = ((const uint16_t*)(from + 1024))[threadIdx.x];
        if (zeros) zeros[to] = g.zeros ? (from + 1024 + 32 * g.per)[threadIdx.x] : 8;
      }
    }
  }
}

// ---- operands ----------------------------------------------------------------------

// Input types: what a lane holds of eight numbers of a token, and of the weights.
template <int IN> struct Q4gType;
template <> struct Q4gType<Q4G_F16> {
  static constexpr int PARTS = 1;
  typedef f16x8 Frag;
  typedef f32x4 Acc;
};
template <> struct Q4gType<Q4G_BF16> {
  static constexpr int PARTS = 1;
  typedef bf16x8 Frag;
  typedef f32x4 Acc;
};
template <> struct Q4gType<Q4G_F32> {
  static constexpr int PARTS = 3;
  typedef bf16x8 Frag;
  typedef f32x4 Acc;
};
template <> struct Q4gType<Q4G_I8> {
  static constexpr int PARTS = 1;
  typedef u32x2 Frag;
  typedef i32x4 Acc;
};

// A word's eight codes.  A byte 0 .. 15 is the 8-bit float (4 exponent bits, 3 of
// mantissa, whose smallest numbers step by 2^-9) that stands for that many 2^-9, so
// the conversion with the scale 2^9 gives the whole number.
template <int IN> __device__ __forceinline__ typename Q4gType<IN>::Frag codes8(unsigned w) {
  const unsigned lo = w & 0x0f0f0f0fu, hi = w >> 4 & 0x0f0f0f0fu;
  if constexpr (IN == Q4G_I8) {
    return u32x2{lo, hi};
  } else if constexpr (IN == Q4G_F16) {
    union {
      f16x2 h[4];
      f16x8 v;
    } r;
    r.h[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.0f, false);
    r.h[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.0f, true);
    r.h[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.0f, false);
    r.h[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.0f, true);
    return r.v;
  } else {
    union {
      bf16x2 h[4];
      bf16x8 v;
    } r;
    r.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, false);
    r.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, true);
    r.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, false);
    r.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, true);
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
#pragma unroll
    for (int k = 0; k < STEPS; k++)
#pragma unroll
      for (int p = 0; p < Q4gType<IN>::PARTS; p++) {
        if constexpr (IN == Q4G_F16)
          acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[k], x[k][p], acc, 0, 0, 0);
        else
          acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[k], x[k][p], acc, 0, 0, 0);
      }
  }
  return acc;
}

// Eight numbers of a token's row as operands; `in`: whether the row has them.
template <int IN>
__device__ __forceinline__ void load_x(const Q4gArgs& a, const void* row, size_t k, bool in, typename Q4gType<IN>::Frag (&x)[Q4gType<IN>::PARTS]) {
  if constexpr (IN == Q4G_I8) {
    x[0] = in ? *(const u32x2*)((const int8_t*)row + k) : u32x2{0, 0};
  } else if constexpr (IN == Q4G_F32) {
    float v[8];
    const float* p = (const float*)row + k;
    if (a.vec) {
      *(u32x4*)&v[0] = in ? *(const u32x4*)p : u32x4{0, 0, 0, 0};
      *(u32x4*)&v[4] = in ? *(const u32x4*)(p + 4) : u32x4{0, 0, 0, 0};
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = in ? p[j] : 0.0f;
    }
    // the upper 8 bits of the mantissa, of what is left, and the rest: each a bf16, their sum
    // the number (a rest below bf16's range is lost: 2^-133)
    union {
      unsigned u[3][4];
      bf16x8 v[3];
    } r;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      unsigned part[3][2];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const float f = v[j + h];
        const unsigned b0 = __float_as_uint(f) & 0xffff0000u;
        const float f1 = f - __uint_as_float(b0);
        const unsigned b1 = __float_as_uint(f1) & 0xffff0000u;
        const float f2 = f1 - __uint_as_float(b1);
        part[0][h] = b0, part[1][h] = b1, part[2][h] = __float_as_uint(f2);
      }
#pragma unroll
      for (int p3 = 0; p3 < 3; p3++) r.u[p3][j / 2] = __builtin_amdgcn_perm(part[p3][1], part[p3][0], 0x07060302u);
    }
#pragma unroll
    for (int p3 = 0; p3 < 3; p3++) x[p3] = r.v[p3];
  } else {
    union {
      u32x4 u;
      uint16_t h[8];
      typename Q4gType<IN>::Frag v;
    } r;
    const uint16_t* p = (const uint16_t*)row + k;
    if (a.vec) {
      r.u = in ? *(const u32x4*)p : u32x4{0, 0, 0, 0};
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) r.h[j] = in ? p[j] : (uint16_t)0;
    }
    x[0] = r.v;
  }
}

// Four scales of 16 bits.
__device__ __forceinline__ f32x4 scales4(u32x2 s, bool bf16) {
  if (bf16)
    return f32x4{__uint_as_float(s[0] << 16), __uint_as_float(s[0] & 0xffff0000u), __uint_as_float(s[1] << 16),
                 __uint_as_float(s[1] & 0xffff0000u)};
  union {
    u32x2 u;
    _Float16 h[4];
  } r;
  r.u = s;
  return f32x4{(float)r.h[0], (float)r.h[1], (float)r.h[2], (float)r.h[3]};
}

// Rows row .. row + 3 of a token's results.
__device__ __forceinline__ void store_rows(const Q4gArgs& a, size_t token, size_t row, f32x4 v) {
  const size_t at = token * a.out_stride + row;
#pragma unroll
  for (int r = 0; r < 4; r++) {
    if (row + r >= a.g.rows) break;
    if (a.out_dtype == F32)
      ((float*)a.out)[at + r] = v[r];
    else if (a.out_dtype == F16)
      ((_Float16*)a.out)[at + r] = from_f32<_Float16>(v[r]);
    else
      ((Bf16*)a.out)[at + r] = from_f32<Bf16>(v[r]);
  }
}

// A work-group of W waves computes RT tiles of 16 rows for NT groups of 16 tokens; its
// waves take every W'th chunk of 128 numbers each and join their sums in LDS, in the waves'
// order.  UNITS: units per chunk, within which scales (of weights and of 8-bit codes) are the same.
template <int IN, int UNITS, int RT, int NT, int W>
__global__ __launch_bounds__(64 * W) void k_q4g_few(Q4gArgs a) {
  typedef Q4gType<IN> Ty;
  typedef typename Ty::Frag Frag;
  constexpr int STEPS = 4 / UNITS;  // operands of 32 numbers per unit
  __shared__ f32x4 red[W][RT][NT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned i = lane & 15, g = lane >> 4;
  const size_t tile0 = (size_t)blockIdx.x * RT, tok0 = (size_t)blockIdx.y * (16 * NT);
  const size_t tiles = (a.g.rows + Q4G_ROWS - 1) / Q4G_ROWS;
  const uint8_t* base[RT];
#pragma unroll
  for (int r = 0; r < RT; r++) base[r] = a.g.data + (tile0 + r < tiles ? tile0 + r : tiles - 1) * a.g.tile_bytes;
  const void* row[NT];
  const float* xscale[NT];
  constexpr int SIZE = IN == Q4G_I8 ? 1 : IN == Q4G_F32 ? 4 : 2;
#pragma unroll
  for (int n = 0; n < NT; n++) {  // tokens that are missing read the last one
    size_t t = tok0 + 16 * n + i;
    t = t < a.ntok ? t : a.ntok - 1;
    row[n] = (const char*)a.x + t * a.x_stride * SIZE;
    xscale[n] = IN == Q4G_I8 ? a.x_scales + t * (a.g.cols / a.x_block) : nullptr;
  }
  const unsigned xlast = IN == Q4G_I8 ? (unsigned)(a.g.cols / a.x_block) - 1 : 0;

  f32x4 sum[RT][NT];
#pragma unroll
  for (int r = 0; r < RT; r++)
#pragma unroll
    for (int n = 0; n < NT; n++) sum[r][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  for (unsigned c = wave; c < a.g.chunks; c += W) {
    u32x4 w[RT];
    u32x2 sc[RT][UNITS];
    unsigned z[RT][UNITS];
    Frag x[NT][4][Ty::PARTS];
    float xs[NT][UNITS];
#pragma unroll
    for (int r = 0; r < RT; r++) {
      const uint8_t* p = base[r] + (size_t)c * a.g.chunk_bytes;
      w[r] = *(const u32x4*)(p + lane * 16);
#pragma unroll
      for (int u = 0; u < UNITS; u++) {
        const unsigned s = u * (128 / UNITS) / a.g.group;
        sc[r][u] = *(const u32x2*)(p + 1024 + 32 * s + 8 * g);
        z[r][u] = a.g.zeros ? *(const unsigned*)(p + 1024 + 32 * a.g.per + 16 * s + 4 * g) : 0x08080808u;
      }
    }
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const size_t k = (size_t)c * Q4G_CHUNK + 32 * j + 8 * g;
        load_x<IN>(a, row[n], k, (size_t)c * Q4G_CHUNK + 32 * j < a.g.cols, x[n][j]);
      }
      if constexpr (IN == Q4G_I8) {
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
          const unsigned at = (c * Q4G_CHUNK + u * (128 / UNITS)) / a.x_block;
          xs[n][u] = xscale[n][at < xlast ? at : xlast];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < UNITS; u++) {
      Frag ones[STEPS];
      typename Ty::Acc total[NT];
#pragma unroll
      for (int k = 0; k < STEPS; k++) ones[k] = ones8<IN>();
#pragma unroll
      for (int n = 0; n < NT; n++) total[n] = products<IN, STEPS>(ones, &x[n][u * STEPS]);
#pragma unroll
      for (int r = 0; r < RT; r++) {
        Frag q[STEPS];
#pragma unroll
        for (int k = 0; k < STEPS; k++) q[k] = codes8<IN>(w[r][u * STEPS + k]);
        const f32x4 s = scales4(sc[r][u], a.g.bf16);
#pragma unroll
        for (int n = 0; n < NT; n++) {
          const typename Ty::Acc acc = products<IN, STEPS>(q, &x[n][u * STEPS]);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const unsigned zero = z[r][u] >> (8 * e) & 255;
            if constexpr (IN == Q4G_I8)
              sum[r][n][e] = __builtin_fmaf((float)(acc[e] - (int)zero * total[n][0]), s[e] * xs[n][u], sum[r][n][e]);
            else
              sum[r][n][e] = __builtin_fmaf(__builtin_fmaf(-(float)zero, total[n][0], acc[e]), s[e], sum[r][n][e]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < RT; r++)
#pragma unroll
    for (int n = 0; n < NT; n++) red[wave][r][n][lane] = sum[r][n];
  __syncthreads();
  for (int k = threadIdx.x; k < RT * NT * 64; k += 64 * W) {
    f32x4 v = ((const f32x4*)red[0])[k];
#pragma unroll
    for (int o = 1; o < W; o++) v = v + ((const f32x4*)red[o])[k];
    const int l = k % 64, n = k / 64 % NT, r = k / 64 / NT;
    const size_t token = tok0 + 16 * n + l % 16;
    if (token < a.ntok) store_rows(a, token, (tile0 + r) * Q4G_ROWS + 4 * (l / 16), v);
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

template <int IN, int UNITS>
static hipError_t q4g_sized(const Q4gArgs& a, hipStream_t st) {
  const size_t tiles = (a.g.rows + Q4G_ROWS - 1) / Q4G_ROWS;
  if (a.ntok <= 16) return launch(k_q4g_few<IN, UNITS, 1, 1, 8>, dim3((unsigned)tiles, 1), 512, 0, st, a);
  return launch(k_q4g_few<IN, UNITS, 2, 2, 4>, dim3((unsigned)((tiles + 1) / 2), (unsigned)((a.ntok + 31) / 32)), 256, 0, st, a);
}

template <int IN>
static hipError_t q4g_units(const Q4gArgs& a, hipStream_t st) {
  const unsigned unit = IN == Q4G_I8 && a.x_block < a.g.group ? a.x_block : a.g.group;
  switch (unit) {
    case 32: return q4g_sized<IN, 4>(a, st);
    case 64: return q4g_sized<IN, 2>(a, st);
    case 128: return q4g_sized<IN, 1>(a, st);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_q4g(Q4gInput in, const Q4gArgs& a, hipStream_t st) {
  if (a.ntok == 0 || a.g.rows == 0) return hipSuccess;
  switch (in) {
    case Q4G_F32: return q4g_units<Q4G_F32>(a, st);
    case Q4G_F16: return q4g_units<Q4G_F16>(a, st);
    case Q4G_BF16: return q4g_units<Q4G_BF16>(a, st);
    case Q4G_I8: return q4g_units<Q4G_I8>(a, st);
  }
  return hipErrorInvalidValue;
}

}  // namespace hale
