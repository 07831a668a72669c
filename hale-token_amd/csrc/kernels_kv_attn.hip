// kernels_kv_attn.hip -- attention over the paged 8-bit key/value cache
// (layout: kv.h), for one to many query rows per sequence.
//
// out[row] = sum_j p_j v_j / sum_j p_j, p_j = 2^(x_j - m), x_j = scale log2(e)
// q . k_j, with the running maximum m and sum of a softmax in one pass over the
// pages.  A wave takes pages of 64 positions, 16 * C query rows each:
//
//   scores  S[position][row] = K Q^T, keys the A operand, queries B;
//   values  O[d][row] = V^T P^T, values the A operand, probabilities B, which
//           leave the first product in the lane and order the second takes.
//
// Products are f16 matrix instructions with f32 sums.  Codes are whole numbers
// up to 127 and so exact in f16; their scales enter as one factor per 16
// positions, on the scores and on the probabilities (there relative to a power of
// two above the largest scale that the row has seen).  Each query row is scaled
// by a power of two to [2^13, 2^14), where f16 holds bf16 and f16 numbers
// exactly (to 2^-28 of the row's largest); an f32 row goes as two f16 numbers,
// high part and rest, good to 2^-23 of its largest, in two products.  The
// probabilities are up to 2^15 (relative to m), rounded to f16 (2^-11 of each)
// for f16 and bf16 results, or kept as two f16 parts (2^-23) for f32 results.
//
// Every row sees its own position, so its sum, relative to a score that it has seen, is 1
// at least and the division needs no guard.  The sum is 0 only where all scores are -inf (an infinite number in the query
// and codes of one sign in that dimension): 0 / 0 makes the row NaN, as any
// other score that is not finite does.
#include <hip/hip_runtime.h>

#include "hale_device.h"
#include "kernels.h"
#include "kv.h"
#include "kv_device.h"

namespace hale {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int ATT_WAVES = 4;
constexpr int P_SHIFT = 15;  // probabilities are held times 2^15

// Eight codes (two words) as f16: byte u beside 0x64 is the f16 number 1024 +
// u, from which 1024 + 128 is taken; both exact.
__device__ __forceinline__ f16x8 codes_f16(unsigned lo, unsigned hi) {
  union {
    unsigned u[4];
    f16x2 h[4];
    f16x8 v;
  } r;
  r.u[0] = __builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u);
  r.u[1] = __builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u);
  r.u[2] = __builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u);
  r.u[3] = __builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u);
  const f16x2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
#pragma unroll
  for (int i = 0; i < 4; i++) r.h[i] = r.h[i] + off;
  return r.v;
}

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// A product as the f32 that it rounds to: else the compiler may round the exact
// product to f16 in one place and the f32 in another, and the two parts of a number
// would not belong together.
__device__ __forceinline__ float rounded(float v) {
  asm("" : "+v"(v));
  return v;
}

// Over the four lanes l, l ^ 16, l ^ 32, l ^ 48 that hold one query row.
__device__ __forceinline__ float row_max(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float row_sum(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// 2^k for k up to 127; 0 below 2^-126.
__device__ __forceinline__ float pow2(int k) { return __uint_as_float((unsigned)(k < -127 ? 0 : k + 127) << 23); }

// A k for which 2^k is above v, v >= 0.  Sums of p_j v_j are kept times 2^-above(sum of p_j), which is
// exact: they are as large as values then, and finite where those are.
__device__ __forceinline__ int above(float v) { return (int)(__float_as_uint(v) >> 23) - 126; }

// v 2^k.
__device__ __forceinline__ f32x4 scaled(f32x4 v, int k) {
  return f32x4{__builtin_ldexpf(v[0], k), __builtin_ldexpf(v[1], k), __builtin_ldexpf(v[2], k), __builtin_ldexpf(v[3], k)};
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The pages first, first + step, .. below end of a page table's row, 64 of them
// held by the lanes of a wave: their places come from a register.
struct PageRow {
  const uint32_t* row;
  unsigned first, step, end;
  __device__ __forceinline__ uint32_t load(unsigned turn, int lane) const {
    const unsigned p = first + (turn + lane) * step;
    return p < end ? row[p] : 0;
  }
  static __device__ __forceinline__ uint32_t place(uint32_t places, unsigned turn) {
    return (uint32_t)__builtin_amdgcn_readlane((int)places, (int)(turn % 64));
  }
};

// The first of eight numbers of the dimension that a lane of group g holds of
// the query operand kk, in the order of the keys' layout.
__device__ __forceinline__ int query_dim(int kc, int kk, int g) {
  return kk / 2 < kc / 2 ? 64 * (kk / 2) + 16 * g + 8 * (kk & 1) : 64 * (kc / 2) + 8 * g;
}

// Four numbers to a row of the output.
__device__ __forceinline__ void store4(int dtype, void* base, size_t at, bool vec, f32x4 v) {
  if (dtype == F32) {
    float* p = (float*)base + at;
    if (vec) {
      *(f32x4*)p = v;
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) p[i] = v[i];
    }
    return;
  }
  union {
    uint16_t h[4];
    _Float16 f[4];
    u32x2 u;
  } r;
  if (dtype == F16) {
#pragma unroll
    for (int i = 0; i < 4; i++) r.f[i] = from_f32<_Float16>(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) r.h[i] = from_f32<Bf16>(v[i]).bits;
  }
  uint16_t* p = (uint16_t*)base + at;
  if (vec) {
    *(u32x2*)p = r.u;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) p[i] = r.h[i];
  }
}

// Row r of an item's queries as lane group g holds it, and the positions it
// sees: lo < position <= hi.  Rows and numbers that are missing read others.
template <typename T, int KC>
__device__ __forceinline__ void query_rows(const KvAttnArgs& a, const KvItem& item, unsigned r, int g, T (&x)[KC][8],
                                           int* hi, int* lo) {
  const bool valid = r < item.rows;
  const unsigned row = item.row0 + (valid ? r : 0), tok = row / (unsigned)a.g.group;
  *hi = valid ? (int)(item.len0 + tok) : -1;
  *lo = a.window ? (int)(item.len0 + tok) - a.window : -1;
  const T* p = (const T*)a.q + (size_t)(item.tok0 + tok) * a.q_stride +
               ((size_t)item.head * a.g.group + row % (unsigned)a.g.group) * a.g.hd;
  if (a.vec) {
#pragma unroll
    for (int kk = 0; kk < KC; kk++) {
      const int d = query_dim(KC, kk, g);
      const T* p8 = p + (d < a.g.hd ? d : 0);
#pragma unroll
      for (int j = 0; j < 8; j += 8 / (int)sizeof(T)) *(u32x2*)&x[kk][j] = *(const u32x2*)(p8 + j);
    }
  } else {
#pragma unroll
    for (int kk = 0; kk < KC; kk++) {
      const int d = query_dim(KC, kk, g);
#pragma unroll
      for (int e = 0; e < 8; e++) x[kk][e] = p[(d < a.g.hd ? d : 0) + e];
    }
  }
}

// The row as f16 operands, scaled by the power of two that takes its largest
// number to [2^13, 2^14), and what its scores are multiplied with for it.
template <typename T, int KC, int P>
__device__ __forceinline__ void split_rows(const T (&raw)[KC][8], bool valid, int hd, int g, float scale,
                                           f16x8 (&q)[P][KC], float* rs) {
  float x[KC][8], top = 0.0f;
#pragma unroll
  for (int kk = 0; kk < KC; kk++)
#pragma unroll
    for (int e = 0; e < 8; e++) {
      x[kk][e] = valid && query_dim(KC, kk, g) < hd ? to_f32(raw[kk][e]) : 0.0f;
      top = fmaxf(top, fabsf(x[kk][e]));
    }
  top = row_max(top);
  int ex = (int)(__float_as_uint(top) >> 23) - 126;
  ex = ex < -100 ? -100 : ex > 128 ? 128 : ex;
  const float up = ex > 100 ? pow2(-100) * pow2(114 - ex) : pow2(14 - ex);
  *rs = ex > 100 ? scale * pow2(100) * pow2(ex - 114) : scale * pow2(ex - 14);
#pragma unroll
  for (int kk = 0; kk < KC; kk++)
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float y = rounded(x[kk][e] * up);
      const _Float16 h = (_Float16)y;
      q[0][kk][e] = h;
      if constexpr (P == 2) q[P - 1][kk][e] = (_Float16)(y - (float)h);
    }
}

// A work-group's four waves take every fourth page each, for the same rows, and join
// their results in LDS; a sequence whose pages are many is divided over work-groups too,
// whose results the joins below put together.  The codes go from memory to registers as
// the operands lie, a page ahead of their use.  Bound by memory: each code is read
// once, for up to 32 rows.  bf16, heads of 128: 32 sequences of 200 to 8000 36.7 us for
// 145 MB (4.0 TB/s), one of 131000 30.4 us for 135 MB (4.4 TB/s; a large copy, half of
// it writes, reaches 4.85).  Read pass after pass they stay in the last-level cache of 256
// MB and take 30.3 and 25.6 us.  One of 4096 in f32 is 7.0 us for 4.3 MB, a chain of latencies: plan,
// table, page, products, the waves' join.
// T: type of queries and results; KC: padded head dimension / 32; C: groups of
// 16 query rows.
template <typename T, int KC, int C>
__global__ __launch_bounds__(64 * ATT_WAVES) void k_kv_attend_few(KvAttnArgs a) {
  constexpr int P = sizeof(T) == 4 ? 2 : 1;  // f16 parts per query number and probability
  constexpr int ND = 2 * KC;          // groups of 16 numbers of the head dimension
  constexpr int LDO = 32 * KC + 4;    // floats per row of the waves' results
  // head dimensions that share this padding: their groups of 16 from NDMIN on may be missing
  constexpr int NDMIN = KC == 2 ? 1 : KC == 3 ? 5 : KC == 4 ? 7 : KC == 6 ? 9 : 13;
  __shared__ float so[ATT_WAVES][16][LDO];
  __shared__ float2 sml[ATT_WAVES][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15, g = lane >> 4;
  const int nd = a.g.hd / 16;
  KvItem item = a.items[blockIdx.x];  // read beside the count: the plan has room for the whole grid
  const unsigned nitems = a.nitems != 0xffffffffu ? a.nitems : a.counts[a.kind];
  for (unsigned it = blockIdx.x; it < nitems; it += gridDim.x) {
    if (it != blockIdx.x) item = a.items[it];
    const uint32_t* table = a.g.table + (size_t)item.row * a.g.max_pages;
    const uint8_t* pool = a.g.pool + a.layer * a.g.layer_bytes + (size_t)item.head * a.g.head_bytes;

    // ---- the pages -------------------------------------------------------------
    u32x4 kreg[KC / 2][4];
    u32x2 khalf[4];
    u32x4 vreg[ND];
    f32x4 ks, vs;
    auto load_k = [&](const uint8_t* base) {
#pragma unroll
      for (int c = 0; c < KC / 2; c++)
#pragma unroll
        for (int mm = 0; mm < 4; mm++) kreg[c][mm] = *(const u32x4*)(base + (c * 4 + mm) * 1024 + lane * 16);
      if constexpr (KC & 1) {
#pragma unroll
        for (int mm = 0; mm < 4; mm++) khalf[mm] = *(const u32x2*)(base + KC / 2 * 4096 + mm * 512 + lane * 8);
      }
      ks = *(const f32x4*)(base + a.g.s_off);
    };
    auto load_v = [&](const uint8_t* base) {
#pragma unroll
      for (int n = 0; n < ND; n++)
        if (n < NDMIN || n < nd) vreg[n] = *(const u32x4*)(base + a.g.v_off + n * 1024 + lane * 16);
      vs = *(const f32x4*)(base + a.g.s_off + 16);
    };
    // lane j holds the place of the wave's page j of 64; a page's keys are read one
    // page ahead of their use, its values behind the use of the last ones
    const PageRow pages{table, item.page0 + wave, ATT_WAVES, item.page1};
    uint32_t places = pages.load(0, lane);
    unsigned p = item.page0 + wave, turn = 0;
    if (p < item.page1) {
      const uint8_t* base = pool + (size_t)pages.place(places, 0) * a.g.page_bytes;
      load_k(base);
      load_v(base);
    }
    // ---- the query rows ------------------------------------------------------
    // loaded whole before any is used
    T raw[C][KC][8];
    int hi[C], lo[C];  // visible: lo < position <= hi
    f16x8 q[C][P][KC];
    float rs[C];  // what a score is multiplied with, but for the keys' scale
#pragma unroll
    for (int c = 0; c < C; c++) query_rows<T, KC>(a, item, 16 * c + i, g, raw[c], &hi[c], &lo[c]);
#pragma unroll
    for (int c = 0; c < C; c++)
      split_rows<T, KC, P>(raw[c], 16 * c + i < item.rows, a.g.hd, g, a.scale, q[c], &rs[c]);
    // pages that every row sees whole: from position `first` to `last`
    const int last = (int)(item.len0 + item.row0 / (unsigned)a.g.group);
    const int first = a.window ? (int)(item.len0 + (item.row0 + item.rows - 1) / (unsigned)a.g.group) - a.window + 1 : 0;

    float m[C], l[C];
    int vk[C];  // 2^vk is above the values' scales so far, and what probabilities are relative to
    f32x4 o[C][ND];
#pragma unroll
    for (int c = 0; c < C; c++) {
      m[c] = -__builtin_inff();
      l[c] = 0.0f;
      vk[c] = -100;  // 2^(15 - vk) has to be an f32
#pragma unroll
      for (int n = 0; n < ND; n++) o[c][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    while (p < item.page1) {
      f32x4 s[C][4];
#pragma unroll
      for (int mm = 0; mm < 4; mm++) {
#pragma unroll
        for (int c = 0; c < C; c++) s[c][mm] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int kk = 0; kk < KC; kk++) {
          f16x8 k8;
          if (kk / 2 < KC / 2) {
            const u32x4 w = kreg[kk / 2][mm];
            k8 = kk & 1 ? codes_f16(w[2], w[3]) : codes_f16(w[0], w[1]);
          } else {
            k8 = codes_f16(khalf[mm][0], khalf[mm][1]);
          }
#pragma unroll
          for (int c = 0; c < C; c++)
#pragma unroll
            for (int h = 0; h < P; h++) s[c][mm] = mfma(k8, q[c][h][kk], s[c][mm]);
        }
      }
      const f32x4 ks_now = ks, vs_now = vs;
      const unsigned pn = p + ATT_WAVES;
      const uint8_t* next = nullptr;
      if (pn < item.page1) {
        if (++turn % 64 == 0) places = pages.load(turn, lane);
        next = pool + (size_t)pages.place(places, turn) * a.g.page_bytes;
        load_k(next);
      }
      const int pos0 = (int)(p * KV_PAGE);
      const bool edge = pos0 + (int)KV_PAGE - 1 > last || pos0 < first;
      f16x8 pf[C][P][2];
#pragma unroll
      for (int c = 0; c < C; c++) {
        float top = -__builtin_inff();
        f32x4 vr = vs_now;
        if (edge) {  // blocks that the row sees nothing of may hold anything
#pragma unroll
          for (int mm = 0; mm < 4; mm++)
            vr[mm] = pos0 + 16 * mm <= hi[c] && pos0 + 16 * mm + 15 > lo[c] ? vr[mm] : 0.0f;
        }
        const float vtop = fmaxf(fmaxf(vr[0], vr[1]), fmaxf(vr[2], vr[3]));
        const int k_now = above(vtop), k_new = k_now > vk[c] ? k_now : vk[c];
        const float shrink = pow2(vk[c] - k_new);
        vk[c] = k_new;
        vr = vr * pow2(P_SHIFT - k_new);
#pragma unroll
        for (int mm = 0; mm < 4; mm++) {
          const float f = rs[c] * ks_now[mm];
#pragma unroll
          for (int r = 0; r < 4; r++) {
            float x = s[c][mm][r] * f;
            if (edge) {
              const int t = pos0 + 16 * mm + 4 * g + r;
              x = t <= hi[c] && t > lo[c] ? x : -__builtin_inff();
            }
            s[c][mm][r] = x;
            top = fmaxf(top, x);
          }
        }
        top = row_max(top);
        const float mnew = fmaxf(m[c], top);
        const float base2 = mnew == -__builtin_inff() ? 0.0f : mnew;  // a row that has seen nothing yet
        const float alpha = exp2_fast(m[c] - base2);
        m[c] = mnew;
        float sum = 0.0f;
#pragma unroll
        for (int mm = 0; mm < 4; mm++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            const float e = exp2_fast(s[c][mm][r] - base2);
            sum += e;
            const float w = rounded(e * vr[mm]);
            const _Float16 h = (_Float16)w;
            pf[c][0][mm / 2][(mm & 1) * 4 + r] = h;
            if constexpr (P == 2) pf[c][1][mm / 2][(mm & 1) * 4 + r] = (_Float16)(w - (float)h);
          }
        l[c] = l[c] * alpha + sum;
        const float f = alpha * shrink;
        if (__builtin_amdgcn_ballot_w64(f != 1.0f)) {
#pragma unroll
          for (int n = 0; n < ND; n++) o[c][n] = o[c][n] * f;
        }
      }
#pragma unroll
      for (int n = 0; n < ND; n++) {
        if (n < NDMIN || n < nd) {
          const f16x8 v0 = codes_f16(vreg[n][0], vreg[n][1]), v1 = codes_f16(vreg[n][2], vreg[n][3]);
#pragma unroll
          for (int c = 0; c < C; c++)
#pragma unroll
            for (int h = 0; h < P; h++) {
              o[c][n] = mfma(v0, pf[c][h][0], o[c][n]);
              o[c][n] = mfma(v1, pf[c][h][1], o[c][n]);
            }
        }
      }
      if (next) load_v(next);
      p = pn;
    }

    // ---- the waves' results joined, 16 rows at a time --------------------------
#pragma unroll
    for (int c = 0; c < C; c++) {
      const float sum = row_sum(l[c]);
      const int scale = vk[c] - P_SHIFT - above(sum);
      __syncthreads();  // the rows before, or the item before, are read
      if (g == 0) sml[wave][i] = float2{m[c], sum};
#pragma unroll
      for (int n = 0; n < ND; n++)
        if (n < NDMIN || n < nd) *(f32x4*)&so[wave][i][16 * n + 4 * g] = scaled(o[c][n], scale);
      __syncthreads();
      const unsigned r = threadIdx.x / 16, row = 16 * c + r;
      if (row < item.rows) {
        float top = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < ATT_WAVES; w++) top = fmaxf(top, sml[w][r].x);
        const float base2 = top == -__builtin_inff() ? 0.0f : top;
        float f[ATT_WAVES], sums[ATT_WAVES], total = 0.0f;
#pragma unroll
        for (int w = 0; w < ATT_WAVES; w++) {
          f[w] = exp2_fast(sml[w][r].x - base2);
          sums[w] = sml[w][r].y;
          total += f[w] * sums[w];
        }
        const int e = above(total);
#pragma unroll
        for (int w = 0; w < ATT_WAVES; w++) f[w] = __builtin_ldexpf(f[w], above(sums[w]) - e);
        const unsigned tok = (item.row0 + row) / (unsigned)a.g.group;
        const unsigned h = item.head * a.g.group + (item.row0 + row) % (unsigned)a.g.group;
        const float inv = pow2(e) / total;
        const size_t prow = (size_t)item.part + row;
        for (int d = threadIdx.x % 16 * 4; d < a.g.hd; d += 64) {
          f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int w = 0; w < ATT_WAVES; w++) v = v + *(const f32x4*)&so[w][r][d] * f[w];
          if (item.part == KV_WHOLE)
            store4(a.dtype, a.out, (size_t)(item.tok0 + tok) * a.out_stride + (size_t)h * a.g.hd + d, a.vec, v * inv);
          else
            *(f32x4*)(a.part_o + prow * a.g.hd + d) = v;
        }
        if (item.part != KV_WHOLE && threadIdx.x % 16 == 0) a.part_ml[prow] = float2{top, total};
      }
    }
  }
}

// ---------------------------------------------------------------------------
// many rows
// ---------------------------------------------------------------------------
//
// A wave holds 16 * C rows of its own, four waves go through the pages
// together: each converts a quarter of a page's codes to f16 in LDS, as the
// operands lie, where all four read them (16 bytes per lane, one behind the
// other: no bank conflicts).  Two buffers, so one barrier a page; the next
// page's codes are read from memory while this one is computed.  Per page of 64
// positions and 16 rows at head dimension 128 the matrix instructions take 512
// cycles and the softmax about 500, so two work-groups share a compute unit, for
// one's products beside the other's softmax (f32 at dimensions 96 and 128 needs the
// registers of both for one, dimensions above 128 the LDS).  For f16 and bf16 the reference m
// follows the maximum only where this is more than 2^8 above it (probabilities are then
// up to 2^15 from 2^7), so that the sums are seldom rescaled.
// 2048 bf16 tokens behind 4000, 32 heads of 128 on 4, take 191 us for 169 GFLOP (882
// TFLOP/s, where a large matrix product reaches 1140).  By the counters, at 2.4 GHz, the vector
// units work for 102 of them and the matrix units for 67, most of that one after the
// other: scores, softmax and values are phases of a wave, which meets the other waves at a
// barrier each page.  Bound by that missing overlap.
// Waves per SIMD that the registers are divided among.  At padded dimension 192 LDS holds one
// work-group, yet half of the registers do, and the whole of them are slower (2048 behind
// 4000: bf16 477 us, 527; f32 612, 693).
constexpr int many_waves(size_t size, int kc) { return (size == 4 ? kc == 2 || kc == 6 : kc <= 6) ? 2 : 1; }

template <typename T, int KC, int C>
__global__ __launch_bounds__(256, many_waves(sizeof(T), KC)) void k_kv_attend_many(KvAttnArgs a) {
  constexpr int P = sizeof(T) == 4 ? 2 : 1, ND = 2 * KC;
  constexpr int NDMIN = KC == 2 ? 1 : KC == 3 ? 5 : KC == 4 ? 7 : KC == 6 ? 9 : 13;
  // KiB (half KiB) of a page that a wave converts: one in four of the keys', the
  // half pieces' and the values'
  constexpr int KS = KC / 2, HS = KC & 1, VS = (ND + 3) / 4;
  constexpr int SLACK = P == 1 ? 8 : 0, SHIFT = P_SHIFT - SLACK;
  extern __shared__ f16x8 lds[];       // [2][keys KC * 4 | values 2 ND][64]
  constexpr int BUF = (KC * 4 + 2 * ND) * 64;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15, g = lane >> 4, nd = a.g.hd / 16;
  const unsigned nitems = a.nitems != 0xffffffffu ? a.nitems : a.counts[a.kind];
  for (unsigned it = blockIdx.x; it < nitems; it += gridDim.x) {
    const KvItem item = a.items[it];
    const uint32_t* table = a.g.table + (size_t)item.row * a.g.max_pages;
    const uint8_t* pool = a.g.pool + a.layer * a.g.layer_bytes + (size_t)item.head * a.g.head_bytes;

    u32x4 kraw[KS], vraw[VS];
    u32x2 hraw;
    f32x4 ks, vs;
    auto fetch = [&](uint32_t page) {
      const uint8_t* base = pool + (size_t)page * a.g.page_bytes;
#pragma unroll
      for (int k = 0; k < KS; k++) kraw[k] = *(const u32x4*)(base + (4 * k + wave) * 1024 + lane * 16);
      if constexpr (HS) hraw = *(const u32x2*)(base + KS * 4096 + wave * 512 + lane * 8);
#pragma unroll
      for (int k = 0; k < VS; k++) {
        const int n = 4 * k + wave;
        vraw[k] = *(const u32x4*)(base + a.g.v_off + (n < nd ? n : 0) * 1024 + lane * 16);
      }
      ks = *(const f32x4*)(base + a.g.s_off);
      vs = *(const f32x4*)(base + a.g.s_off + 16);
    };
    auto convert = [&](f16x8* buf) {
#pragma unroll
      for (int k = 0; k < KS; k++) {  // positions 16 wave .. of operands 2 k and 2 k + 1
        f16x8* at = buf + (wave * KC + 2 * k) * 64 + lane;
        at[0] = codes_f16(kraw[k][0], kraw[k][1]);
        at[64] = codes_f16(kraw[k][2], kraw[k][3]);
      }
      if constexpr (HS) buf[(wave * KC + KC - 1) * 64 + lane] = codes_f16(hraw[0], hraw[1]);
#pragma unroll
      for (int k = 0; k < VS; k++) {
        const int n = 4 * k + wave;
        if (ND % 4 && n >= ND) continue;
        f16x8* at = buf + (KC * 4 + 2 * n) * 64 + lane;
        at[0] = codes_f16(vraw[k][0], vraw[k][1]);
        at[64] = codes_f16(vraw[k][2], vraw[k][3]);
      }
    };
    const PageRow pages{table, item.page0, 1, item.page1};
    uint32_t places = pages.load(0, lane);
    unsigned p = item.page0;
    fetch(pages.place(places, 0));

    // ---- the query rows
    int hi[C], lo[C];
    float rs[C];
    f16x8 q[C][P][KC];
    const unsigned wrow = wave * 16 * C;  // the wave's first row of the item
#pragma unroll
    for (int c = 0; c < C; c++) {
      T x8[KC][8];
      query_rows<T, KC>(a, item, wrow + 16 * c + i, g, x8, &hi[c], &lo[c]);
      split_rows<T, KC, P>(x8, wrow + 16 * c + i < item.rows, a.g.hd, g, a.scale, q[c], &rs[c]);
    }
    // positions that every row of the wave sees: from `first` to `last`; any: to `end`, from `begin`
    const unsigned group = a.g.group, wlast = wrow + 16 * C < item.rows ? wrow + 16 * C - 1 : item.rows - 1;
    const bool present = wrow < item.rows;
    const int last = (int)(item.len0 + (item.row0 + wrow) / group), end = (int)(item.len0 + (item.row0 + wlast) / group);
    const int first = a.window ? end - a.window + 1 : 0, begin = a.window ? last - a.window + 1 : 0;

    float m[C], l[C];
    int vk[C];
    f32x4 o[C][ND];
#pragma unroll
    for (int c = 0; c < C; c++) {
      m[c] = -__builtin_inff();
      l[c] = 0.0f;
      vk[c] = -100;  // 2^(15 - vk) has to be an f32
#pragma unroll
      for (int n = 0; n < ND; n++) o[c][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    convert(lds);
    __syncthreads();

    for (unsigned turn = 0; p < item.page1; p++) {
      const f16x8* buf = lds + (turn & 1) * BUF;
      f16x8* other = lds + (~turn & 1) * BUF;
      const f32x4 ks_now = ks, vs_now = vs;
      const bool more = p + 1 < item.page1;
      if (++turn % 64 == 0) places = pages.load(turn, lane);
      if (more) fetch(pages.place(places, turn));
      const int pos0 = (int)(p * KV_PAGE);
      if (present && pos0 <= end && pos0 + (int)KV_PAGE > begin) {
        // operands are read from LDS one group ahead of their products, and products
        // of one sum are several others apart
        f32x4 s[C][4];
        f16x8 kf[2][4], vf[2][2][2];
#pragma unroll
        for (int mm = 0; mm < 4; mm++) {
          kf[0][mm] = buf[mm * KC * 64 + lane];
#pragma unroll
          for (int c = 0; c < C; c++) s[c][mm] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int kk = 0; kk < KC; kk++) {
          if (kk + 1 < KC) {
#pragma unroll
            for (int mm = 0; mm < 4; mm++) kf[(kk + 1) & 1][mm] = buf[(mm * KC + kk + 1) * 64 + lane];
          }
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int h = 0; h < P; h++)
#pragma unroll
            for (int mm = 0; mm < 4; mm++)
#pragma unroll
              for (int c = 0; c < C; c++) s[c][mm] = mfma(kf[kk & 1][mm], q[c][h][kk], s[c][mm]);
          __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        auto read_v = [&](int pair) {  // groups 2 pair and 2 pair + 1 of the dimension
#pragma unroll
          for (int x = 0; x < 4; x++) vf[pair & 1][x / 2][x % 2] = buf[(KC * 4 + 4 * pair + x) * 64 + lane];
        };
        read_v(0);
        const bool edge = pos0 + (int)KV_PAGE - 1 > last || pos0 < first;
        const float vall = fmaxf(fmaxf(vs_now[0], vs_now[1]), fmaxf(vs_now[2], vs_now[3]));
        f16x8 pf[C][P][2];
#pragma unroll
        for (int c = 0; c < C; c++) {
          f32x4 vr = vs_now, f = ks_now * rs[c];
          float vtop = vall;
          if (edge) {
#pragma unroll
            for (int mm = 0; mm < 4; mm++) {
              // blocks that the row sees nothing of may hold anything
              vr[mm] = pos0 + 16 * mm <= hi[c] && pos0 + 16 * mm + 15 > lo[c] ? vr[mm] : 0.0f;
              f[mm] = fmaxf(f[mm], 0x1p-120f);  // not 0: hidden scores stay -inf
#pragma unroll
              for (int r = 0; r < 4; r++) {
                const int t = pos0 + 16 * mm + 4 * g + r;
                s[c][mm][r] = t <= hi[c] && t > lo[c] ? s[c][mm][r] : -__builtin_inff();
              }
            }
            vtop = fmaxf(fmaxf(vr[0], vr[1]), fmaxf(vr[2], vr[3]));
          }
          float top = -__builtin_inff();
#pragma unroll
          for (int mm = 0; mm < 4; mm++)
            top = fmaxf(top, f[mm] * fmaxf(fmaxf(s[c][mm][0], s[c][mm][1]), fmaxf(s[c][mm][2], s[c][mm][3])));
          top = row_max(top);
          const int k_now = above(vtop), k_new = k_now > vk[c] ? k_now : vk[c];
          const float mnew = top > m[c] + (float)SLACK ? top : m[c];
          const float ref = mnew == -__builtin_inff() ? 0.0f : mnew;
          const float alpha = exp2_fast(m[c] - ref), scale = alpha * pow2(vk[c] - k_new);
          m[c] = mnew;
          vk[c] = k_new;
          l[c] *= alpha;
          vr = vr * pow2(SHIFT - k_new);
          float sum = 0.0f;
#pragma unroll
          for (int mm = 0; mm < 4; mm++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
              const float e = exp2_fast(__builtin_fmaf(s[c][mm][r], f[mm], -ref));
              sum += e;
              if constexpr (P == 1) {
                pf[c][0][mm / 2][(mm & 1) * 4 + r] = (_Float16)(e * vr[mm]);
              } else {
                const float w = rounded(e * vr[mm]);
                const _Float16 h = (_Float16)w;
                pf[c][0][mm / 2][(mm & 1) * 4 + r] = h;
                pf[c][P - 1][mm / 2][(mm & 1) * 4 + r] = (_Float16)(w - (float)h);
              }
            }
          l[c] += sum;
          if (__builtin_amdgcn_ballot_w64(scale != 1.0f)) {
#pragma unroll
            for (int n = 0; n < ND; n++) o[c][n] = o[c][n] * scale;
          }
        }
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int pair = 0; pair < ND / 2; pair++) {
          if (pair + 1 < ND / 2) read_v(pair + 1);
          __builtin_amdgcn_sched_barrier(0);
          // (a last group that the head dimension has not takes what lies in its place, and is not stored)
#pragma unroll
          for (int h = 0; h < P; h++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
              for (int x = 0; x < 2; x++)
#pragma unroll
                for (int c = 0; c < C; c++) o[c][2 * pair + x] = mfma(vf[pair & 1][x][j], pf[c][h][j], o[c][2 * pair + x]);
          __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
      }
      if (more) convert(other);
      __syncthreads();
    }

#pragma unroll
    for (int c = 0; c < C; c++) {
      const unsigned r = wrow + 16 * c + i;
      const float total = row_sum(l[c]), up = pow2(vk[c] - SHIFT), down = pow2(-above(total));
      if (r >= item.rows) continue;
      const unsigned tok = (item.row0 + r) / group, h = item.head * group + (item.row0 + r) % group;
      const float inv = up / total;
#pragma unroll
      for (int n = 0; n < ND; n++)
        if (n < NDMIN || n < nd) {
          const int d = 16 * n + 4 * g;
          if (item.part == KV_WHOLE)
            store4(a.dtype, a.out, (size_t)(item.tok0 + tok) * a.out_stride + (size_t)h * a.g.hd + d, a.vec, o[c][n] * inv);
          else
            *(f32x4*)(a.part_o + ((size_t)item.part + r) * a.g.hd + d) = o[c][n] * down * up;
        }
      if (item.part != KV_WHOLE && g == 0) a.part_ml[(size_t)item.part + r] = float2{m[c], total};
    }
  }
}

// Parts of one row: all of a step's at most.
constexpr unsigned JOIN_PARTS = 2 * (KV_FEW_GROUPS > KV_MANY_GROUPS ? KV_FEW_GROUPS : KV_MANY_GROUPS);
constexpr int JOIN_BITS = 10;
static_assert(JOIN_PARTS <= 1u << JOIN_BITS, "the sum of a row's parts");

// The joins of a launch and their one series: of steps apart, or of those that may share and do not
// (a.kind 2).
template <typename Join> __device__ __forceinline__ Join join_of(const KvAttnArgs& a, unsigned it) {
  if constexpr (__is_same(Join, KvJoin)) return a.joins[it];
  else return a.share_joins[it];
}
__device__ __forceinline__ KvSeries series_of(const KvJoin& j) { return {j.part0, j.parts, j.step}; }
__device__ __forceinline__ KvSeries series_of(const KvShareJoin& j) { return j.of[0]; }
template <typename Join> __device__ __forceinline__ unsigned joins_of(const KvAttnArgs& a) {
  return a.njoins != 0xffffffffu ? a.njoins : a.counts[__is_same(Join, KvJoin) ? a.kind + 2 : 2];
}

// Joins of few parts, or of many rows: a work-group takes as many rows as its
// threads hold at four numbers each, the parts one behind the other.  A chain of three
// reads: 5.1 us for 32 sequences of up to 7 parts, 4 rows of 128 each.
template <typename Join>
__global__ __launch_bounds__(256) void k_kv_join_rows(KvAttnArgs a) {
  const int t = threadIdx.x;
  const int quads = a.g.hd / 4, lanes = quads <= 16 ? 16 : quads <= 32 ? 32 : 64, x = t % lanes;
  const unsigned njoins = joins_of<Join>(a);
  for (unsigned it = blockIdx.x; it < njoins; it += gridDim.x) {
    const Join join = join_of<Join>(a, it);
    const KvSeries of = series_of(join);
    const unsigned row = blockIdx.y * (256 / lanes) + t / lanes;
    if (row >= join.rows || x >= quads) continue;
    const float2* ml = a.part_ml + (size_t)of.part0 + row;
    const float* po = a.part_o + ((size_t)of.part0 + row) * a.g.hd + 4 * x;
    const size_t step = (size_t)of.step * a.g.hd;
    float top = -__builtin_inff(), most = 0.0f, total = 0.0f;
#pragma unroll 4
    for (unsigned k = 0; k < of.parts; k++) {
      const float2 part = ml[(size_t)k * of.step];
      top = fmaxf(top, part.x);
      most = fmaxf(most, part.y);
    }
    const int e = above(most) + JOIN_BITS;  // 2^e is above the row's sum
    const float base2 = top == -__builtin_inff() ? 0.0f : top;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (unsigned k = 0; k < of.parts; k++) {
      const float2 part = ml[(size_t)k * of.step];
      const float w = exp2_fast(part.x - base2);
      total += w * part.y;
      v = v + *(const f32x4*)(po + k * step) * (w * pow2(above(part.y) - e));
    }
    const unsigned tok = (join.row0 + row) / (unsigned)a.g.group;
    const unsigned h = join.head * a.g.group + (join.row0 + row) % (unsigned)a.g.group;
    const float inv = pow2(e) / total;
    store4(a.dtype, a.out, (size_t)(join.tok0 + tok) * a.out_stride + (size_t)h * a.g.hd + 4 * x, a.vec, v * inv);
  }
}

// Joins the partial results of one row: a work-group, whose threads take four
// numbers each of every so many'th part; the slices are added in their order.  16 parts
// a slice are read while the weights are found.  5.5 us for 128 parts of 32 rows of 128.
template <typename Join>
__global__ __launch_bounds__(256) void k_kv_join(KvAttnArgs a) {
  constexpr int AHEAD = 16;
  __shared__ float sw[JOIN_PARTS];
  __shared__ float red[8];
  __shared__ f32x4 sv[256];
  const int t = threadIdx.x, wave = t >> 6;
  const int quads = a.g.hd / 4, lanes = quads <= 16 ? 16 : quads <= 32 ? 32 : 64, slices = 256 / lanes;
  const int x = t % lanes, slice = t / lanes;
  const unsigned njoins = joins_of<Join>(a);
  for (unsigned it = blockIdx.x; it < njoins; it += gridDim.x) {
    const Join join = join_of<Join>(a, it);
    const KvSeries of = series_of(join);
    const unsigned row = blockIdx.y;
    if (row >= join.rows) continue;
    const float2* ml = a.part_ml + (size_t)of.part0 + row;
    const float* po = a.part_o + ((size_t)of.part0 + row) * a.g.hd + 4 * x;
    const size_t step = (size_t)of.step * a.g.hd;
    f32x4 early[AHEAD];  // the first parts, on their way while the weights are found
    if (x < quads) {
#pragma unroll
      for (int k = 0; k < AHEAD; k++) {
        const unsigned part = slice + slices * k;
        early[k] = *(const f32x4*)(po + (part < of.parts ? part : 0) * step);
      }
    }
    float2 mine[JOIN_PARTS / 256];
    float top = -__builtin_inff(), total = 0.0f;
#pragma unroll
    for (int k = 0; k < (int)JOIN_PARTS / 256; k++) {
      const unsigned part = t + 256 * k;
      mine[k] = part < of.parts ? ml[(size_t)part * of.step] : float2{-__builtin_inff(), 0.0f};
      top = fmaxf(top, mine[k].x);
    }
    top = wave_max_f32(top);
    __syncthreads();  // the row before is read
    if (t % 64 == 0) red[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float base2 = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
    for (int k = 0; k < (int)JOIN_PARTS / 256; k++) {
      const unsigned part = t + 256 * k;
      const float w = exp2_fast(mine[k].x - base2);
      if (part < of.parts) sw[part] = w * pow2(above(mine[k].y));
      total += w * mine[k].y;
    }
#pragma unroll
    for (int o = 32; o; o /= 2) total += __shfl_xor(total, o);
    if (t % 64 == 0) red[4 + wave] = total;
    __syncthreads();
    total = (red[4] + red[5]) + (red[6] + red[7]);
    const int e = above(total);
    const float down = pow2(-e);
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (x < quads) {
#pragma unroll
      for (int k = 0; k < AHEAD; k++) {
        const unsigned part = slice + slices * k;
        if (part < of.parts) v = v + early[k] * (sw[part] * down);
      }
#pragma unroll 8
      for (unsigned k = slice + slices * AHEAD; k < of.parts; k += slices) v = v + *(const f32x4*)(po + k * step) * (sw[k] * down);
    }
    sv[t] = v;
    __syncthreads();
    if (slice == 0 && x < quads) {
      for (int k = 1; k < slices; k++) v = v + sv[x + lanes * k];
      const unsigned tok = (join.row0 + row) / (unsigned)a.g.group;
      const unsigned h = join.head * a.g.group + (join.row0 + row) % (unsigned)a.g.group;
      const float inv = pow2(e) / total;
      store4(a.dtype, a.out, (size_t)(join.tok0 + tok) * a.out_stride + (size_t)h * a.g.hd + 4 * x, a.vec, v * inv);
    }
  }
}

// Joins a row's partial results over its own pages with those over shared ones: SLICES
// groups of threads take every so many'th part of the series laid end to end, four numbers of
// the head dimension a thread, and put theirs together in LDS in the slices' order.  A chain of
// three reads: 4.7 us for 32 sequences, 32 heads of 128, four shared parts and one or two of their own
// (a launch alone 3.5).  Of many parts the places, maxima and sums are brought to LDS by all of a row's threads
// first, which changes no result: 2 sequences behind 11000, 2 heads of 128, f16, 45 parts, with the attention 12.9
// us, 13.8 where each slice looks for its own.  (A work-group a row, as in k_kv_join, or eight parts at a
// time take 100 registers for 70: 11.2, but 32 sequences of 40 rows behind 4000 40.9 for 37.5.)
constexpr int SHARE_SLICES = 4;
constexpr unsigned SHARE_WIDE = 16, SHARE_STAGED = 256;  // many: more than the first, up to the second
static_assert(KV_SHARE_PARTS <= 1u << JOIN_BITS, "the sum of a row's parts");

__global__ __launch_bounds__(256) void k_kv_join_shared(KvAttnArgs a) {
  constexpr int S = SHARE_SLICES;
  constexpr int PER = 256 / 16 / S;  // rows at most
  __shared__ f32x4 sv[256];
  __shared__ float2 sml[256];
  __shared__ unsigned at_part[PER][SHARE_STAGED];
  __shared__ float2 ml_part[PER][SHARE_STAGED];
  const int t = threadIdx.x;
  const int quads = a.g.hd / 4, lanes = quads <= 16 ? 16 : quads <= 32 ? 32 : 64, x = t % lanes;
  const int slice = t / lanes % S, per = 256 / lanes / S;
  const unsigned njoins = a.njoins != 0xffffffffu ? a.njoins : a.counts[2];
  for (unsigned it = blockIdx.x; it < njoins; it += gridDim.x) {
    const KvShareJoin join = a.share_joins[it];
    const unsigned row = blockIdx.y * per + t / lanes / S;
    const bool mine = row < join.rows && x < quads;
    unsigned parts = 0;
#pragma unroll
    for (int s = 0; s <= KV_SHARE_LEVELS; s++) parts += s < (int)join.n ? join.of[s].parts : 0;
    float top = -__builtin_inff(), most = 0.0f, total = 0.0f;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    int e = 0;
    // the slice's parts, each by its place and its maximum and sum
    auto slice_of = [&](auto&& each) {
      each([&](size_t, float2 part) {
        top = fmaxf(top, part.x);
        most = fmaxf(most, part.y);
      });
      e = above(most) + JOIN_BITS;  // 2^e is above the sum
      const float base2 = top == -__builtin_inff() ? 0.0f : top;
      each([&](size_t at, float2 part) {
        const float w = exp2_fast(part.x - base2);
        total += w * part.y;
        v = v + *(const f32x4*)(a.part_o + at * a.g.hd + 4 * x) * (w * pow2(above(part.y) - e));
      });
      // as large as values, times 2^-above(total)
      v = scaled(v, e - above(total));
    };
    if (parts > SHARE_WIDE && parts <= SHARE_STAGED) {
      const int here = t / lanes / S, threads = lanes * S;
      if (row < join.rows) {
        for (unsigned k = t % threads; k < parts; k += threads) {
          unsigned from = k, at = 0;
#pragma unroll
          for (int s = 0; s <= KV_SHARE_LEVELS; s++) {
            const KvSeries& r = join.of[s];
            const bool in = s < (int)join.n && from < r.parts;
            if (in) at = r.part0 + row + from * r.step;
            from = in || s >= (int)join.n ? 0xffffffffu : from - r.parts;
          }
          at_part[here][k] = at;
          ml_part[here][k] = a.part_ml[at];
        }
      }
      __syncthreads();
      if (mine)
        slice_of([&](auto&& f) {
#pragma unroll 4
          for (unsigned k = slice; k < parts; k += S) f((size_t)at_part[here][k], ml_part[here][k]);
        });
    } else if (mine) {
      slice_of([&](auto&& f) {
        unsigned from = slice;
#pragma unroll
        for (int s = 0; s <= KV_SHARE_LEVELS; s++) {
          if (s >= (int)join.n) break;
          const KvSeries& r = join.of[s];
#pragma unroll 4
          for (; from < r.parts; from += S) {
            const size_t at = (size_t)r.part0 + row + (size_t)from * r.step;
            f(at, a.part_ml[at]);
          }
          from -= r.parts;
        }
      });
    }
    __syncthreads();  // the join before is read
    sv[t] = v;
    sml[t] = float2{top, total};
    __syncthreads();
    if (!mine || slice) continue;
    float f[S], sums[S];
    top = -__builtin_inff();
    total = 0.0f;
#pragma unroll
    for (int k = 0; k < S; k++) top = fmaxf(top, sml[t + k * lanes].x);
    const float base2 = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
    for (int k = 0; k < S; k++) {
      f[k] = exp2_fast(sml[t + k * lanes].x - base2);
      sums[k] = sml[t + k * lanes].y;
      total += f[k] * sums[k];
    }
    e = above(total);
    v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < S; k++) v = v + sv[t + k * lanes] * __builtin_ldexpf(f[k], above(sums[k]) - e);
    const unsigned tok = (join.row0 + row) / (unsigned)a.g.group;
    const unsigned h = join.head * a.g.group + (join.row0 + row) % (unsigned)a.g.group;
    store4(a.dtype, a.out, (size_t)(join.tok0 + tok) * a.out_stride + (size_t)h * a.g.hd + 4 * x, a.vec, v * (pow2(e) / total));
  }
}

template <typename T, int KC>
static hipError_t few_sized(const KvAttnArgs& a, int cols, unsigned grid, hipStream_t st) {
  if (cols == 1) return launch(k_kv_attend_few<T, KC, 1>, grid, 64 * ATT_WAVES, 0, st, a);
  if constexpr (KC <= 4) {
    if (cols == 2) return launch(k_kv_attend_few<T, KC, 2>, grid, 64 * ATT_WAVES, 0, st, a);
  }
  return hipErrorInvalidValue;
}

template <typename T, int KC>
static hipError_t many_sized(const KvAttnArgs& a, unsigned grid, hipStream_t st) {
  constexpr int C = KC <= 4 ? 2 : 1;
  const uint32_t lds = 2 * (KC * 4 + 4 * KC) * 64 * 16;
  static_assert(C * 64 == (KC <= 4 ? 128 : 64), "kv_many_rows");
  if (lds > 65536) {  // more than a kernel has unasked
    const hipError_t e = hipFuncSetAttribute((const void*)k_kv_attend_many<T, KC, C>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  return launch(k_kv_attend_many<T, KC, C>, grid, 256, lds, st, a);
}

#define HALE_KV_SIZED(fn, T, ...)              \
  switch (a.g.chunks) {                        \
    case 2: return fn<T, 2>(a, __VA_ARGS__);   \
    case 3: return fn<T, 3>(a, __VA_ARGS__);   \
    case 4: return fn<T, 4>(a, __VA_ARGS__);   \
    case 6: return fn<T, 6>(a, __VA_ARGS__);   \
    case 8: return fn<T, 8>(a, __VA_ARGS__);   \
    default: return hipErrorInvalidValue;      \
  }

hipError_t launch_kv_attend_few(const KvAttnArgs& a, int cols, unsigned grid, hipStream_t st) {
  if (grid == 0) return hipSuccess;
  if (a.dtype == F32) HALE_KV_SIZED(few_sized, float, cols, grid, st)
  if (a.dtype == F16) HALE_KV_SIZED(few_sized, _Float16, cols, grid, st)
  HALE_KV_SIZED(few_sized, Bf16, cols, grid, st)
}

hipError_t launch_kv_attend_many(const KvAttnArgs& a, unsigned grid, hipStream_t st) {
  if (grid == 0) return hipSuccess;
  if (a.dtype == F32) HALE_KV_SIZED(many_sized, float, grid, st)
  if (a.dtype == F16) HALE_KV_SIZED(many_sized, _Float16, grid, st)
  HALE_KV_SIZED(many_sized, Bf16, grid, st)
}

hipError_t launch_kv_join(const KvAttnArgs& a, unsigned grid, unsigned rows, unsigned parts, hipStream_t st) {
  if (grid == 0) return hipSuccess;
  if (a.kind == 2 && !a.alone) {
    const unsigned lanes = a.g.hd <= 64 ? 16 : a.g.hd <= 128 ? 32 : 64, per = 256 / lanes / SHARE_SLICES;
    return launch(k_kv_join_shared, dim3(grid, (rows + per - 1) / per), 256, 0, st, a);
  }
  // (with the attention, by row / rows together: 16 sequences of 1000, 4 parts 13.3 / 11.9 us;
  // of 6000, 8 parts 25.1 / 24.1; 4 of 3000, 12 parts 11.5 / 11.7; one of 131000, 512 parts
  // 31.1 / 54.5.  Many rows are the more work-groups: 300 behind 8000 102 / 68.)
  if (a.kind != 1 && rows <= kv_few_rows(a.g.hd) && parts > 8)
    return launch(a.alone ? k_kv_join<KvShareJoin> : k_kv_join<KvJoin>, dim3(grid, rows), 256, 0, st, a);
  const unsigned per = a.g.hd <= 64 ? 16 : a.g.hd <= 128 ? 8 : 4;
  return launch(a.alone ? k_kv_join_rows<KvShareJoin> : k_kv_join_rows<KvJoin>, dim3(grid, (rows + per - 1) / per), 256, 0, st, a);
}

}  // namespace hale
