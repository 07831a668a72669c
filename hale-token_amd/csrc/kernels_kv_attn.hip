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
#include <hip/hip_runtime.h>

#include "hale_device.h"
#include "kernels.h"
#include "kv.h"
#include "kv_device.h"

namespace hale {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int ATT_WAVES = 4;
constexpr float P_SHIFT = 15.0f;  // probabilities are held times 2^15

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

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

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

// T: type of queries and results; KC: padded head dimension / 32; C: groups of
// 16 query rows.
template <typename T, int KC, int C>
__global__ __launch_bounds__(64 * ATT_WAVES) void k_kv_attend(KvAttnArgs a) {
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
  const unsigned nitems = a.nitems != 0xffffffffu ? a.nitems : a.counts[0];
  for (unsigned it = blockIdx.x; it < nitems; it += gridDim.x) {
    const KvItem item = a.items[it];
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
    // a page's place is read one page ahead of its keys, these one page ahead of
    // their use, its values behind the use of the last ones
    unsigned p = item.page0 + wave;
    uint32_t ahead = 0;
    if (p < item.page1) {
      const uint8_t* base = pool + (size_t)table[p] * a.g.page_bytes;
      if (p + ATT_WAVES < item.page1) ahead = table[p + ATT_WAVES];
      load_k(base);
      load_v(base);
    }
    // ---- the query rows ------------------------------------------------------
    // loaded whole before any is used; rows and numbers that are missing read others
    T raw[C][KC][8];
    int hi[C], lo[C];  // visible: lo < position <= hi
#pragma unroll
    for (int c = 0; c < C; c++) {
      const unsigned r = 16 * c + i;
      const bool valid = r < item.rows;
      const unsigned row = item.row0 + (valid ? r : 0), tok = row / (unsigned)a.g.group;
      hi[c] = valid ? (int)(item.len0 + tok) : -1;
      lo[c] = a.window ? (int)(item.len0 + tok) - a.window : -1;
      const T* x = (const T*)a.q + (size_t)(item.tok0 + tok) * a.q_stride +
                   ((size_t)item.head * a.g.group + row % (unsigned)a.g.group) * a.g.hd;
      if (a.vec) {
#pragma unroll
        for (int kk = 0; kk < KC; kk++) {
          const int d = query_dim(KC, kk, g);
          const T* p8 = x + (d < a.g.hd ? d : 0);
          *(u32x2*)&raw[c][kk][0] = *(const u32x2*)p8;
          *(u32x2*)&raw[c][kk][8 / sizeof(T)] = *(const u32x2*)(p8 + 8 / sizeof(T));
          if constexpr (sizeof(T) == 4) {
            *(u32x2*)&raw[c][kk][4] = *(const u32x2*)(p8 + 4);
            *(u32x2*)&raw[c][kk][6] = *(const u32x2*)(p8 + 6);
          }
        }
      } else {
#pragma unroll
        for (int kk = 0; kk < KC; kk++) {
          const int d = query_dim(KC, kk, g);
#pragma unroll
          for (int e = 0; e < 8; e++) raw[c][kk][e] = x[(d < a.g.hd ? d : 0) + e];
        }
      }
    }
    f16x8 q[C][P][KC];
    float rs[C];  // what a score is multiplied with, but for the keys' scale
#pragma unroll
    for (int c = 0; c < C; c++) {
      float x[KC][8], top = 0.0f;
#pragma unroll
      for (int kk = 0; kk < KC; kk++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
          x[kk][e] = 16 * c + i < item.rows && query_dim(KC, kk, g) < a.g.hd ? to_f32(raw[c][kk][e]) : 0.0f;
          top = fmaxf(top, fabsf(x[kk][e]));
        }
      top = row_max(top);
      // the power of two that takes the row's largest to [2^13, 2^14)
      int ex = (int)(__float_as_uint(top) >> 23) - 126;
      ex = ex < -100 ? -100 : ex > 128 ? 128 : ex;
      const float up = ex > 100 ? pow2(-100) * pow2(114 - ex) : pow2(14 - ex);
      rs[c] = ex > 100 ? a.scale * pow2(100) * pow2(ex - 114) : a.scale * pow2(ex - 14);
#pragma unroll
      for (int kk = 0; kk < KC; kk++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float y = x[kk][e] * up;
          const _Float16 h = (_Float16)y;
          q[c][0][kk][e] = h;
          if constexpr (P == 2) q[c][1][kk][e] = (_Float16)(y - (float)h);
        }
    }
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
      vk[c] = -126;
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
        next = pool + (size_t)ahead * a.g.page_bytes;
        if (pn + ATT_WAVES < item.page1) ahead = table[pn + ATT_WAVES];
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
        const int k_now = (int)(__float_as_uint(vtop) >> 23) - 126, k_new = k_now > vk[c] ? k_now : vk[c];
        const float shrink = pow2(vk[c] - k_new);
        vk[c] = k_new;
        vr = vr * pow2(-k_new);
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
            const float e = exp2_fast(s[c][mm][r] - base2 + P_SHIFT);
            sum += e;
            const float w = e * vr[mm];
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
      __syncthreads();  // the rows before, or the item before, are read
      if (g == 0) sml[wave][i] = float2{m[c], sum};
#pragma unroll
      for (int n = 0; n < ND; n++)
        if (n < NDMIN || n < nd) *(f32x4*)&so[wave][i][16 * n + 4 * g] = o[c][n] * pow2(vk[c]);
      __syncthreads();
      const unsigned r = threadIdx.x / 16, row = 16 * c + r;
      if (row < item.rows) {
        float top = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < ATT_WAVES; w++) top = fmaxf(top, sml[w][r].x);
        const float base2 = top == -__builtin_inff() ? 0.0f : top;
        float f[ATT_WAVES], total = 0.0f;
#pragma unroll
        for (int w = 0; w < ATT_WAVES; w++) {
          f[w] = exp2_fast(sml[w][r].x - base2);
          total += f[w] * sml[w][r].y;
        }
        const unsigned tok = (item.row0 + row) / (unsigned)a.g.group;
        const unsigned h = item.head * a.g.group + (item.row0 + row) % (unsigned)a.g.group;
        const float inv = total > 0.0f ? 1.0f / total : 0.0f;  // nothing visible: zeros
        const size_t prow = (size_t)item.part * (16 * C) + row;
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

// Joins the partial results of one row: a work-group, whose threads take four
// numbers each of every so many'th part; the slices are added in their order.
__global__ __launch_bounds__(256) void k_kv_join(KvAttnArgs a, int rows_per_part) {
  __shared__ float sw[KV_MAX_PARTS];
  __shared__ float red[8];
  __shared__ f32x4 sv[256];
  const int t = threadIdx.x, wave = t >> 6;
  const int quads = a.g.hd / 4, lanes = quads <= 16 ? 16 : quads <= 32 ? 32 : 64, slices = 256 / lanes;
  const int x = t % lanes, slice = t / lanes;
  const unsigned njoins = a.njoins != 0xffffffffu ? a.njoins : a.counts[1];
  for (unsigned it = blockIdx.x; it < njoins; it += gridDim.x) {
    const KvJoin join = a.joins[it];
    const unsigned row = blockIdx.y;
    if (row >= join.rows) continue;
    const float2* ml = a.part_ml + (size_t)join.part0 * rows_per_part + row;
    const float* po = a.part_o + ((size_t)join.part0 * rows_per_part + row) * a.g.hd + 4 * x;
    const size_t step = (size_t)rows_per_part * a.g.hd;
    float2 mine[KV_MAX_PARTS / 256];
    float top = -__builtin_inff(), total = 0.0f;
#pragma unroll
    for (int k = 0; k < (int)KV_MAX_PARTS / 256; k++) {
      const unsigned part = t + 256 * k;
      mine[k] = part < join.parts ? ml[(size_t)part * rows_per_part] : float2{-__builtin_inff(), 0.0f};
      top = fmaxf(top, mine[k].x);
    }
    top = wave_max_f32(top);
    __syncthreads();  // the row before is read
    if (t % 64 == 0) red[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float base2 = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
    for (int k = 0; k < (int)KV_MAX_PARTS / 256; k++) {
      const unsigned part = t + 256 * k;
      const float w = exp2_fast(mine[k].x - base2);
      if (part < join.parts) sw[part] = w;
      total += w * mine[k].y;
    }
#pragma unroll
    for (int o = 32; o; o /= 2) total += __shfl_xor(total, o);
    if (t % 64 == 0) red[4 + wave] = total;
    __syncthreads();
    total = (red[4] + red[5]) + (red[6] + red[7]);
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (x < quads) {
#pragma unroll 4
      for (unsigned k = slice; k < join.parts; k += slices) v = v + *(const f32x4*)(po + k * step) * sw[k];
    }
    sv[t] = v;
    __syncthreads();
    if (slice == 0 && x < quads) {
      for (int k = 1; k < slices; k++) v = v + sv[x + lanes * k];
      const unsigned tok = (join.row0 + row) / (unsigned)a.g.group;
      const unsigned h = join.head * a.g.group + (join.row0 + row) % (unsigned)a.g.group;
      const float inv = total > 0.0f ? 1.0f / total : 0.0f;
      store4(a.dtype, a.out, (size_t)(join.tok0 + tok) * a.out_stride + (size_t)h * a.g.hd + 4 * x, a.vec, v * inv);
    }
  }
}

template <typename T, int KC>
static hipError_t attend_cols(const KvAttnArgs& a, int cols, unsigned grid, hipStream_t st) {
  if (cols == 1) return launch(k_kv_attend<T, KC, 1>, grid, 64 * ATT_WAVES, 0, st, a);
  if constexpr (KC <= 4) {
    if (cols == 2) return launch(k_kv_attend<T, KC, 2>, grid, 64 * ATT_WAVES, 0, st, a);
  }
  return hipErrorInvalidValue;
}

template <typename T>
static hipError_t attend_typed(const KvAttnArgs& a, int cols, unsigned grid, hipStream_t st) {
  switch (a.g.chunks) {
    case 2: return attend_cols<T, 2>(a, cols, grid, st);
    case 3: return attend_cols<T, 3>(a, cols, grid, st);
    case 4: return attend_cols<T, 4>(a, cols, grid, st);
    case 6: return attend_cols<T, 6>(a, cols, grid, st);
    case 8: return attend_cols<T, 8>(a, cols, grid, st);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_kv_attention(const KvAttnArgs& a, int cols, unsigned grid_items, unsigned grid_joins,
                               hipStream_t st) {
  if (grid_items == 0) return hipSuccess;
  hipError_t e = a.dtype == F32   ? attend_typed<float>(a, cols, grid_items, st)
                 : a.dtype == F16 ? attend_typed<_Float16>(a, cols, grid_items, st)
                                  : attend_typed<Bf16>(a, cols, grid_items, st);
  if (e == hipSuccess && grid_joins)
    e = launch(k_kv_join, dim3(grid_joins, 16u * cols), 256, 0, st, a, 16 * cols);
  return e;
}

}  // namespace hale
