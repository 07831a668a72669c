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
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

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

// Eight numbers of a row from p on, by its type.
__device__ __forceinline__ void load8(int dtype, const void* base, size_t at, bool vec, float* x) {
  if (dtype == F32) {
    const float* p = (const float*)base + at;
    if (vec) {
      const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        x[i] = a[i];
        x[i + 4] = b[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = p[i];
    }
    return;
  }
  union {
    u32x2 u[2];
    uint16_t h[8];
    _Float16 f[8];
  } r;
  const uint16_t* p = (const uint16_t*)base + at;
  if (vec) {
    r.u[0] = *(const u32x2*)p;
    r.u[1] = *(const u32x2*)(p + 4);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) r.h[i] = p[i];
  }
  if (dtype == F16) {
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = (float)r.f[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = __uint_as_float((unsigned)r.h[i] << 16);
  }
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

// KC: padded head dimension / 32; C: groups of 16 query rows; P: f16 parts per
// query number and probability.
template <int KC, int C, int P>
__global__ __launch_bounds__(64 * ATT_WAVES) void k_kv_attend(KvAttnArgs a) {
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
    const KvStepSeq sq = a.seqs[item.seq];
    const uint32_t* table = a.g.table + (size_t)sq.row * a.g.max_pages;
    const uint8_t* pool = a.g.pool + a.layer * a.g.layer_bytes + (size_t)item.head * a.g.head_bytes;

    // ---- the query rows ------------------------------------------------------
    f16x8 q[C][P][KC];
    float rs[C];      // what a score is multiplied with, but for the keys' scale
    int hi[C], lo[C];  // visible: lo < position <= hi
#pragma unroll
    for (int c = 0; c < C; c++) {
      const unsigned r = 16 * c + i;
      const bool valid = r < item.rows;
      const unsigned row = item.row0 + (valid ? r : 0), tok = row / (unsigned)a.g.group;
      hi[c] = valid ? (int)(sq.len0 + tok) : -1;
      lo[c] = a.window ? (int)(sq.len0 + tok) - a.window : -1;
      const size_t at = (size_t)(sq.tok0 + tok) * a.q_stride +
                        ((size_t)item.head * a.g.group + row % (unsigned)a.g.group) * a.g.hd;
      float x[KC][8], top = 0.0f;
#pragma unroll
      for (int kk = 0; kk < KC; kk++) {
        const int d0 = kk / 2 < KC / 2 ? 64 * (kk / 2) + 16 * g + 8 * (kk & 1) : 64 * (KC / 2) + 8 * g;
#pragma unroll
        for (int e = 0; e < 8; e++) x[kk][e] = 0.0f;
        if (valid && d0 < a.g.hd) load8(a.dtype, a.q, at + d0, a.vec, x[kk]);
#pragma unroll
        for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[kk][e]));
      }
      top = row_max(top);
      int ex = 0;
      if (top > 0.0f && top < __builtin_inff()) (void)frexpf(top, &ex);
      ex = ex < -100 ? -100 : ex;
      const float up = ldexpf(1.0f, 14 - ex);
      rs[c] = a.scale * ldexpf(1.0f, ex - 14);
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
    const int last = (int)(sq.len0 + item.row0 / (unsigned)a.g.group);
    const int first = a.window ? (int)(sq.len0 + (item.row0 + item.rows - 1) / (unsigned)a.g.group) - a.window + 1 : 0;

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
    unsigned p = item.page0 + wave;
    const uint8_t* base = nullptr;
    if (p < item.page1) {
      base = pool + (size_t)table[p] * a.g.page_bytes;
      load_k(base);
      load_v(base);
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
        next = pool + (size_t)table[pn] * a.g.page_bytes;
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
      base = next;
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
            store4(a.dtype, a.out, (size_t)(sq.tok0 + tok) * a.out_stride + (size_t)h * a.g.hd + d, a.vec, v * inv);
          else
            *(f32x4*)(a.part_o + prow * a.g.hd + d) = v;
        }
        if (item.part != KV_WHOLE && threadIdx.x % 16 == 0) a.part_ml[prow] = float2{top, total};
      }
    }
  }
}

// Joins the partial results of an item's rows: a work-group per 16 rows, 16
// threads per row, the parts in their order.
__global__ __launch_bounds__(256) void k_kv_join(KvAttnArgs a, int rows_per_part) {
  __shared__ float sw[16][65];
  const int r = threadIdx.x / 16, j = threadIdx.x % 16;
  const unsigned njoins = a.njoins != 0xffffffffu ? a.njoins : a.counts[1];
  for (unsigned it = blockIdx.x; it < njoins; it += gridDim.x) {
    const KvJoin join = a.joins[it];
    const unsigned row = 16 * blockIdx.y + r;
    const bool valid = row < join.rows;
    const float2* ml = a.part_ml + (size_t)join.part0 * rows_per_part + row;
    const float* po = a.part_o + ((size_t)join.part0 * rows_per_part + row) * a.g.hd;
    float top = -__builtin_inff();
    if (valid)
      for (unsigned k = j; k < join.parts; k += 16) top = fmaxf(top, ml[(size_t)k * rows_per_part].x);
#pragma unroll
    for (int x = 1; x < 16; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
    const float base2 = top == -__builtin_inff() ? 0.0f : top;
    float total = 0.0f;
    f32x4 v[4];
#pragma unroll
    for (int n = 0; n < 4; n++) v[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (unsigned k0 = 0; k0 < join.parts; k0 += 64) {
      const unsigned n = join.parts - k0 < 64 ? join.parts - k0 : 64;
      __syncthreads();
      if (valid)
        for (unsigned k = j; k < n; k += 16) {
          const float2 x = ml[(size_t)(k0 + k) * rows_per_part];
          const float w = exp2_fast(x.x - base2);
          sw[r][k] = w;
          total += w * x.y;
        }
      __syncthreads();
      if (valid)
        for (unsigned k = 0; k < n; k++) {
          const float w = sw[r][k];
          const float* src = po + (size_t)(k0 + k) * rows_per_part * a.g.hd;
#pragma unroll
          for (int x = 0; x < 4; x++)
            if (64 * x + 4 * j < a.g.hd) v[x] = v[x] + *(const f32x4*)(src + 64 * x + 4 * j) * w;
        }
    }
#pragma unroll
    for (int x = 1; x < 16; x *= 2) total += __shfl_xor(total, x);
    if (valid) {
      const KvStepSeq sq = a.seqs[join.seq];
      const unsigned tok = (join.row0 + row) / (unsigned)a.g.group;
      const unsigned h = join.head * a.g.group + (join.row0 + row) % (unsigned)a.g.group;
      const float inv = total > 0.0f ? 1.0f / total : 0.0f;
#pragma unroll
      for (int x = 0; x < 4; x++)
        if (64 * x + 4 * j < a.g.hd)
          store4(a.dtype, a.out, (size_t)(sq.tok0 + tok) * a.out_stride + (size_t)h * a.g.hd + 64 * x + 4 * j, a.vec,
                 v[x] * inv);
    }
  }
}

template <int KC, int P>
static hipError_t attend_cols(const KvAttnArgs& a, int cols, unsigned grid, hipStream_t st) {
  if (cols == 1) return launch(k_kv_attend<KC, 1, P>, grid, 64 * ATT_WAVES, 0, st, a);
  if constexpr (KC <= 6) {
    if (cols == 2) return launch(k_kv_attend<KC, 2, P>, grid, 64 * ATT_WAVES, 0, st, a);
  }
  return hipErrorInvalidValue;
}

template <int P>
static hipError_t attend_parts(const KvAttnArgs& a, int cols, unsigned grid, hipStream_t st) {
  switch (a.g.chunks) {
    case 2: return attend_cols<2, P>(a, cols, grid, st);
    case 3: return attend_cols<3, P>(a, cols, grid, st);
    case 4: return attend_cols<4, P>(a, cols, grid, st);
    case 6: return attend_cols<6, P>(a, cols, grid, st);
    case 8: return attend_cols<8, P>(a, cols, grid, st);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_kv_attention(const KvAttnArgs& a, int cols, unsigned grid_items, unsigned grid_joins,
                               hipStream_t st) {
  if (grid_items == 0) return hipSuccess;
  hipError_t e = a.dtype == F32 ? attend_parts<2>(a, cols, grid_items, st) : attend_parts<1>(a, cols, grid_items, st);
  if (e == hipSuccess && grid_joins)
    e = launch(k_kv_join, dim3(grid_joins, (unsigned)cols), 256, 0, st, a, 16 * cols);
  return e;
}

}  // namespace hale
