// kernels_norm_q8.hip -- the residual's addition and RMS norm of rows, handing
// on 8 bits with a scale per block.
//
// s = x + delta (in f32, rounded to the type), u = s w, r = 1 / sqrt(sum(s^2) / n
// + eps), y = r u; a block's scale is r max|u| / 127 and its codes are 127 u /
// max|u| to the nearest whole number, ties to even.  r is no part of the codes:
// they follow from u alone, which 64 bits hold exactly (24 bits times 24), so that
// every code is the nearest one.  The squares are summed in 64 bits too, where no f32
// number's square leaves the range.
#include <hip/hip_runtime.h>

#include "hale_device.h"
#include "kernels.h"
#include "kv_device.h"
#include "step_ops.h"

namespace hale {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// Eight numbers of a row as they lie.
template <typename T> struct Eight {
  alignas(16) T v[8];
  template <bool VEC> __device__ __forceinline__ void load(const void* base, size_t at) {
    const T* p = (const T*)base + at;
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < 8; j += 16 / (int)sizeof(T)) *(u32x4*)&v[j] = *(const u32x4*)(p + j);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = p[j];
    }
  }
  template <bool VEC> __device__ __forceinline__ void store(void* base, size_t at) const {
    T* p = (T*)base + at;
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < 8; j += 16 / (int)sizeof(T)) *(u32x4*)(p + j) = *(const u32x4*)&v[j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) p[j] = v[j];
    }
  }
  // Rounded to nearest even; a NaN stays one.
  __device__ __forceinline__ void round(const float (&f)[8]) {
    if constexpr (sizeof(T) == 2 && !__is_same(T, _Float16)) {  // two at a time, without a branch for NaNs
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const bf16x2 r = __builtin_convertvector(f32x2{f[j], f[j + 1]}, bf16x2);
        __builtin_memcpy(&v[j], &r, 4);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = from_f32<T>(f[j]);
    }
  }
};

__device__ __forceinline__ double from_words(unsigned lo, unsigned hi) {
  return __longlong_as_double((long long)((unsigned long long)hi << 32 | lo));
}
// A number of 64 bits as an f32 that rounds to f16 and bf16 as it does itself: the leading 13
// bits, the last of them set where anything was cut off (11 for f16, the next, and whether there are more).
// The nearest f32 would be rounded a second time, and a number beside a border of the 16 bits could
// come to lie on it.  f32 holds 13 bits down to 2^-137, below what bf16 rounds to 0.
__device__ __forceinline__ float odd_f32(double d) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(d);
  const unsigned hi = (unsigned)(b >> 32), rest = (hi & 0xffu) | (unsigned)b;
  return (float)from_words(0, (hi & ~0xffu) | (rest ? 0x100u : 0u));
}

template <int CTRL> __device__ __forceinline__ double dpp64(double v) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(v);
  return from_words((unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)b, CTRL, 0xF, 0xF, false),
                    (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(b >> 32), CTRL, 0xF, 0xF, false));
}
// Over the whole wave, from within rows of 16 lanes outward.
template <typename Op> __device__ __forceinline__ double over_rows(double v, Op op) {
  unsigned long long b = (unsigned long long)__double_as_longlong(v);
  auto lo = __builtin_amdgcn_permlane16_swap((unsigned)b, (unsigned)b, false, false);
  auto hi = __builtin_amdgcn_permlane16_swap((unsigned)(b >> 32), (unsigned)(b >> 32), false, false);
  v = op(from_words(lo[0], hi[0]), from_words(lo[1], hi[1]));
  b = (unsigned long long)__double_as_longlong(v);
  lo = __builtin_amdgcn_permlane32_swap((unsigned)b, (unsigned)b, false, false);
  hi = __builtin_amdgcn_permlane32_swap((unsigned)(b >> 32), (unsigned)(b >> 32), false, false);
  return op(from_words(lo[0], hi[0]), from_words(lo[1], hi[1]));
}
struct Add64 { __device__ double operator()(double a, double b) const { return a + b; } };
struct Max64 { __device__ double operator()(double a, double b) const { return fmax(a, b); } };

// The code of u, inv = 127 / top: the nearest whole number to 127 u / top.  The
// product is good to 2^-51 of at most 127; where it lies that near to a border, both
// sides of 254 |u| <> (2 k + 1) top are compared exactly (each product and its rounding).
__device__ __forceinline__ int code_of(double u, double top, double inv) {
  const double t = u * inv, q = rint(t);
  if (fabs(fabs(t - q) - 0.5) < 1e-12) {
    const double k = floor(fabs(t)), a = fabs(u), odd = 2 * k + 1;
    const double p = 254 * a, pe = __builtin_fma(254.0, a, -p), r = odd * top, re = __builtin_fma(odd, top, -r);
    const double d = (p - r) + (pe - re);
    const int m = (int)k, c = d > 0 ? m + 1 : d < 0 ? m : m + (m & 1);
    return u < 0 ? -c : c;
  }
  return (int)q;
}

// A work-group of NT threads per row, C groups of eight numbers a thread, all of them on
// their way at once and read before anything is written.  Four groups a thread spill
// (64-bit codes of 32 numbers), hence 1024 threads and 16384 numbers at most.  Blocks of 32, 64 and 128 numbers lie in 4, 8 and 16
// neighbouring lanes.
template <typename T, int NT, int C, bool VEC>
__global__ __launch_bounds__(NT) void k_norm_q8(NormQ8Args a) {
  constexpr int W = NT / 64;
  __shared__ double red[2][W];
  const int t = threadIdx.x, wave = t >> 6;
  const size_t row = blockIdx.x;
  const unsigned groups = a.n / 8;
  Eight<T> sum8[C], delta[C];
  Eight<float> weight[C];
  float s[C][8], w[C][8];
#pragma unroll
  for (int c = 0; c < C; c++) {  // groups behind the row are some of it, and count for nothing
    const unsigned at = 8 * min((unsigned)(t + NT * c), groups - 1);
    sum8[c].template load<VEC>(a.x, row * a.x_stride + at);
    if (a.delta) delta[c].template load<VEC>(a.delta, row * a.delta_stride + at);
    weight[c].template load<VEC>(a.w, at);
  }
#pragma unroll
  for (int c = 0; c < C; c++) {
    if (a.delta) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; j++) f[j] = to_f32(sum8[c].v[j]) + to_f32(delta[c].v[j]);
      sum8[c].round(f);
    }
    const bool in = (unsigned)(t + NT * c) < groups;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      s[c][j] = in ? to_f32(sum8[c].v[j]) : 0.0f;
      w[c][j] = in ? weight[c].v[j] : 0.0f;
    }
  }
  double sum = 0, top[C];
#pragma unroll
  for (int c = 0; c < C; c++) {
    double most = 0, odd = 0;  // odd: not a number where some u is not finite
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const double v = s[c][j], u = v * (double)w[c][j];
      sum = __builtin_fma(v, v, sum);
      most = fmax(most, fabs(u));
      odd = __builtin_fma(u, 0.0, odd);
    }
    top[c] = odd == 0 ? most : __builtin_inf();
  }
  sum = sum + dpp64<0xB1>(sum);
  sum = sum + dpp64<0x4E>(sum);
  sum = sum + dpp64<0x141>(sum);
  sum = sum + dpp64<0x140>(sum);
  sum = over_rows(sum, Add64());
  if (a.block == 0) {
    double most = top[0];
#pragma unroll
    for (int c = 1; c < C; c++) most = fmax(most, top[c]);
    most = fmax(most, dpp64<0xB1>(most));
    most = fmax(most, dpp64<0x4E>(most));
    most = fmax(most, dpp64<0x141>(most));
    most = fmax(most, dpp64<0x140>(most));
    most = over_rows(most, Max64());
    if (W > 1 && t % 64 == 0) red[1][wave] = most;
    top[0] = most;
  }
  if constexpr (W > 1) {
    if (t % 64 == 0) red[0][wave] = sum;
    __syncthreads();
    sum = red[0][0];
#pragma unroll
    for (int k = 1; k < W; k++) sum += red[0][k];
    if (a.block == 0) {
      top[0] = red[1][0];
#pragma unroll
      for (int k = 1; k < W; k++) top[0] = fmax(top[0], red[1][k]);
    }
  }
  // a row with a number that is not finite: nothing of it is
  const double r = sum < __builtin_inf() ? 1.0 / sqrt(sum / (double)a.n + (double)a.eps) : __builtin_nan("");
#pragma unroll
  for (int c = 0; c < C; c++) {
    const unsigned at = (unsigned)(t + NT * c);
    double m = a.block == 0 ? top[0] : top[c];
    if (a.block) {
      m = fmax(m, dpp64<0xB1>(m));
      m = fmax(m, dpp64<0x4E>(m));
      if (a.block > 32) m = fmax(m, dpp64<0x141>(m));
      if (a.block > 64) m = fmax(m, dpp64<0x140>(m));
    }
    const bool finite = m < __builtin_inf() && r < __builtin_inf();
    const double inv = finite && m > 0 ? 127.0 / m : 0.0;
    if (at >= groups) continue;
    unsigned q[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      q[h] = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int i = 4 * h + j;
        // (m and not inv: 0 times a number that is not finite)
        const int code = finite ? code_of((double)s[c][i] * (double)w[c][i], m, inv) : 0;
        q[h] |= (unsigned)(code & 255) << (8 * j);
      }
    }
    int8_t* pq = a.q + row * a.n + 8 * at;
    if constexpr (VEC) {
      *(u32x2*)pq = u32x2{q[0], q[1]};
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) pq[j] = (int8_t)(q[j / 4] >> (8 * (j % 4)));
    }
    const float scale = finite ? (float)(r * m / 127.0) : __builtin_nanf("");
    if (a.block == 0) {
      if (at == 0) a.scales[row] = scale;
    } else if (8 * at % a.block == 0) {
      a.scales[row * (a.n / a.block) + 8 * at / a.block] = scale;
    }
    if (a.sum) sum8[c].template store<VEC>(a.sum, row * a.sum_stride + 8 * at);
    if (a.y) {
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const double d = (double)s[c][j] * (double)w[c][j] * r;
        if constexpr (sizeof(T) == 2) y[j] = odd_f32(d);
        else y[j] = (float)d;
      }
      Eight<T> y8;
      y8.round(y);
      y8.template store<VEC>(a.y, row * a.y_stride + 8 * at);
    }
  }
}

template <typename T, bool VEC>
static hipError_t norm_sized(const NormQ8Args& a, size_t rows, hipStream_t st) {
  const unsigned groups = a.n / 8, grid = (unsigned)rows;
  if (groups <= 64) return launch(k_norm_q8<T, 64, 1, VEC>, grid, 64, 0, st, a);
  if (groups <= 256) return launch(k_norm_q8<T, 256, 1, VEC>, grid, 256, 0, st, a);
  if (groups <= 512) return launch(k_norm_q8<T, 256, 2, VEC>, grid, 256, 0, st, a);
  if (groups <= 1024) return launch(k_norm_q8<T, 512, 2, VEC>, grid, 512, 0, st, a);
  return launch(k_norm_q8<T, 1024, 2, VEC>, grid, 1024, 0, st, a);
}

hipError_t launch_norm_q8(int dtype, const NormQ8Args& a, size_t rows, hipStream_t st) {
  if (rows == 0) return hipSuccess;
  if (dtype == F32) return a.vec ? norm_sized<float, true>(a, rows, st) : norm_sized<float, false>(a, rows, st);
  if (dtype == F16) return a.vec ? norm_sized<_Float16, true>(a, rows, st) : norm_sized<_Float16, false>(a, rows, st);
  return a.vec ? norm_sized<Bf16, true>(a, rows, st) : norm_sized<Bf16, false>(a, rows, st);
}

}  // namespace hale
