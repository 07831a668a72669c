// kernels_logits.hip -- rules on logits: penalties for tokens that occur
// already, biases, and masks of the tokens that a grammar allows.
//
// For each row and token, in f32: with c the occurrences among the row's
// tokens and g those among the generated ones (behind the prompt),
//   c > 0: x > 0 ? x / repetition : x * repetition
//   g > 0: (x - frequency g) - presence
//   x + bias; then -inf where the mask's bit is 0.
// A token that no rule names keeps its bits.
#include <hip/hip_runtime.h>

#include "hale_device.h"
#include "kernels.h"
#include "kv_device.h"
#include "step_ops.h"

namespace hale {

constexpr int LG_THREADS = 256;
constexpr unsigned LG_OCCURS = 0x80000000u;  // beside the count of generated ones

template <typename T> __device__ __forceinline__ T lowest_of();
template <> __device__ __forceinline__ float lowest_of<float>() { return -__builtin_inff(); }
template <> __device__ __forceinline__ _Float16 lowest_of<_Float16>() { return (_Float16)-__builtin_inff(); }
template <> __device__ __forceinline__ Bf16 lowest_of<Bf16>() { return {0xff80}; }

__device__ __forceinline__ int64_t clamped(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }

// A work-group takes 256 * 8 * C neighbouring tokens of a row: it counts, in LDS, the
// row's tokens that fall among them, finds the last bias of each, and applies all of it in
// one pass over the logits, which are on their way meanwhile.  Counts and the biases'
// places are whole numbers, so the order of the atomics leaves no trace.
template <typename T, int C, bool VEC>
__global__ __launch_bounds__(LG_THREADS) void k_logits(LogitsArgs a) {
  constexpr unsigned SLICE = LG_THREADS * 8 * C;
  __shared__ unsigned count[SLICE], place[SLICE];
  const unsigned t = threadIdx.x;
  const size_t row = blockIdx.x, first = (size_t)blockIdx.y * SLICE;
  const unsigned size = (unsigned)(a.vocab - first < SLICE ? a.vocab - first : SLICE);
  const T* in = (const T*)a.in + row * a.in_stride + first;
  T* out = (T*)a.out + row * a.out_stride + first;
  const hale_logits_rules& r = a.r;

  alignas(16) T x[C][8];
#pragma unroll
  for (int c = 0; c < C; c++) {
    const unsigned at = (c * LG_THREADS + t) * 8;
    if (VEC && at + 8 <= size) {
#pragma unroll
      for (int j = 0; j < 8; j += 16 / (int)sizeof(T)) *(u32x4*)&x[c][j] = *(const u32x4*)(in + at + j);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (at + j < size) x[c][j] = in[at + j];
    }
  }
  const uint32_t* mask = nullptr;
  if (r.mask) {
    const int64_t m = r.mask_row ? (int64_t)r.mask_row[row] : (int64_t)row;
    if (m >= 0 && m < (int64_t)r.mask_rows) mask = r.mask + (size_t)m * r.mask_stride;
  }
  unsigned keep[C];
#pragma unroll
  for (int c = 0; c < C; c++) {
    const unsigned at = (c * LG_THREADS + t) * 8;
    keep[c] = mask && at < size ? mask[(first + at) / 32] >> at % 32 & 255 : 255;
  }
  int64_t b0 = 0, b1 = 0, t0 = 0, t1 = 0, made = 0;
  if (r.tokens) {
    t0 = clamped(r.token_start[row], 0, (int64_t)r.ntokens);
    t1 = clamped(r.token_start[row + 1], t0, (int64_t)r.ntokens);
    made = r.prompt_len ? clamped(r.prompt_len[row], 0, t1 - t0) : 0;
  }
  if (r.bias_tokens) {
    b0 = clamped(r.bias_start[row], 0, (int64_t)r.nbiases);
    b1 = clamped(r.bias_start[row + 1], b0, (int64_t)r.nbiases);
  }
  const float repetition = r.repetition ? r.repetition[row] : 1.0f;
  const float frequency = r.frequency ? r.frequency[row] : 0.0f, presence = r.presence ? r.presence[row] : 0.0f;
  const bool any = t1 > t0 || b1 > b0;
  if (any) {
    for (unsigned k = 4 * t; k < SLICE; k += 4 * LG_THREADS) {
      *(u32x4*)&count[k] = u32x4{0, 0, 0, 0};
      *(u32x4*)&place[k] = u32x4{0, 0, 0, 0};
    }
    __syncthreads();
    made += t0;
#pragma unroll 8
    for (int64_t k = t0 + t; k < t1; k += LG_THREADS) {
      const size_t at = (size_t)(int64_t)r.tokens[k] - first;  // a token below `first`, or negative, is past all sizes
      if (at < size) {
        if (k >= made) atomicAdd(&count[at], 1u);
        atomicOr(&count[at], LG_OCCURS);
      }
    }
    for (int64_t k = b0 + t; k < b1; k += LG_THREADS) {
      const size_t at = (size_t)(int64_t)r.bias_tokens[k] - first;
      if (at < size) atomicMax(&place[at], (unsigned)(k - b0 + 1));
    }
    __syncthreads();
  }
#pragma unroll
  for (int c = 0; c < C; c++) {
    const unsigned at = (c * LG_THREADS + t) * 8;
    if (at >= size) continue;
    if (any) {
      unsigned n[8], p[8];
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        *(u32x4*)&n[j] = *(const u32x4*)&count[at + j];
        *(u32x4*)&p[j] = *(const u32x4*)&place[at + j];
      }
#pragma unroll
      for (int j = 0; j < 8; j++) {
        if (!(n[j] | p[j])) continue;
        float v = to_f32(x[c][j]);
        if (n[j]) {
          v = v > 0.0f ? v / repetition : v * repetition;
          const unsigned g = n[j] & ~LG_OCCURS;
          if (g) v = (v - frequency * (float)g) - presence;
        }
        if (p[j]) v = v + r.bias[b0 + (int64_t)p[j] - 1];
        x[c][j] = from_f32<T>(v);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (!(keep[c] >> j & 1)) x[c][j] = lowest_of<T>();
    if (VEC && at + 8 <= size) {
#pragma unroll
      for (int j = 0; j < 8; j += 16 / (int)sizeof(T)) *(u32x4*)(out + at + j) = *(const u32x4*)&x[c][j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (at + j < size) out[at + j] = x[c][j];
    }
  }
}

template <typename T, int C>
static hipError_t logits_sized(const LogitsArgs& a, size_t rows, hipStream_t st) {
  const unsigned slices = (unsigned)((a.vocab + LG_THREADS * 8 * C - 1) / (LG_THREADS * 8 * C));
  const dim3 grid((unsigned)rows, slices);
  return a.vec ? launch(k_logits<T, C, true>, grid, LG_THREADS, 0, st, a) : launch(k_logits<T, C, false>, grid, LG_THREADS, 0, st, a);
}

hipError_t launch_logits(int dtype, const LogitsArgs& a, size_t rows, hipStream_t st) {
  if (rows == 0 || a.vocab == 0) return hipSuccess;
  if (dtype == F32) return logits_sized<float, 1>(a, rows, st);
  if (dtype == F16) return logits_sized<_Float16, 1>(a, rows, st);
  return logits_sized<Bf16, 1>(a, rows, st);
}

}  // namespace hale
