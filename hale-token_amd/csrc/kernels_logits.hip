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

constexpr int LG_THREADS = 512, LG_AHEAD = 8;
constexpr unsigned LG_OCCURS = 0x80000000u;  // in the prompt, beside the count of generated ones

template <typename T> __device__ __forceinline__ T lowest_of();
template <> __device__ __forceinline__ float lowest_of<float>() { return -__builtin_inff(); }
template <> __device__ __forceinline__ _Float16 lowest_of<_Float16>() { return (_Float16)-__builtin_inff(); }
template <> __device__ __forceinline__ Bf16 lowest_of<Bf16>() { return {0xff80}; }

__device__ __forceinline__ int64_t clamped(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }

// A work-group takes 512 * 8 * C neighbouring tokens of a row: in LDS it counts the row's
// tokens that fall among them, and then finds the last bias of each, while the logits are on their
// way, eight neighbours to a thread.  Counts and the biases' places are whole numbers, so
// the order of the atomics leaves no trace.  The one table serves both in turn, and tokens
// are read eight to a thread at a time: 64 rows of 151936 bf16 with up to 4000 tokens and 300 biases
// each 17.0 us (15.3 where the logits stay in the caches; 24 with a table for each, a token a thread
// at a time and two atomics for it; 15.9 with 256 threads).  Of the 15.3 reading and writing the
// logits alone takes 5.9, the mask 0.9, the tokens 5.4 and the biases 3.  Bound by each
// work-group's chain of reads (offsets, tokens, table) in little more than one round of them.  One row
// of f32 4.7 us, a launch alone 3.5.
template <typename T, int C, bool VEC>
__global__ __launch_bounds__(LG_THREADS) void k_logits(LogitsArgs a) {
  constexpr unsigned SLICE = LG_THREADS * 8 * C;
  __shared__ unsigned table[SLICE];
  __shared__ float biases[LG_THREADS];  // the first ones
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
  unsigned keep[C], named[C];  // a bit per logit: its mask's, and whether a rule has changed it
#pragma unroll
  for (int c = 0; c < C; c++) {
    const unsigned at = (c * LG_THREADS + t) * 8;
    keep[c] = mask && at < size ? mask[(first + at) / 32] >> at % 32 & 255 : 255;
    named[c] = 0;
  }
  int64_t b0 = 0, b1 = 0, t0 = 0, t1 = 0, made = 0;
  if (r.tokens) {
    t0 = clamped(r.token_start[row], 0, (int64_t)r.ntokens);
    t1 = clamped(r.token_start[row + 1], t0, (int64_t)r.ntokens);
    made = t0 + (r.prompt_len ? clamped(r.prompt_len[row], 0, t1 - t0) : 0);
  }
  if (r.bias_tokens) {
    b0 = clamped(r.bias_start[row], 0, (int64_t)r.nbiases);
    b1 = clamped(r.bias_start[row + 1], b0, (int64_t)r.nbiases);
  }
  int32_t bias_token = 0;
  if (b1 > b0) {  // on their way beside the row's tokens
    const int64_t k = b0 + t < b1 ? b0 + t : b1 - 1;
    bias_token = r.bias_tokens[k];
    biases[t] = r.bias[k];
  }
  float v[C][8];
  if (t1 > t0 || b1 > b0) {
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int j = 0; j < 8; j += 4) *(u32x4*)&table[(c * LG_THREADS + t) * 8 + j] = u32x4{0, 0, 0, 0};
  }
  if (t1 > t0) {
    const float repetition = r.repetition ? r.repetition[row] : 1.0f;
    const float frequency = r.frequency ? r.frequency[row] : 0.0f, presence = r.presence ? r.presence[row] : 0.0f;
    __syncthreads();
    // several tokens a thread at a time, on their way together
    const int32_t* tokens = r.tokens + t0;
    const unsigned n_tokens = (unsigned)(t1 - t0), n_prompt = (unsigned)(made - t0);
    for (unsigned from = t; from < n_tokens; from += LG_AHEAD * LG_THREADS) {
      int32_t token[LG_AHEAD];
#pragma unroll
      for (int k = 0; k < LG_AHEAD; k++) token[k] = tokens[min(from + k * LG_THREADS, n_tokens - 1)];
#pragma unroll
      for (int k = 0; k < LG_AHEAD; k++) {
        const size_t at = (size_t)(int64_t)token[k] - first;  // a token below `first`, or negative, is past all sizes
        if (at < size && from + k * LG_THREADS < n_tokens) {
          if (from + k * LG_THREADS >= n_prompt) atomicAdd(&table[at], 1u);
          else atomicOr(&table[at], LG_OCCURS);
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < C; c++) {
      unsigned n[8];
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        u32x4* own = (u32x4*)&table[(c * LG_THREADS + t) * 8 + j];
        *(u32x4*)&n[j] = *own;
        if (b1 > b0) *own = u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int j = 0; j < 8; j++) {
        if (!n[j]) continue;
        float y = to_f32(x[c][j]);
        y = y > 0.0f ? y / repetition : y * repetition;
        const unsigned g = n[j] & ~LG_OCCURS;
        if (g) y = (y - frequency * (float)g) - presence;
        v[c][j] = y;
        named[c] |= 1u << j;
      }
    }
  }
  if (b1 > b0) {
    __syncthreads();
    for (int64_t k = b0 + t; k < b1; k += LG_THREADS) {
      const size_t at = (size_t)(int64_t)(k < b0 + LG_THREADS ? bias_token : r.bias_tokens[k]) - first;
      if (at < size) atomicMax(&table[at], (unsigned)(k - b0 + 1));
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < C; c++) {
      unsigned p[8];
#pragma unroll
      for (int j = 0; j < 8; j += 4) *(u32x4*)&p[j] = *(const u32x4*)&table[(c * LG_THREADS + t) * 8 + j];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        if (!p[j]) continue;
        const float bias = p[j] <= LG_THREADS ? biases[p[j] - 1] : r.bias[b0 + (int64_t)p[j] - 1];
        v[c][j] = (named[c] >> j & 1 ? v[c][j] : to_f32(x[c][j])) + bias;
        named[c] |= 1u << j;
      }
    }
  }
#pragma unroll
  for (int c = 0; c < C; c++) {
    const unsigned at = (c * LG_THREADS + t) * 8;
    if (at >= size) continue;
    if (named[c]) {
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const T y = from_f32<T>(v[c][j]);
        if (named[c] >> j & 1) x[c][j] = y;
      }
    }
    if (keep[c] != 255) {
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (!(keep[c] >> j & 1)) x[c][j] = lowest_of<T>();
    }
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

template <typename T> static hipError_t logits_typed(const LogitsArgs& a, size_t rows, hipStream_t st) {
  // few rows: short work-groups; many: fewer passes over the rows' tokens (64 rows of 151936 15.1 us, 16.6
  // with half the slice; one 6.1, 4.7 with half)
  const bool large = rows * a.vocab >= (size_t)1 << 22;
  return large ? logits_sized<T, 2>(a, rows, st) : logits_sized<T, 1>(a, rows, st);
}

hipError_t launch_logits(int dtype, const LogitsArgs& a, size_t rows, hipStream_t st) {
  if (rows == 0 || a.vocab == 0) return hipSuccess;
  if (dtype == F32) return logits_typed<float>(a, rows, st);
  if (dtype == F16) return logits_typed<_Float16>(a, rows, st);
  return logits_typed<Bf16>(a, rows, st);
}

}  // namespace hale
