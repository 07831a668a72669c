// step_ops.hip -- host runtime of the operators around a serving step's
// layers: handles and argument checks of norms that hand on 8 bits, products of
// 4-bit weights with group scales, and rules on logits.
#include <hip/hip_runtime.h>

#include <cmath>
#include <memory>
#include <new>

#include "context.h"
#include "hale_device.h"
#include "host_call.h"
#include "kernels.h"
#include "step_ops.h"

using namespace hale;

// ---------------------------------------------------------------------------
// norms
// ---------------------------------------------------------------------------

extern "C" int hale_rms_norm_q8_device(hale_ctx* c, int dtype, size_t rows, size_t n, const void* x, size_t x_stride,
                                       const void* delta, size_t delta_stride, const float* weight, float eps,
                                       size_t block, void* sum, size_t sum_stride, void* y, size_t y_stride,
                                       int8_t* quants, float* scales) {
  if (!c) return ctx_fail(nullptr, HALE_EINVAL, "rms_norm_q8: NULL argument");
  if (!float_type(dtype)) return ctx_fail(c, HALE_EINVAL, "rms_norm_q8: dtype %d is not f32, f16 or bf16", dtype);
  if (n == 0 || n > NORM_Q8_MAX || n % 32)
    return ctx_fail(c, HALE_EINVAL, "rms_norm_q8: length %zu is not a multiple of 32 in 32..%zu", n, NORM_Q8_MAX);
  if ((block != 32 && block != 64 && block != 128 && block != n) || n % block)
    return ctx_fail(c, HALE_EINVAL, "rms_norm_q8: blocks of %zu in rows of %zu", block, n);
  if (!(eps >= 0.0f) || !std::isfinite(eps)) return ctx_fail(c, HALE_EINVAL, "rms_norm_q8: eps %g", (double)eps);
  if (rows >= STEP_ROWS) return ctx_fail(c, HALE_EINVAL, "rms_norm_q8: %zu rows", rows);
  if (rows == 0) return HALE_OK;
  if (!x || !weight || !quants || !scales) return ctx_fail(c, HALE_EINVAL, "rms_norm_q8: NULL argument");
  if (x_stride < n || (delta && delta_stride < n) || (sum && sum_stride < n) || (y && y_stride < n))
    return ctx_fail(c, HALE_EINVAL, "rms_norm_q8: a stride below the length %zu", n);
  if (!aligned(x, dtype) || !aligned(delta, dtype) || !aligned(sum, dtype) || !aligned(y, dtype) ||
      !aligned(weight, HALE_F32) || !aligned(scales, HALE_F32))
    return ctx_fail(c, HALE_EINVAL, "rms_norm_q8: not aligned to its type");
  // rows in place: another stride would write rows that are read later
  for (int i = 0; i < 2; i++) {
    const void* out = i ? y : sum;
    const size_t stride = i ? y_stride : sum_stride;
    if (out && rows > 1 && ((out == x && stride != x_stride) || (out == delta && stride != delta_stride)))
      return ctx_fail(c, HALE_EINVAL, "rms_norm_q8: in place with different strides");
  }
  if (sum && sum == y) return ctx_fail(c, HALE_EINVAL, "rms_norm_q8: two outputs in one place");
  NormQ8Args a{};
  a.x = x, a.delta = delta, a.w = weight, a.sum = sum, a.y = y, a.q = quants, a.scales = scales;
  a.x_stride = x_stride, a.delta_stride = delta_stride, a.sum_stride = sum_stride, a.y_stride = y_stride;
  a.n = (unsigned)n;
  a.block = block == 32 || block == 64 || block == 128 ? (unsigned)block : 0;
  a.eps = eps;
  uintptr_t any = (uintptr_t)x | (uintptr_t)weight | x_stride * type_bytes(dtype);
  if (delta) any |= (uintptr_t)delta | delta_stride * type_bytes(dtype);
  if (sum) any |= (uintptr_t)sum | sum_stride * type_bytes(dtype);
  if (y) any |= (uintptr_t)y | y_stride * type_bytes(dtype);
  a.vec = any % 16 == 0 && (uintptr_t)quants % 8 == 0;
  CALL_TRY
  std::lock_guard<std::recursive_mutex> lk(c->mu);
  CALL_CHK(c, hipSetDevice(c->device));
  CALL_LAUNCH(c, K_NORM_Q8, launch_norm_q8(dtype, a, rows, c->stream));
  return HALE_OK;
  CALL_CATCH(c)
}

// ---------------------------------------------------------------------------
// 4-bit weights with group scales
// ---------------------------------------------------------------------------

struct hale_q4g {
  hale_ctx* ctx = nullptr;
  Q4gGeom g{};
};

// A matrix from device memory, or from host memory (checked and sent first).
static int q4g_make(hale_ctx* c, size_t rows, size_t cols, size_t group, int scale_dtype, const uint8_t* codes,
                    const void* scales, const uint8_t* zeros, bool host, hale_q4g** out) {
  if (!c || !out) return ctx_fail(c, HALE_EINVAL, "q4g_upload: NULL argument");
  *out = nullptr;
  if (!codes || !scales) return ctx_fail(c, HALE_EINVAL, "q4g_upload: NULL argument");
  if (group != 32 && group != 64 && group != 128)
    return ctx_fail(c, HALE_EINVAL, "q4g_upload: groups of %zu (32, 64 or 128)", group);
  if (scale_dtype != HALE_F16 && scale_dtype != HALE_BF16)
    return ctx_fail(c, HALE_EINVAL, "q4g_upload: scales of dtype %d are not f16 or bf16", scale_dtype);
  if (rows == 0 || rows > (1u << 27) || cols == 0 || cols > (1u << 30) || cols % group)
    return ctx_fail(c, HALE_EINVAL, "q4g_upload: %zu rows of %zu in groups of %zu", rows, cols, group);
  if ((uintptr_t)scales % 2) return ctx_fail(c, HALE_EINVAL, "q4g_upload: scales are not aligned");
  const size_t groups = rows * (cols / group);
  if (host && zeros)
    for (size_t i = 0; i < groups; i++)
      if (zeros[i] > 15) return ctx_fail(c, HALE_EINVAL, "q4g_upload: zero %u of group %zu is above 15", zeros[i], i);
  CALL_TRY
  std::lock_guard<std::recursive_mutex> lk(c->mu);
  CALL_CHK(c, hipSetDevice(c->device));
  bool cap = false;
  const int rc = capturing(c, &cap);
  if (rc) return rc;
  if (cap) return ctx_fail(c, HALE_EINVAL, "q4g_upload while the stream is being captured");
  std::unique_ptr<hale_q4g> m(new hale_q4g);
  m->ctx = c;
  Q4gGeom& g = m->g;
  g.rows = rows;
  g.cols = cols;
  g.group = (unsigned)group;
  g.chunks = (unsigned)((cols + Q4G_CHUNK - 1) / Q4G_CHUNK);
  g.per = (unsigned)(Q4G_CHUNK / group);
  g.zeros = zeros != nullptr;
  g.bf16 = scale_dtype == HALE_BF16;
  g.scales_at = (size_t)g.chunks * 1024;
  const size_t zeros_at = g.scales_at + (size_t)g.chunks * 32 * g.per;
  g.tile_bytes = round_up(zeros_at + (g.zeros ? (size_t)g.chunks * 16 * g.per : 0), 128);
  const size_t tiles = (rows + Q4G_ROWS - 1) / Q4G_ROWS, bytes = tiles * g.tile_bytes;
  const size_t parts = q4g_part_tiles(tiles) * 1024, done = round_up(q4g_part_tiles(tiles) * 4, 256);
  if (hipMalloc(&g.data, bytes + parts + done + 64) != hipSuccess)
    return ctx_fail(c, HALE_ENOMEM, "q4g_upload: %zu bytes of weights and workspace", bytes + parts + done + 64);
  g.parts = (float*)(g.data + bytes);
  g.done = (unsigned*)(g.data + bytes + parts);
  g.zero_data = g.zeros ? g.data + zeros_at : g.data + bytes + parts + done;
  g.zero_chunk = g.zeros ? 16 * g.per : 0;
  g.zero_tile = g.zeros ? g.tile_bytes : 0;
  uint8_t* sent = nullptr;
  hipError_t e = done ? hipMemsetAsync(g.done, 0, done, c->stream) : hipSuccess;
  if (e == hipSuccess) e = hipMemsetAsync(g.data + bytes + parts + done, Q4G_OFFSET + 8, 64, c->stream);
  if (host) {
    const size_t cb = round_up(rows * (cols / 2), 256), sb = round_up(groups * 2, 256);
    if (hipMalloc(&sent, cb + sb + groups) != hipSuccess) {
      (void)hipFree(g.data);
      return ctx_fail(c, HALE_ENOMEM, "q4g_upload: %zu bytes on the way", cb + sb + groups);
    }
    if (e == hipSuccess) e = hipMemcpyAsync(sent, codes, rows * (cols / 2), hipMemcpyHostToDevice, c->stream);
    if (e == hipSuccess) e = hipMemcpyAsync(sent + cb, scales, groups * 2, hipMemcpyHostToDevice, c->stream);
    if (e == hipSuccess && zeros) e = hipMemcpyAsync(sent + cb + sb, zeros, groups, hipMemcpyHostToDevice, c->stream);
    codes = sent;
    scales = sent + cb;
    if (zeros) zeros = sent + cb + sb;
  }
  if (e == hipSuccess) {
    ctx_prof_begin(c, K_REPACK);
    e = launch_q4g_pack(g, codes, (const uint16_t*)scales, zeros, c->stream);
    ctx_prof_end(c);
  }
  const hipError_t s = hipStreamSynchronize(c->stream);
  if (e == hipSuccess) e = s;
  (void)hipFree(sent);
  if (e != hipSuccess) {
    (void)hipFree(g.data);
    return ctx_fail(c, HALE_EHIP, "q4g_upload: %s", hipGetErrorString(e));
  }
  *out = m.release();
  return HALE_OK;
  CALL_CATCH(c)
}

extern "C" int hale_q4g_upload(hale_ctx* c, size_t rows, size_t cols, size_t group, int scale_dtype,
                               const uint8_t* codes, const void* scales, const uint8_t* zeros, hale_q4g** out) {
  return q4g_make(c, rows, cols, group, scale_dtype, codes, scales, zeros, true, out);
}
extern "C" int hale_q4g_upload_device(hale_ctx* c, size_t rows, size_t cols, size_t group, int scale_dtype,
                                      const uint8_t* codes, const void* scales, const uint8_t* zeros, hale_q4g** out) {
  return q4g_make(c, rows, cols, group, scale_dtype, codes, scales, zeros, false, out);
}

extern "C" void hale_q4g_destroy(hale_q4g* m) {
  if (!m) return;
  hale_ctx* c = m->ctx;
  std::lock_guard<std::recursive_mutex> lk(c->mu);
  (void)hipSetDevice(c->device);
  (void)hipStreamSynchronize(c->stream);
  (void)hipFree(m->g.data);
  delete m;
}

extern "C" int hale_q4g_shape(const hale_q4g* m, size_t* rows, size_t* cols, size_t* group, int* scale_dtype,
                              int* has_zeros) {
  if (!m) return ctx_fail(nullptr, HALE_EINVAL, "q4g_shape: NULL argument");
  if (rows) *rows = m->g.rows;
  if (cols) *cols = m->g.cols;
  if (group) *group = m->g.group;
  if (scale_dtype) *scale_dtype = m->g.bf16 ? HALE_BF16 : HALE_F16;
  if (has_zeros) *has_zeros = m->g.zeros;
  return HALE_OK;
}

extern "C" int hale_q4g_download(hale_q4g* m, uint8_t* codes, void* scales, uint8_t* zeros) {
  if (!m || !codes || !scales) return ctx_fail(m ? m->ctx : nullptr, HALE_EINVAL, "q4g_download: NULL argument");
  hale_ctx* c = m->ctx;
  CALL_TRY
  std::lock_guard<std::recursive_mutex> lk(c->mu);
  CALL_CHK(c, hipSetDevice(c->device));
  bool cap = false;
  const int rc = capturing(c, &cap);
  if (rc) return rc;
  if (cap) return ctx_fail(c, HALE_EINVAL, "q4g_download while the stream is being captured");
  const Q4gGeom& g = m->g;
  const size_t groups = g.rows * (g.cols / g.group), n = g.rows * (g.cols / 2);
  const size_t cb = round_up(n, 256), sb = round_up(groups * 2, 256);
  uint8_t* back = nullptr;
  if (hipMalloc(&back, cb + sb + groups) != hipSuccess)
    return ctx_fail(c, HALE_ENOMEM, "q4g_download: %zu bytes on the way", cb + sb + groups);
  hipError_t e = launch_q4g_unpack(g, back, (uint16_t*)(back + cb), back + cb + sb, c->stream);
  if (e == hipSuccess) e = hipMemcpyAsync(codes, back, n, hipMemcpyDeviceToHost, c->stream);
  if (e == hipSuccess) e = hipMemcpyAsync(scales, back + cb, groups * 2, hipMemcpyDeviceToHost, c->stream);
  if (e == hipSuccess && zeros) e = hipMemcpyAsync(zeros, back + cb + sb, groups, hipMemcpyDeviceToHost, c->stream);
  const hipError_t s = hipStreamSynchronize(c->stream);
  if (e == hipSuccess) e = s;
  (void)hipFree(back);
  if (e != hipSuccess) return ctx_fail(c, HALE_EHIP, "q4g_download: %s", hipGetErrorString(e));
  return HALE_OK;
  CALL_CATCH(c)
}

static int q4g_run(hale_q4g* m, Q4gInput in, Q4gArgs& a, int dtype, size_t ntok, void* out, size_t out_stride) {
  hale_ctx* c = m->ctx;
  if (!float_type(dtype)) return ctx_fail(c, HALE_EINVAL, "q4g_matmul: dtype %d is not f32, f16 or bf16", dtype);
  if (ntok > (1u << 20)) return ctx_fail(c, HALE_EINVAL, "q4g_matmul: %zu tokens, at most 2^20", ntok);
  if (ntok * m->g.rows > ((size_t)1 << 35))
    return ctx_fail(c, HALE_EINVAL, "q4g_matmul: %zu results of %zu tokens, at most 2^35 in all", m->g.rows, ntok);
  if (ntok == 0) return HALE_OK;
  if (!a.x || !out || (in == Q4G_I8 && !a.x_scales)) return ctx_fail(c, HALE_EINVAL, "q4g_matmul: NULL argument");
  if (a.x_stride < m->g.cols || out_stride < m->g.rows)
    return ctx_fail(c, HALE_EINVAL, "q4g_matmul: strides %zu and %zu below %zu and %zu", a.x_stride, out_stride, m->g.cols, m->g.rows);
  if (!aligned(out, dtype) || (in == Q4G_I8 ? (uintptr_t)a.x % 8 || !aligned(a.x_scales, HALE_F32) : !aligned(a.x, dtype)))
    return ctx_fail(c, HALE_EINVAL, "q4g_matmul: not aligned");
  a.g = m->g;
  a.ntok = ntok;
  a.out_dtype = dtype;
  a.out = out;
  a.out_stride = out_stride;
  a.out_vec = ((uintptr_t)out | out_stride * type_bytes(dtype)) % (4 * type_bytes(dtype)) == 0;
  CALL_TRY
  std::lock_guard<std::recursive_mutex> lk(c->mu);
  CALL_CHK(c, hipSetDevice(c->device));
  CALL_LAUNCH(c, K_Q4G, launch_q4g(in, a, c->stream));
  return HALE_OK;
  CALL_CATCH(c)
}

extern "C" int hale_q4g_matmul_device(hale_q4g* m, int dtype, size_t ntok, const void* x, size_t x_stride, void* out,
                                      size_t out_stride) {
  if (!m) return ctx_fail(nullptr, HALE_EINVAL, "q4g_matmul: NULL argument");
  Q4gArgs a{};
  a.x = x;
  a.x_stride = x_stride;
  const Q4gInput in = dtype == HALE_F32 ? Q4G_F32 : dtype == HALE_F16 ? Q4G_F16 : Q4G_BF16;
  return q4g_run(m, in, a, dtype, ntok, out, out_stride);
}

extern "C" int hale_q4g_matmul_q8_device(hale_q4g* m, size_t ntok, size_t block, const int8_t* quants,
                                         const float* scales, int dtype, void* out, size_t out_stride) {
  if (!m) return ctx_fail(nullptr, HALE_EINVAL, "q4g_matmul_q8: NULL argument");
  if ((block != 32 && block != 64 && block != 128 && block != m->g.cols) || m->g.cols % block)
    return ctx_fail(m->ctx, HALE_EINVAL, "q4g_matmul_q8: blocks of %zu in rows of %zu", block, m->g.cols);
  Q4gArgs a{};
  a.x = quants;
  a.x_scales = scales;
  a.x_stride = m->g.cols;
  a.x_shift = block == 32 ? 5 : block == 64 ? 6 : block == 128 ? 7 : 31;
  a.x_per = (unsigned)(m->g.cols / block);
  return q4g_run(m, Q4G_I8, a, dtype, ntok, out, out_stride);
}

// ---------------------------------------------------------------------------
// logits
// ---------------------------------------------------------------------------

extern "C" int hale_logits_device(hale_ctx* c, int dtype, size_t rows, size_t vocab, const void* logits, size_t stride,
                                  const hale_logits_rules* rules, void* out, size_t out_stride) {
  if (!c || !rules) return ctx_fail(c, HALE_EINVAL, "logits: NULL argument");
  if (!float_type(dtype)) return ctx_fail(c, HALE_EINVAL, "logits: dtype %d is not f32, f16 or bf16", dtype);
  if (rows >= STEP_ROWS || vocab > (1u << 26)) return ctx_fail(c, HALE_EINVAL, "logits: %zu rows of %zu", rows, vocab);
  if (rules->ntokens >= (1ull << 31) || rules->nbiases >= (1ull << 31))
    return ctx_fail(c, HALE_EINVAL, "logits: %zu tokens and %zu biases", rules->ntokens, rules->nbiases);
  if (rows == 0 || vocab == 0) return HALE_OK;
  if (!logits || !out) return ctx_fail(c, HALE_EINVAL, "logits: NULL argument");
  if (stride < vocab || out_stride < vocab)
    return ctx_fail(c, HALE_EINVAL, "logits: strides %zu and %zu below %zu", stride, out_stride, vocab);
  if (!aligned(logits, dtype) || !aligned(out, dtype)) return ctx_fail(c, HALE_EINVAL, "logits: not aligned to its type");
  if (logits == out && stride != out_stride && rows > 1)
    return ctx_fail(c, HALE_EINVAL, "logits: in place with different strides");
  LogitsArgs a{};
  a.r = *rules;
  const hale_logits_rules& r = *rules;
  if (r.tokens && !r.token_start) return ctx_fail(c, HALE_EINVAL, "logits: tokens without token_start");
  if (r.bias_tokens && (!r.bias || !r.bias_start)) return ctx_fail(c, HALE_EINVAL, "logits: biases without values or bias_start");
  if (r.mask) {
    if (r.mask_stride < (vocab + 31) / 32)
      return ctx_fail(c, HALE_EINVAL, "logits: a mask stride of %zu words for %zu tokens", r.mask_stride, vocab);
    if (!r.mask_row && r.mask_rows < rows)
      return ctx_fail(c, HALE_EINVAL, "logits: %zu masks for %zu rows", r.mask_rows, rows);
  }
  for (const void* p : {(const void*)r.tokens, (const void*)r.repetition, (const void*)r.frequency, (const void*)r.presence,
                        (const void*)r.bias_tokens, (const void*)r.bias, (const void*)r.mask, (const void*)r.mask_row})
    if ((uintptr_t)p % 4) return ctx_fail(c, HALE_EINVAL, "logits: a rule's array is not aligned");
  for (const void* p : {(const void*)r.token_start, (const void*)r.prompt_len, (const void*)r.bias_start})
    if ((uintptr_t)p % 8) return ctx_fail(c, HALE_EINVAL, "logits: a rule's array is not aligned");
  a.in = logits;
  a.out = out;
  a.in_stride = stride;
  a.out_stride = out_stride;
  a.vocab = vocab;
  a.vec = ((uintptr_t)logits | (uintptr_t)out | stride * type_bytes(dtype) | out_stride * type_bytes(dtype)) % 16 == 0;
  CALL_TRY
  std::lock_guard<std::recursive_mutex> lk(c->mu);
  CALL_CHK(c, hipSetDevice(c->device));
  CALL_LAUNCH(c, K_LOGITS, launch_logits(dtype, a, rows, c->stream));
  return HALE_OK;
  CALL_CATCH(c)
}
