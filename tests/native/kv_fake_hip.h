// A HIP runtime in host memory under the key/value cache's host side
// (hale-token_amd/csrc/kv.hip, host pass), so that its steps, uploads, graphs
// and failures run on the CPU under AddressSanitizer.  Uploads are carried
// out, kernels that compute are only noted.
#pragma once

#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <new>
#include <set>
#include <string>
#include <vector>

#include "context.h"
#include "kv.h"

#define CHECK(cond)                                                    \
  do {                                                                 \
    if (!(cond)) {                                                     \
      fprintf(stderr, "line %d: %s does not hold\n", __LINE__, #cond); \
      exit(1);                                                         \
    }                                                                  \
  } while (0)

// What the fake runtime is told and what it saw.
struct Fake {
  bool capturing = false;
  int allocs_until_failure = -1;         // of any kind; -1: none fails
  std::set<void*> device, host;          // allocated now
  int uploads = 0;
  std::vector<hale::KvAttnArgs> attends;  // in the order of the calls
  std::vector<hale::KvAppendArgs> appends;
  std::vector<size_t> read_counts;
  int ropes = 0;
};
static Fake fake;

static bool fails() { return fake.allocs_until_failure >= 0 && fake.allocs_until_failure-- == 0; }

void* operator new(size_t n) {
  void* p = fails() ? nullptr : malloc(n);
  if (!p) throw std::bad_alloc();
  return p;
}
void* operator new(size_t n, const std::nothrow_t&) noexcept { return fails() ? nullptr : malloc(n); }
void operator delete(void* p) noexcept { free(p); }
void operator delete(void* p, size_t) noexcept { free(p); }

extern "C" {
hipError_t hipMalloc(void** p, size_t n) {
  if (fails()) return hipErrorOutOfMemory;
  *p = malloc(n);
  const int left = fake.allocs_until_failure;  // the fake's own books never fail
  fake.allocs_until_failure = -1;
  fake.device.insert(*p);
  fake.allocs_until_failure = left;
  return *p ? hipSuccess : hipErrorOutOfMemory;
}
hipError_t hipFree(void* p) {
  if (!p) return hipSuccess;
  CHECK(fake.device.erase(p) == 1);
  free(p);
  return hipSuccess;
}
hipError_t hipHostMalloc(void** p, size_t n, unsigned) {
  if (fails()) return hipErrorOutOfMemory;
  *p = malloc(n);
  const int left = fake.allocs_until_failure;
  fake.allocs_until_failure = -1;
  fake.host.insert(*p);
  fake.allocs_until_failure = left;
  return *p ? hipSuccess : hipErrorOutOfMemory;
}
hipError_t hipHostFree(void* p) {
  CHECK(fake.host.erase(p) == 1);
  free(p);
  return hipSuccess;
}
hipError_t hipMemsetAsync(void* p, int v, size_t n, hipStream_t) {
  memset(p, v, n);
  return hipSuccess;
}
hipError_t hipMemcpyAsync(void* d, const void* s, size_t n, hipMemcpyKind, hipStream_t) {
  memcpy(d, s, n);
  return hipSuccess;
}
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) {
  *s = fake.capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
  return hipSuccess;
}
const char* hipGetErrorString(hipError_t) { return "an error of the fake runtime"; }
}

namespace hale {

int ctx_fail(hale_ctx* c, int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  fake.allocs_until_failure = -1;
  if (c) c->err = buf;
  return code;
}
void ctx_prof_begin(hale_ctx*, int) {}
void ctx_prof_end(hale_ctx*) {}

hipError_t launch_kv_upload(const KvUploadArgs& a, hipStream_t) {
  CHECK(!fake.capturing);
  CHECK(a.pieces >= 0 && a.pieces <= KV_MAX_PIECES);
  fake.uploads++;
  *a.done = a.number;
  const uint32_t* s = a.src;
  for (int p = 0; p < a.pieces; p++) {
    CHECK(a.words[p] % 4 == 0);
    memcpy(a.dst[p], s, a.words[p] * 4);
    s += a.words[p];
  }
  for (unsigned i = 0; i < a.npairs; i++) a.table[a.pairs[2 * i]] = a.pairs[2 * i + 1];
  for (unsigned i = 0; i < a.ncopies; i++)
    memcpy(a.pool + a.copies[i].dst * a.page_bytes, a.pool + a.copies[i].src * a.page_bytes, a.page_bytes);
  return hipSuccess;
}
hipError_t launch_kv_append(int, const KvAppendArgs& a, unsigned, hipStream_t) {
  fake.allocs_until_failure = -1;
  fake.appends.push_back(a);
  return hipSuccess;
}
hipError_t launch_kv_read(const KvGeom&, size_t, uint32_t, size_t, size_t count, float*, float*, hipStream_t) {
  fake.read_counts.push_back(count);
  return hipSuccess;
}
hipError_t launch_kv_attend_few(const KvAttnArgs& a, int, unsigned, hipStream_t) {
  fake.allocs_until_failure = -1;
  fake.attends.push_back(a);
  return hipSuccess;
}
hipError_t launch_kv_attend_many(const KvAttnArgs& a, unsigned, hipStream_t) {
  fake.allocs_until_failure = -1;
  fake.attends.push_back(a);
  return hipSuccess;
}
hipError_t launch_kv_join(const KvAttnArgs&, unsigned, unsigned, unsigned, hipStream_t) { return hipSuccess; }
hipError_t launch_rope(int, const RopeArgs&, hipStream_t) {
  fake.ropes++;
  return hipSuccess;
}
hipError_t launch_copy(void* d, const void* s, size_t n16, hipStream_t) {
  memcpy(d, s, n16 * 16);
  return hipSuccess;
}

}  // namespace hale
