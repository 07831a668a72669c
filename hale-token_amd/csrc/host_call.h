// host_call.h -- what the C entry points of the host runtime have in common:
// checks of HIP calls, launches seen by the profiler, exceptions turned into
// statuses, and checks of types and addresses.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <new>

#include "context.h"

#define CALL_CHK(ctx, call)                                                                          \
  do {                                                                                               \
    hipError_t e_ = (call);                                                                          \
    if (e_ != hipSuccess)                                                                            \
      return hale::ctx_fail((ctx), HALE_EHIP, "%s failed: %s", #call, hipGetErrorString(e_));        \
  } while (0)

// Launches `call` (returning hipError_t) bracketed for the profiler.
#define CALL_LAUNCH(ctx, kind, call)  \
  do {                                \
    hale::ctx_prof_begin((ctx), (kind)); \
    hipError_t le_ = (call);          \
    hale::ctx_prof_end((ctx));        \
    CALL_CHK((ctx), le_);             \
  } while (0)

// No C++ exception leaves a C entry point.
#define CALL_TRY try {
#define CALL_CATCH(ctx)                                                                      \
  }                                                                                          \
  catch (const std::bad_alloc&) { return hale::ctx_fail((ctx), HALE_ENOMEM, "out of host memory"); } \
  catch (...) { return hale::ctx_fail((ctx), HALE_EHIP, "unexpected failure"); }

namespace hale {

inline bool float_type(int dtype) { return dtype == HALE_F32 || dtype == HALE_F16 || dtype == HALE_BF16; }
inline size_t type_bytes(int dtype) { return dtype == HALE_F32 ? 4 : 2; }
inline size_t round_up(size_t v, size_t a) { return (v + a - 1) / a * a; }
inline bool aligned(const void* p, int dtype) { return (uintptr_t)p % type_bytes(dtype) == 0; }

// Whether the context's stream is being captured.
inline int capturing(hale_ctx* c, bool* yes) {
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  CALL_CHK(c, hipStreamIsCapturing(c->stream, &st));
  *yes = st != hipStreamCaptureStatusNone;
  return HALE_OK;
}

}  // namespace hale
