// context.h -- the context and graph handles behind include/hale_moe.h, and
// what the host runtime's files share.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <mutex>
#include <string>
#include <vector>

#include "../../include/hale_moe.h"
#include "kernels.h"

using hale::K_KINDS;

namespace hale {

// One key/value cache that a captured graph stores to or attends over, or whose
// positions it rotates by.  A replay runs on the cache's step of that moment: its
// buffers must not have moved since, and for stores and attention it has to be a step
// of the same tokens per sequence.
struct KvUse {
  hale_kv_cache* kv;
  uint64_t serial;  // of the cache: its address may be another's by now
  uint64_t epoch;  // counts moves of the cache's buffers
  bool step;  // stores or attends
  uint64_t shape;  // what those calls' sizes follow from: tokens per sequence
};
// HALE_OK, or why the graph cannot be replayed now (kv.hip).
int kv_check_replay(hale_ctx* c, const std::vector<KvUse>& uses);

int ctx_fail(hale_ctx* c, int code, const char* fmt, ...);
// Brackets the kernels launched between them for the per-kernel profiler.
void ctx_prof_begin(hale_ctx* c, int kind);
void ctx_prof_end(hale_ctx* c);

}  // namespace hale

struct ProfRecord {
  int kind;
  hipEvent_t start, stop;
};

struct hale_ctx {
  int device = 0;
  hipStream_t stream = nullptr;
  std::recursive_mutex mu;
  std::string err;
  // scratch of the synchronous single-matrix / single-expert entry points
  void* scratch = nullptr;
  size_t scratch_bytes = 0;
  // wall timer
  hipEvent_t t0 = nullptr, t1 = nullptr;
  // per-kernel profiler
  bool prof_on = false;
  std::vector<hipEvent_t> ev_pool;
  std::vector<ProfRecord> recs;
  int open_kind = -1;
  bool prof_saved = false;  // prof_on while a capture runs (profiling is off then)
  double prof_ms[K_KINDS] = {};
  uint64_t prof_n[K_KINDS] = {};
  // Graphs keep the device addresses they were captured with.  While any
  // graph of this context exists, scratch that a call outgrows is retired
  // here instead of freed, so that replaying an older graph never touches
  // freed memory; the last hale_graph_destroy frees it.
  int live_graphs = 0;
  std::vector<void*> retired;
  // this device's copy of the fixed scratch array (forward without allocation)
  void* fixed_scratch = nullptr;
  // pinned host staging of the synchronous host-slice entry points: inputs
  // are copied in and outputs out of it by the CPU, the GPU copies from and
  // to it (every such call ends with a stream synchronize, so the next one
  // may reuse it)
  void* pinned = nullptr;
  size_t pinned_bytes = 0;
  std::vector<hale_kv_cache*> kvs;  // the context's key/value caches
  // key/value cache calls recorded by the capture in progress (see KvUse)
  std::vector<hale::KvUse> kv_uses;
};

namespace hale {

// Device memory that a call has outgrown: freed at once, or kept until the last
// graph of the context is destroyed when a graph may still use it.
inline void ctx_release(hale_ctx* c, void* p) {
  if (!p) return;
  if (c->live_graphs == 0) {
    (void)hipFree(p);
    return;
  }
  try {
    c->retired.push_back(p);
  } catch (...) {  // no room to remember it: it stays for good
  }
}

}  // namespace hale

struct hale_graph {
  hale_ctx* ctx = nullptr;
  hipGraph_t graph = nullptr;
  hipGraphExec_t exec = nullptr;
  std::vector<hale::KvUse> kv_uses;
};
