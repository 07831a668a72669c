// kv.hip -- host runtime of rotary positions and of the paged 8-bit key/value
// cache: handles, argument checks, the steps' plans and their way to the
// device.  Page bookkeeping is kv_pages.cpp, kernels are kernels_kv.hip and
// kernels_kv_attn.hip.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <memory>
#include <new>

#include "context.h"
#include "hale_device.h"
#include "kernels.h"
#include "kv.h"
#include "rope_freq.h"

using namespace hale;

#define KVCHK(ctx, call)                                                                       \
  do {                                                                                         \
    hipError_t e_ = (call);                                                                    \
    if (e_ != hipSuccess)                                                                      \
      return ctx_fail((ctx), HALE_EHIP, "%s failed: %s", #call, hipGetErrorString(e_));        \
  } while (0)

// Launches `call` (returning hipError_t) bracketed for the profiler.
#define KV_LAUNCH(ctx, kind, call)  \
  do {                              \
    ctx_prof_begin((ctx), (kind));  \
    hipError_t le_ = (call);        \
    ctx_prof_end((ctx));            \
    KVCHK((ctx), le_);              \
  } while (0)

// No C++ exception leaves a C entry point.
#define KV_TRY try {
#define KV_CATCH(ctx)                                                                  \
  }                                                                                    \
  catch (const std::bad_alloc&) { return ctx_fail((ctx), HALE_ENOMEM, "out of host memory"); } \
  catch (...) { return ctx_fail((ctx), HALE_EHIP, "unexpected failure"); }

static bool float_type(int dtype) { return dtype == HALE_F32 || dtype == HALE_F16 || dtype == HALE_BF16; }
static size_t type_bytes(int dtype) { return dtype == HALE_F32 ? 4 : 2; }
static size_t round_up(size_t v, size_t a) { return (v + a - 1) / a * a; }
static bool aligned(const void* p, int dtype) { return (uintptr_t)p % type_bytes(dtype) == 0; }

static int capturing(hale_ctx* c, bool* yes) {
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  KVCHK(c, hipStreamIsCapturing(c->stream, &st));
  *yes = st != hipStreamCaptureStatusNone;
  return HALE_OK;
}

// ---------------------------------------------------------------------------
// rotary positions
// ---------------------------------------------------------------------------

struct hale_rope {
  hale_ctx* ctx = nullptr;
  hale_rope_config config{};
  std::vector<double> freq;
  double* turns = nullptr;  // device: freq / 2 pi
};

extern "C" int hale_rope_create(hale_ctx* c, const hale_rope_config* config, hale_rope** out) {
  if (!c || !config || !out) return ctx_fail(c, HALE_EINVAL, "rope_create: NULL argument");
  *out = nullptr;
  KV_TRY
  std::vector<double> freq;
  std::string err;
  if (!rope_frequencies(*config, &freq, &err)) return ctx_fail(c, HALE_EINVAL, "rope: %s", err.c_str());
  std::vector<double> turns(freq.size());
  for (size_t i = 0; i < freq.size(); i++) turns[i] = freq[i] / (2.0 * M_PI);
  std::lock_guard<std::recursive_mutex> lk(c->mu);
  bool cap = false;
  KVCHK(c, hipSetDevice(c->device));
  const int rc = capturing(c, &cap);
  if (rc) return rc;
  if (cap) return ctx_fail(c, HALE_EINVAL, "rope_create while the stream is being captured");
  hale_rope* r = new hale_rope;
  r->ctx = c;
  r->config = *config;
  r->freq.swap(freq);
  hipError_t e = hipMalloc(&r->turns, turns.size() * 8);
  if (e == hipSuccess) e = hipMemcpyAsync(r->turns, turns.data(), turns.size() * 8, hipMemcpyHostToDevice, c->stream);
  if (e == hipSuccess) e = hipStreamSynchronize(c->stream);
  if (e != hipSuccess) {
    (void)hipFree(r->turns);
    delete r;
    return ctx_fail(c, HALE_ENOMEM, "rope tables: %s", hipGetErrorString(e));
  }
  *out = r;
  return HALE_OK;
  KV_CATCH(c)
}

extern "C" void hale_rope_destroy(hale_rope* r) {
  if (!r) return;
  hale_ctx* c = r->ctx;
  std::lock_guard<std::recursive_mutex> lk(c->mu);
  (void)hipSetDevice(c->device);
  (void)hipStreamSynchronize(c->stream);
  (void)hipFree(r->turns);
  delete r;
}

extern "C" int hale_rope_frequencies(const hale_rope* r, double* freq, size_t n) {
  if (!r || !freq) return ctx_fail(r ? r->ctx : nullptr, HALE_EINVAL, "rope_frequencies: NULL argument");
  if (n != r->freq.size())
    return ctx_fail(r->ctx, HALE_EINVAL, "rope_frequencies: %zu frequencies, not %zu", r->freq.size(), n);
  std::memcpy(freq, r->freq.data(), n * sizeof(double));
  return HALE_OK;
}

// Notes a captured rotation whose positions are those of a cache's step.
static int note_positions(hale_ctx* c, const int32_t* pos);

extern "C" int hale_rope_device(hale_rope* r, int dtype, size_t rows, const int32_t* pos, const void* q,
                                size_t q_heads, size_t q_stride, void* q_out, size_t q_out_stride, const void* k,
                                size_t k_heads, size_t k_stride, void* k_out, size_t k_out_stride) {
  if (!r) return ctx_fail(nullptr, HALE_EINVAL, "rope: NULL argument");
  hale_ctx* c = r->ctx;
  if (!float_type(dtype)) return ctx_fail(c, HALE_EINVAL, "rope: dtype %d is not f32, f16 or bf16", dtype);
  if (q_heads > 65536 || k_heads > 65536 || rows >= (1ull << 31))
    return ctx_fail(c, HALE_EINVAL, "rope: %zu rows of %zu and %zu heads", rows, q_heads, k_heads);
  if (rows == 0 || q_heads + k_heads == 0) return HALE_OK;
  if (!pos || (uintptr_t)pos % 4) return ctx_fail(c, HALE_EINVAL, "rope: positions are NULL or not aligned");
  RopeArgs a{};
  const void* src[2] = {q, k};
  void* dst[2] = {q_out, k_out};
  const size_t heads[2] = {q_heads, k_heads}, in[2] = {q_stride, k_stride}, out[2] = {q_out_stride, k_out_stride};
  const size_t hd = r->config.head_dim;
  for (int i = 0; i < 2; i++) {
    a.heads[i] = (int)heads[i];
    if (!heads[i]) continue;
    if (!src[i] || !dst[i]) return ctx_fail(c, HALE_EINVAL, "rope: NULL argument");
    if (in[i] < heads[i] * hd || out[i] < heads[i] * hd)
      return ctx_fail(c, HALE_EINVAL, "rope: strides %zu and %zu below %zu heads of %zu", in[i], out[i], heads[i], hd);
    if (!aligned(src[i], dtype) || !aligned(dst[i], dtype)) return ctx_fail(c, HALE_EINVAL, "rope: not aligned to its type");
    if (src[i] == dst[i] && in[i] != out[i] && rows > 1)
      return ctx_fail(c, HALE_EINVAL, "rope: in place with different strides");
    a.src[i] = src[i];
    a.dst[i] = dst[i];
    a.src_stride[i] = in[i];
    a.dst_stride[i] = out[i];
  }
  a.pos = pos;
  a.turns = r->turns;
  a.rows = rows;
  a.hd = (int)hd;
  a.half = (int)(r->config.rotary_dim / 2);
  a.interleaved = r->config.layout == HALE_ROPE_INTERLEAVED;
  a.factor = (float)r->config.attention_factor;
  KV_TRY
  std::lock_guard<std::recursive_mutex> lk(c->mu);
  KVCHK(c, hipSetDevice(c->device));
  const int rc = note_positions(c, pos);
  if (rc) return rc;
  KV_LAUNCH(c, K_ROPE, launch_rope(dtype, a, c->stream));
  return HALE_OK;
  KV_CATCH(c)
}

// ---------------------------------------------------------------------------
// the cache
// ---------------------------------------------------------------------------

namespace {

// Pinned host memory that the device reads plans from: a ring of buffers, one
// per upload.  Upload n, when it runs, reports that upload n - 1 has been read,
// so a buffer's next use waits (for the stream) only where the host is a whole
// ring ahead.
struct Staging {
  char* base = nullptr;
  size_t bytes = 0;
  uint32_t number = 0;  // the upload that read it last
};
constexpr int STAGINGS = 32;

struct View {  // the plan of the current step under one window, for f32 or the half types
  size_t window = 0;
  bool f32 = false;
  KvPlan plan;
  KvPlan next;  // of the step that is being put together
};

// Sections of the plan's device buffer, in 32-bit words (multiples of four).
// Their places hold until the buffer grows, so captured kernels keep them.
struct Sections {
  size_t counts = 0, positions = 0, blocks = 0, items[KV_MAX_VIEWS] = {},  // few, `many` words on many
         many = 0, joins[KV_MAX_VIEWS] = {},                         // likewise
         many_joins = 0, words = 0;
};
constexpr size_t COUNT_WORDS = 4 + 4 * KV_MAX_VIEWS;  // blocks; then few, many and their joins per view

}  // namespace

struct hale_kv_cache {
  hale_ctx* ctx = nullptr;
  uint64_t serial = 0, epoch = 0;
  KvShape shape{};
  size_t layers = 0;
  KvPages pages;
  KvGeom geom{};
  uint32_t* table = nullptr;
  uint32_t* plan = nullptr;
  Sections at;
  size_t cap_tokens = 0;
  float* part_o = nullptr;
  float2* part_ml = nullptr;
  Staging staging[STAGINGS];
  uint32_t uploads = 0;       // so far
  uint32_t* done = nullptr;   // pinned: the last upload known to have been read
  // the current step
  bool stepped = false;
  size_t tokens = 0, blocks = 0;
  uint64_t step_shape = 0;
  std::vector<KvStepSeq> seqs;
  std::vector<KvCopy> copies;  // pages that the next upload copies
  View views[KV_MAX_VIEWS];
  int nviews = 0;
};

static uint64_t g_kv_serial = 0;
static std::mutex g_kv_serial_mu;

// One upload being put together in pinned memory: pieces for the plan's
// sections, the list of page copies and the page table's changes.
namespace {

struct Upload {
  hale_kv_cache* kv;
  Staging* s = nullptr;
  KvUploadArgs a{};
  size_t used = 0;
  bool refused = false;  // a piece that there is no room for
  explicit Upload(hale_kv_cache* k) : kv(k) {}

  int begin(size_t bytes) {
    hale_ctx* c = kv->ctx;
    s = &kv->staging[kv->uploads % STAGINGS];
    if (s->number && (int32_t)(__atomic_load_n(kv->done, __ATOMIC_ACQUIRE) - s->number) < 0)
      KVCHK(c, hipStreamSynchronize(c->stream));
    s->number = 0;
    if (s->bytes < bytes) {
      if (s->base) (void)hipHostFree(s->base);
      s->base = nullptr;
      s->bytes = 0;
      const size_t want = round_up(bytes * 2, 65536);
      if (hipHostMalloc(&s->base, want, hipHostMallocDefault) != hipSuccess) {
        s->base = nullptr;
        return ctx_fail(c, HALE_ENOMEM, "pinned staging of %zu bytes", want);
      }
      s->bytes = want;
    }
    return HALE_OK;
  }
  // bytes that go to dst, as a piece of whole quads of words
  void put(void* dst, const void* src, size_t bytes) {
    const size_t words = round_up(bytes, 16) / 4;
    if (!words) return;
    if (a.pieces == KV_MAX_PIECES || used + words * 4 > s->bytes) {
      refused = true;
      return;
    }
    char* p = s->base + used;
    std::memcpy(p, src, bytes);
    std::memset(p + bytes, 0, words * 4 - bytes);
    a.dst[a.pieces] = (uint32_t*)dst;
    a.words[a.pieces++] = (unsigned)words;
    used += words * 4;
  }
  int end() {
    hale_ctx* c = kv->ctx;
    auto& dirty = kv->pages.dirty;
    if (refused) return ctx_fail(c, HALE_EHIP, "kv: a plan of more than %d pieces", KV_MAX_PIECES);
    uint32_t* pairs = (uint32_t*)(s->base + used);
    for (size_t i = 0; i < dirty.size(); i++) {
      pairs[2 * i] = dirty[i];
      pairs[2 * i + 1] = kv->pages.entry(dirty[i]);
    }
    KvCopy* copies = (KvCopy*)(pairs + 2 * dirty.size());
    if (!kv->copies.empty()) std::memcpy(copies, kv->copies.data(), kv->copies.size() * sizeof(KvCopy));
    a.src = (const uint32_t*)s->base;
    a.pairs = pairs;
    a.npairs = (unsigned)dirty.size();
    a.table = kv->table;
    a.copies = copies;
    a.ncopies = (unsigned)kv->copies.size();
    a.pool = kv->geom.pool;
    a.page_bytes = kv->geom.page_bytes;
    a.done = kv->done;
    a.number = kv->uploads++;  // from the first one's 0 on: numbers count from 1
    KV_LAUNCH(c, K_KV_PAGES, launch_kv_upload(a, c->stream));
    s->number = kv->uploads;
    dirty.clear();
    kv->copies.clear();
    return HALE_OK;
  }
};

}  // namespace

// Bytes of an upload: its pieces, each rounded up, the table's changes and the copies.
static size_t upload_bytes(const hale_kv_cache* kv, size_t piece_bytes) {
  return piece_bytes + 16 * KV_MAX_PIECES + kv->pages.dirty.size() * 8 + kv->copies.size() * sizeof(KvCopy);
}

// Sends the page table's changes and makes the page copies of kv->copies.
static int send_pages(hale_kv_cache* kv) {
  if (kv->pages.dirty.empty() && kv->copies.empty()) return HALE_OK;
  Upload u(kv);
  const int rc = u.begin(upload_bytes(kv, 0));
  return rc ? rc : u.end();
}

static void free_device(hale_kv_cache* kv) {
  for (void* p : {(void*)kv->geom.pool, (void*)kv->table, (void*)kv->part_o, (void*)kv->part_ml}) (void)hipFree(p);
  ctx_release(kv->ctx, kv->plan);
  for (Staging& s : kv->staging) {
    if (s.base) (void)hipHostFree(s.base);
  }
  if (kv->done) (void)hipHostFree(kv->done);
}

static Sections sections(const hale_kv_cache* kv, size_t tokens) {
  Sections s;
  const size_t n = kv->pages.max_seqs(), items = kv_max_items(kv->shape, tokens, n), joins = items - KV_MAX_PARTS;
  s.many = items * sizeof(KvItem) / 4;
  s.many_joins = joins * sizeof(KvJoin) / 4;
  size_t w = COUNT_WORDS;
  s.positions = w, w += round_up(tokens, 4);
  s.blocks = w, w += round_up(kv_max_blocks(tokens, n) * sizeof(KvBlock) / 4, 4);
  for (int v = 0; v < KV_MAX_VIEWS; v++) {
    s.items[v] = w, w += 2 * s.many;
    s.joins[v] = w, w += 2 * s.many_joins;
  }
  s.words = w;
  return s;
}

// Plan buffers for steps of `tokens` tokens.
static int grow_plan(hale_kv_cache* kv, size_t tokens) {
  if (kv->plan && tokens <= kv->cap_tokens) return HALE_OK;
  hale_ctx* c = kv->ctx;
  bool cap = false;
  const int rc = capturing(c, &cap);
  if (rc) return rc;
  if (cap) return ctx_fail(c, HALE_EINVAL, "kv: the plan must grow to %zu tokens while the stream is being captured", tokens);
  tokens = round_up(std::max(tokens, kv->cap_tokens * 2), 256);
  const Sections s = sections(kv, tokens);
  uint32_t* p = nullptr;
  KVCHK(c, hipStreamSynchronize(c->stream));
  if (hipMalloc(&p, s.words * 4) != hipSuccess)
    return ctx_fail(c, HALE_ENOMEM, "kv: plan buffers of %zu bytes", s.words * 4);
  ctx_release(c, kv->plan);  // a graph's rotation may read the positions in it
  kv->plan = p;
  kv->at = s;
  kv->cap_tokens = tokens;
  kv->epoch++;
  kv->stepped = false;
  return HALE_OK;
}

static int make_pool(hale_ctx* c, size_t page_bytes, size_t pages, uint8_t** out) {
  *out = nullptr;
  if (pages > (SIZE_MAX >> 8) / page_bytes)  // the product would wrap
    return ctx_fail(c, HALE_ENOMEM, "kv: a pool of %zu pages of %zu bytes", pages, page_bytes);
  const size_t bytes = page_bytes * pages;
  if (hipMalloc(out, bytes) != hipSuccess) {
    *out = nullptr;
    return ctx_fail(c, HALE_ENOMEM, "kv: a pool of %zu bytes", bytes);
  }
  // padded key numbers and positions never stored are code -128, scale 0: finite
  hipError_t e = hipMemsetAsync(*out, 0, bytes, c->stream);
  if (e == hipSuccess) e = hipStreamSynchronize(c->stream);
  if (e != hipSuccess) {
    (void)hipFree(*out);
    *out = nullptr;
    return ctx_fail(c, HALE_EHIP, "kv: clearing the pool: %s", hipGetErrorString(e));
  }
  return HALE_OK;
}

extern "C" int hale_kv_create(hale_ctx* c, size_t layers, size_t heads, size_t kv_heads, size_t hd, size_t num_pages,
                              size_t max_seqs, size_t max_len, hale_kv_cache** out) {
  if (!c || !out) return ctx_fail(c, HALE_EINVAL, "kv_create: NULL argument");
  *out = nullptr;
  if (layers == 0 || layers > 4096) return ctx_fail(c, HALE_EINVAL, "kv_create: %zu layers outside 1..4096", layers);
  if (kv_heads == 0 || heads == 0 || heads % kv_heads || heads > 4096)
    return ctx_fail(c, HALE_EINVAL, "kv_create: num_heads %zu must be a positive multiple of num_kv_heads %zu, at most 4096", heads, kv_heads);
  if (hd < 16 || hd > 256 || hd % 16)
    return ctx_fail(c, HALE_EINVAL, "kv_create: head_dim %zu must be a multiple of 16 in 16..256", hd);
  if (num_pages == 0 || num_pages > (1u << 30)) return ctx_fail(c, HALE_EINVAL, "kv_create: %zu pages outside 1..2^30", num_pages);
  if (max_seqs == 0 || max_seqs > 65536) return ctx_fail(c, HALE_EINVAL, "kv_create: max_seqs %zu outside 1..65536", max_seqs);
  if (max_len == 0 || max_len > (1u << 30)) return ctx_fail(c, HALE_EINVAL, "kv_create: max_len %zu outside 1..2^30", max_len);
  const size_t row = (max_len + KV_PAGE - 1) / KV_PAGE;
  if (row * max_seqs > (1u << 30))
    return ctx_fail(c, HALE_EINVAL, "kv_create: a page table of %zu sequences x %zu pages", max_seqs, row);
  hale_kv_cache* kv = nullptr;
  KV_TRY
  std::lock_guard<std::recursive_mutex> lk(c->mu);
  KVCHK(c, hipSetDevice(c->device));
  bool cap = false;
  int rc = capturing(c, &cap);
  if (rc) return rc;
  if (cap) return ctx_fail(c, HALE_EINVAL, "kv_create while the stream is being captured");
  c->kvs.reserve(c->kvs.size() + 1);
  std::unique_ptr<hale_kv_cache> own(new hale_kv_cache);
  kv = own.get();
  kv->ctx = c;
  {
    std::lock_guard<std::mutex> g(g_kv_serial_mu);
    kv->serial = ++g_kv_serial;
  }
  kv->shape = {heads, kv_heads, hd};
  kv->layers = layers;
  kv->pages.init(num_pages, max_seqs, max_len);
  KvGeom& g = kv->geom;
  g.chunks = kv_chunks(hd);
  g.hd = (int)hd;
  g.kv_heads = (int)kv_heads;
  g.group = (int)(heads / kv_heads);
  g.v_off = (unsigned)(KV_PAGE * 32 * g.chunks);
  g.s_off = g.v_off + (unsigned)(KV_PAGE * hd);
  g.head_bytes = g.s_off + 128;  // eight scales, the region a multiple of a line
  g.layer_bytes = (size_t)g.head_bytes * kv_heads;
  g.page_bytes = g.layer_bytes * layers;
  g.max_pages = (unsigned)row;
  rc = make_pool(c, g.page_bytes, num_pages, &g.pool);
  const size_t part_rows = kv_part_rows(hd);
  if (!rc && (hipMalloc(&kv->table, row * max_seqs * 4) != hipSuccess ||
              hipMalloc(&kv->part_o, part_rows * hd * 4) != hipSuccess ||
              hipMalloc(&kv->part_ml, part_rows * sizeof(float2)) != hipSuccess))
    rc = ctx_fail(c, HALE_ENOMEM, "kv_create: page table and workspace");
  if (!rc && hipHostMalloc(&kv->done, 64, hipHostMallocDefault) != hipSuccess) {
    kv->done = nullptr;
    rc = ctx_fail(c, HALE_ENOMEM, "kv_create: pinned memory");
  }
  if (!rc) *kv->done = 0;
  if (!rc && (hipMemsetAsync(kv->table, 0, row * max_seqs * 4, c->stream) != hipSuccess ||
              hipStreamSynchronize(c->stream) != hipSuccess))
    rc = ctx_fail(c, HALE_EHIP, "kv_create: clearing the page table");
  if (!rc) rc = grow_plan(kv, std::max<size_t>(max_seqs, 256));
  if (rc) {
    free_device(kv);
    return rc;
  }
  g.table = kv->table;
  c->kvs.push_back(kv);
  *out = own.release();
  return HALE_OK;
  KV_CATCH(c)
}

extern "C" void hale_kv_destroy(hale_kv_cache* kv) {
  if (!kv) return;
  hale_ctx* c = kv->ctx;
  std::lock_guard<std::recursive_mutex> lk(c->mu);
  (void)hipSetDevice(c->device);
  (void)hipStreamSynchronize(c->stream);
  free_device(kv);
  c->kvs.erase(std::remove(c->kvs.begin(), c->kvs.end(), kv), c->kvs.end());
  delete kv;
}

static int status(hale_kv_cache* kv, const char* what, KvPages::Status st, const std::string& err) {
  if (st == KvPages::OK) return HALE_OK;
  return ctx_fail(kv->ctx, st == KvPages::FULL ? HALE_ENOMEM : HALE_EINVAL, "%s: %s", what, err.c_str());
}

// A sequence whose positions went away is no longer part of the step.
static void leaves_step(hale_kv_cache* kv, uint32_t seq) {
  for (const KvStepSeq& s : kv->seqs)
    if (s.row == seq) kv->stepped = false;
}

extern "C" int hale_kv_seq_create(hale_kv_cache* kv, uint32_t* seq) {
  if (!kv || !seq) return ctx_fail(kv ? kv->ctx : nullptr, HALE_EINVAL, "kv_seq_create: NULL argument");
  KV_TRY
  std::lock_guard<std::recursive_mutex> lk(kv->ctx->mu);
  std::string err;
  return status(kv, "kv_seq_create", kv->pages.create(seq, &err), err);
  KV_CATCH(kv->ctx)
}

extern "C" int hale_kv_seq_free(hale_kv_cache* kv, uint32_t seq) {
  if (!kv) return ctx_fail(nullptr, HALE_EINVAL, "kv_seq_free: NULL argument");
  KV_TRY
  std::lock_guard<std::recursive_mutex> lk(kv->ctx->mu);
  std::string err;
  const int rc = status(kv, "kv_seq_free", kv->pages.free(seq, &err), err);
  if (!rc) leaves_step(kv, seq);
  return rc;
  KV_CATCH(kv->ctx)
}

extern "C" int hale_kv_seq_fork(hale_kv_cache* kv, uint32_t seq, size_t n, uint32_t* out) {
  if (!kv || (n && !out)) return ctx_fail(kv ? kv->ctx : nullptr, HALE_EINVAL, "kv_seq_fork: NULL argument");
  KV_TRY
  std::lock_guard<std::recursive_mutex> lk(kv->ctx->mu);
  std::string err;
  return status(kv, "kv_seq_fork", kv->pages.fork(seq, n, out, &err), err);
  KV_CATCH(kv->ctx)
}

// Page moves are enqueued at once, in the order of the calls: not while the
// stream is being captured, where they would run at the replay.
static int moves_allowed(hale_kv_cache* kv, const char* what) {
  KVCHK(kv->ctx, hipSetDevice(kv->ctx->device));
  bool cap = false;
  const int rc = capturing(kv->ctx, &cap);
  if (rc) return rc;
  if (cap) return ctx_fail(kv->ctx, HALE_EINVAL, "%s while the stream is being captured", what);
  return kv->copies.empty() ? HALE_OK : send_pages(kv);  // copies whose launch failed
}

extern "C" int hale_kv_seq_copy(hale_kv_cache* kv, uint32_t seq, uint32_t* out) {
  if (!kv || !out) return ctx_fail(kv ? kv->ctx : nullptr, HALE_EINVAL, "kv_seq_copy: NULL argument");
  KV_TRY
  std::lock_guard<std::recursive_mutex> lk(kv->ctx->mu);
  int rc = moves_allowed(kv, "kv_seq_copy");
  if (rc) return rc;
  std::string err;
  size_t len = 0;
  rc = status(kv, "kv_seq_copy", kv->pages.len(seq, &len, &err), err);
  if (rc) return rc;
  Upload u(kv);  // its memory before the sequence
  rc = u.begin(upload_bytes(kv, (len + KV_PAGE - 1) / KV_PAGE * (8 + sizeof(KvCopy))));
  if (!rc) rc = status(kv, "kv_seq_copy", kv->pages.copy(seq, out, &kv->copies, &err), err);
  return rc ? rc : u.end();
  KV_CATCH(kv->ctx)
}

extern "C" int hale_kv_seq_truncate(hale_kv_cache* kv, uint32_t seq, size_t len) {
  if (!kv) return ctx_fail(nullptr, HALE_EINVAL, "kv_seq_truncate: NULL argument");
  KV_TRY
  std::lock_guard<std::recursive_mutex> lk(kv->ctx->mu);
  std::string err;
  const int rc = status(kv, "kv_seq_truncate", kv->pages.truncate(seq, len, &err), err);
  if (!rc) leaves_step(kv, seq);
  return rc;
  KV_CATCH(kv->ctx)
}

extern "C" int hale_kv_seq_len(const hale_kv_cache* kv, uint32_t seq, size_t* len) {
  if (!kv || !len) return ctx_fail(kv ? kv->ctx : nullptr, HALE_EINVAL, "kv_seq_len: NULL argument");
  KV_TRY
  std::lock_guard<std::recursive_mutex> lk(kv->ctx->mu);
  std::string err;
  return status(const_cast<hale_kv_cache*>(kv), "kv_seq_len", kv->pages.len(seq, len, &err), err);
  KV_CATCH(kv->ctx)
}

extern "C" int hale_kv_pages(const hale_kv_cache* kv, size_t* total, size_t* used) {
  if (!kv) return ctx_fail(nullptr, HALE_EINVAL, "kv_pages: NULL argument");
  std::lock_guard<std::recursive_mutex> lk(kv->ctx->mu);
  if (total) *total = kv->pages.pages();
  if (used) *used = kv->pages.used();
  return HALE_OK;
}

extern "C" int hale_kv_compact(hale_kv_cache* kv, size_t* moved) {
  if (!kv) return ctx_fail(nullptr, HALE_EINVAL, "kv_compact: NULL argument");
  KV_TRY
  std::lock_guard<std::recursive_mutex> lk(kv->ctx->mu);
  int rc = moves_allowed(kv, "kv_compact");
  if (rc) return rc;
  size_t pages = 0, entries = 0;
  kv->pages.compact_size(&pages, &entries);
  Upload u(kv);  // its memory before the moves
  rc = u.begin(upload_bytes(kv, pages * sizeof(KvCopy) + entries * 8));
  if (rc) return rc;
  kv->pages.compact(&kv->copies);
  if (moved) *moved = pages;
  return pages || !kv->pages.dirty.empty() ? u.end() : HALE_OK;
  KV_CATCH(kv->ctx)
}

extern "C" int hale_kv_resize(hale_kv_cache* kv, size_t num_pages) {
  if (!kv) return ctx_fail(nullptr, HALE_EINVAL, "kv_resize: NULL argument");
  hale_ctx* c = kv->ctx;
  KV_TRY
  std::lock_guard<std::recursive_mutex> lk(c->mu);
  int rc = moves_allowed(kv, "kv_resize");
  if (rc) return rc;
  if (c->live_graphs) return ctx_fail(c, HALE_EINVAL, "kv_resize: %d graphs of the context hold the pool's address", c->live_graphs);
  const size_t used = kv->pages.used();
  if (num_pages < used || num_pages == 0 || num_pages > (1u << 30))
    return ctx_fail(c, HALE_EINVAL, "kv_resize: %zu pages, but %zu are in use", num_pages, used);
  rc = hale_kv_compact(kv, nullptr);
  if (rc) return rc;
  uint8_t* pool = nullptr;
  rc = make_pool(c, kv->geom.page_bytes, num_pages, &pool);
  if (rc) return rc;
  hipError_t e = hipSuccess;
  if (used) e = launch_copy(pool, kv->geom.pool, used * kv->geom.page_bytes / 16, c->stream);
  if (e == hipSuccess) e = hipStreamSynchronize(c->stream);
  if (e == hipSuccess) {
    try {
      kv->pages.resize(num_pages);
    } catch (...) {
      e = hipErrorOutOfMemory;
    }
  }
  if (e != hipSuccess) {
    (void)hipFree(pool);
    return ctx_fail(c, HALE_ENOMEM, "kv_resize: %s", hipGetErrorString(e));
  }
  (void)hipFree(kv->geom.pool);
  kv->geom.pool = pool;
  kv->epoch++;
  return HALE_OK;
  KV_CATCH(c)
}

// ---------------------------------------------------------------------------
// steps
// ---------------------------------------------------------------------------

static size_t plan_bytes(const KvPlan& p) {
  return (p.few.size() + p.many.size()) * sizeof(KvItem) + (p.few_joins.size() + p.many_joins.size()) * sizeof(KvJoin) + 32;
}
static void put_view(hale_kv_cache* kv, Upload& u, int i) {
  View& v = kv->views[i];
  const uint32_t n[4] = {(uint32_t)v.plan.few.size(), (uint32_t)v.plan.many.size(), (uint32_t)v.plan.few_joins.size(),
                         (uint32_t)v.plan.many_joins.size()};
  u.put(kv->plan + kv->at.counts + 4 + 4 * i, n, sizeof n);
  u.put(kv->plan + kv->at.items[i], v.plan.few.data(), v.plan.few.size() * sizeof(KvItem));
  u.put(kv->plan + kv->at.items[i] + kv->at.many, v.plan.many.data(), v.plan.many.size() * sizeof(KvItem));
  u.put(kv->plan + kv->at.joins[i], v.plan.few_joins.data(), v.plan.few_joins.size() * sizeof(KvJoin));
  u.put(kv->plan + kv->at.joins[i] + kv->at.many_joins, v.plan.many_joins.data(), v.plan.many_joins.size() * sizeof(KvJoin));
}

extern "C" int hale_kv_reserve(hale_kv_cache* kv, size_t max_tokens) {
  if (!kv) return ctx_fail(nullptr, HALE_EINVAL, "kv_reserve: NULL argument");
  hale_ctx* c = kv->ctx;
  KV_TRY
  std::lock_guard<std::recursive_mutex> lk(c->mu);
  KVCHK(c, hipSetDevice(c->device));
  if (max_tokens > (size_t)0x7fffffff / kv->shape.heads)
    return ctx_fail(c, HALE_EINVAL, "kv_reserve: %zu tokens of %zu heads", max_tokens, kv->shape.heads);
  return grow_plan(kv, max_tokens);
  KV_CATCH(c)
}

extern "C" int hale_kv_step(hale_kv_cache* kv, size_t nseq, const uint32_t* seqs, const uint32_t* ntok) {
  if (!kv || (nseq && (!seqs || !ntok))) return ctx_fail(kv ? kv->ctx : nullptr, HALE_EINVAL, "kv_step: NULL argument");
  hale_ctx* c = kv->ctx;
  KV_TRY
  std::lock_guard<std::recursive_mutex> lk(c->mu);
  int rc = moves_allowed(kv, "kv_step");
  if (rc) return rc;
  if (nseq > kv->pages.max_seqs()) return ctx_fail(c, HALE_EINVAL, "kv_step: %zu sequences, at most %zu", nseq, kv->pages.max_seqs());
  size_t tokens = 0;
  for (size_t i = 0; i < nseq; i++) tokens += ntok[i];
  if (tokens > (size_t)0x7fffffff / kv->shape.heads)
    return ctx_fail(c, HALE_EINVAL, "kv_step: %zu tokens of %zu heads", tokens, kv->shape.heads);
  std::string err;
  rc = status(kv, "kv_step", kv->pages.check_step(nseq, seqs, ntok, &err), err);
  if (rc) return rc;
  // all that may run out of memory first: until then the current step stands
  std::vector<KvStepSeq> next;
  std::vector<KvBlock> blocks;
  blocks.reserve(kv_max_blocks(tokens, nseq));
  std::vector<int32_t> positions(tokens);
  kv->pages.preview(nseq, seqs, ntok, &next);
  kv_blocks(next, kv->pages.max_pages(), &blocks);
  uint64_t shape = 1469598103934665603ull;  // FNV-1a over the tokens per sequence
  auto mix = [&](uint32_t v) {
    for (int b = 0; b < 4; b++) shape = (shape ^ (v >> (8 * b) & 255)) * 1099511628211ull;
  };
  mix((uint32_t)nseq);
  for (const KvStepSeq& s : next) {
    mix(s.ntok);
    for (uint32_t t = 0; t < s.ntok; t++) positions[s.tok0 + t] = (int32_t)(s.len0 + t);
  }
  kv->pages.reserve_step(nseq, seqs, ntok, &kv->copies);
  size_t bytes = tokens * 4 + blocks.size() * sizeof(KvBlock) + 64;
  bytes += kv->pages.step_changes() * 8 + kv->pages.step_copies() * sizeof(KvCopy);
  for (int i = 0; i < kv->nviews; i++) {
    kv_plan(kv->shape, next, kv->views[i].window, kv->views[i].f32, &kv->views[i].next);
    bytes += plan_bytes(kv->views[i].next);
  }
  Upload u(kv);
  rc = u.begin(upload_bytes(kv, bytes));
  if (!rc) rc = grow_plan(kv, tokens);
  if (rc) return rc;
  kv->stepped = false;
  kv->seqs.swap(next);
  for (int i = 0; i < kv->nviews; i++) std::swap(kv->views[i].plan, kv->views[i].next);
  const uint32_t n[4] = {(uint32_t)blocks.size(), (uint32_t)tokens, 0, 0};
  u.put(kv->plan + kv->at.counts, n, sizeof n);
  u.put(kv->plan + kv->at.positions, positions.data(), tokens * 4);
  u.put(kv->plan + kv->at.blocks, blocks.data(), blocks.size() * sizeof(KvBlock));
  for (int i = 0; i < kv->nviews; i++) put_view(kv, u, i);
  rc = status(kv, "kv_step", kv->pages.step(nseq, seqs, ntok, nullptr, &kv->copies, &err), err);
  if (!rc) rc = u.end();
  if (rc) return rc;
  kv->tokens = tokens;
  kv->step_shape = shape;
  kv->blocks = blocks.size();
  kv->stepped = true;
  return HALE_OK;
  KV_CATCH(c)
}

extern "C" int hale_kv_positions(const hale_kv_cache* kv, const int32_t** out) {
  if (!kv || !out) return ctx_fail(kv ? kv->ctx : nullptr, HALE_EINVAL, "kv_positions: NULL argument");
  std::lock_guard<std::recursive_mutex> lk(kv->ctx->mu);
  *out = (const int32_t*)(kv->plan + kv->at.positions);
  return HALE_OK;
}

// What append and attention have in common: the step's state, and whether the
// call is being captured (then it is noted for the graph).
static int layer_call(hale_kv_cache* kv, const char* what, size_t layer, int dtype, size_t ntok, bool* cap) {
  hale_ctx* c = kv->ctx;
  if (layer >= kv->layers) return ctx_fail(c, HALE_EINVAL, "%s: layer %zu of %zu", what, layer, kv->layers);
  if (!float_type(dtype)) return ctx_fail(c, HALE_EINVAL, "%s: dtype %d is not f32, f16 or bf16", what, dtype);
  if (!kv->stepped) return ctx_fail(c, HALE_EINVAL, "%s without a current step", what);
  if (ntok != kv->tokens) return ctx_fail(c, HALE_EINVAL, "%s: %zu tokens, but the step has %zu", what, ntok, kv->tokens);
  KVCHK(c, hipSetDevice(c->device));
  int rc = capturing(c, cap);
  if (rc) return rc;
  if (!*cap) return send_pages(kv);  // table changes since the step
  for (KvUse& u : c->kv_uses) {
    if (u.kv != kv) continue;
    if (u.epoch != kv->epoch || (u.step && u.shape != kv->step_shape))
      return ctx_fail(c, HALE_EINVAL, "%s: the graph holds calls for another step of this cache", what);
    u.step = true;
    u.shape = kv->step_shape;
    return HALE_OK;
  }
  c->kv_uses.push_back({kv, kv->serial, kv->epoch, true, kv->step_shape});
  return HALE_OK;
}

static int note_positions(hale_ctx* c, const int32_t* pos) {
  for (hale_kv_cache* kv : c->kvs) {
    const uintptr_t at = (uintptr_t)pos, first = (uintptr_t)(kv->plan + kv->at.positions);
    if (at < first || at >= first + 4 * kv->cap_tokens) continue;
    bool cap = false;
    const int rc = capturing(c, &cap);
    if (rc || !cap) return rc;
    for (const KvUse& u : c->kv_uses)
      if (u.kv == kv) return HALE_OK;
    c->kv_uses.push_back({kv, kv->serial, kv->epoch, false, 0});
    return HALE_OK;
  }
  return HALE_OK;
}

int hale::kv_check_replay(hale_ctx* c, const std::vector<KvUse>& uses) {
  KVCHK(c, hipSetDevice(c->device));
  bool cap = false;
  int rc = capturing(c, &cap);
  if (rc) return rc;
  if (cap) return ctx_fail(c, HALE_EINVAL, "graph_launch of a key/value cache's graph while the stream is being captured");
  for (const KvUse& u : uses) {
    if (std::find(c->kvs.begin(), c->kvs.end(), u.kv) == c->kvs.end() || u.kv->serial != u.serial)
      return ctx_fail(c, HALE_EINVAL, "graph_launch: its key/value cache is gone");
    if (u.kv->epoch != u.epoch)
      return ctx_fail(c, HALE_EINVAL, "graph_launch: its key/value cache's buffers grew since the capture");
    if (!u.step) continue;
    if (!u.kv->stepped || u.kv->step_shape != u.shape)
      return ctx_fail(c, HALE_EINVAL, "graph_launch: the key/value cache's step is not of the captured tokens per sequence");
    rc = send_pages(u.kv);
    if (rc) return rc;
  }
  return HALE_OK;
}

extern "C" int hale_kv_append_device(hale_kv_cache* kv, size_t layer, int dtype, size_t ntok, const void* k,
                                     size_t k_stride, const void* v, size_t v_stride) {
  if (!kv) return ctx_fail(nullptr, HALE_EINVAL, "kv_append: NULL argument");
  hale_ctx* c = kv->ctx;
  KV_TRY
  std::lock_guard<std::recursive_mutex> lk(c->mu);
  if (float_type(dtype) && ntok) {
    const size_t row = kv->shape.kv_heads * kv->shape.head_dim;
    if (!k || !v) return ctx_fail(c, HALE_EINVAL, "kv_append: NULL argument");
    if (k_stride < row || v_stride < row)
      return ctx_fail(c, HALE_EINVAL, "kv_append: strides %zu and %zu below %zu", k_stride, v_stride, row);
    if (!aligned(k, dtype) || !aligned(v, dtype)) return ctx_fail(c, HALE_EINVAL, "kv_append: not aligned to its type");
  }
  bool cap = false;
  int rc = layer_call(kv, "kv_append", layer, dtype, ntok, &cap);
  if (rc || ntok == 0) return rc;
  KvAppendArgs a{};
  a.g = kv->geom;
  a.layer = layer;
  a.blocks = (const KvBlock*)(kv->plan + kv->at.blocks);
  a.count = cap ? kv->plan + kv->at.counts : nullptr;
  a.nblocks = (unsigned)kv->blocks;
  a.k = k;
  a.v = v;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  const size_t both = (uintptr_t)k | (uintptr_t)v | k_stride * type_bytes(dtype) | v_stride * type_bytes(dtype);
  a.vec = both % 16 == 0;  // head_dim is a multiple of 16
  // later steps of these tokens may touch one block more per sequence
  const size_t grid = cap ? kv_max_blocks(ntok, kv->seqs.size()) : kv->blocks;
  KV_LAUNCH(c, K_KV_STORE, launch_kv_append(dtype, a, (unsigned)grid, c->stream));
  return HALE_OK;
  KV_CATCH(c)
}

extern "C" int hale_kv_attention_device(hale_kv_cache* kv, size_t layer, int dtype, size_t ntok, const void* q,
                                        size_t q_stride, float scale, size_t window, void* out, size_t out_stride) {
  if (!kv) return ctx_fail(nullptr, HALE_EINVAL, "kv_attention: NULL argument");
  hale_ctx* c = kv->ctx;
  KV_TRY
  std::lock_guard<std::recursive_mutex> lk(c->mu);
  // scores are in powers of two: scale log2(e) has to be finite as well
  if (!(scale > 0.0f) || !std::isfinite(scale * 2.0f))
    return ctx_fail(c, HALE_EINVAL, "kv_attention: scale %g is not positive and below 2^127", (double)scale);
  if (float_type(dtype) && ntok) {
    const size_t row = kv->shape.heads * kv->shape.head_dim;
    if (!q || !out) return ctx_fail(c, HALE_EINVAL, "kv_attention: NULL argument");
    if (q_stride < row || out_stride < row)
      return ctx_fail(c, HALE_EINVAL, "kv_attention: strides %zu and %zu below %zu", q_stride, out_stride, row);
    if (!aligned(q, dtype) || !aligned(out, dtype)) return ctx_fail(c, HALE_EINVAL, "kv_attention: not aligned to its type");
  }
  bool cap = false;
  int rc = layer_call(kv, "kv_attention", layer, dtype, ntok, &cap);
  if (rc || ntok == 0) return rc;
  if (window >= kv->pages.max_len()) window = 0;  // sees everything
  int i = 0;
  const bool f32 = dtype == HALE_F32;
  while (i < kv->nviews && (kv->views[i].window != window || kv->views[i].f32 != f32)) i++;
  if (i == kv->nviews) {
    int windows = 0;  // others than this one
    for (int k = 0; k < i; k++) {
      bool counted = kv->views[k].window == window;
      for (int j = 0; j < k; j++) counted |= kv->views[j].window == kv->views[k].window;
      windows += !counted;
    }
    if (windows == HALE_KV_MAX_WINDOWS)
      return ctx_fail(c, HALE_EINVAL, "kv_attention: window %zu is a fifth one (at most %d)", window, HALE_KV_MAX_WINDOWS);
    if (cap) return ctx_fail(c, HALE_EINVAL, "kv_attention: first call with window %zu and this type in a capture; make it once before", window);
    View& v = kv->views[i];
    v.window = window;
    v.f32 = f32;
    kv_plan(kv->shape, kv->seqs, window, f32, &v.plan);
    Upload u(kv);
    rc = u.begin(upload_bytes(kv, plan_bytes(v.plan)));
    if (rc) return rc;
    put_view(kv, u, i);
    rc = u.end();
    if (rc) return rc;
    kv->nviews = i + 1;
  }
  const View& v = kv->views[i];
  KvAttnArgs a{};
  a.g = kv->geom;
  a.layer = layer;
  a.dtype = dtype;
  a.q = q;
  a.out = out;
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.scale = scale * 1.44269504088896340736f;
  a.window = (int)window;
  const KvItem* items = (const KvItem*)(kv->plan + kv->at.items[i]);
  const KvJoin* joins = (const KvJoin*)(kv->plan + kv->at.joins[i]);
  a.counts = kv->plan + kv->at.counts + 4 + 4 * i;
  a.part_o = kv->part_o;
  a.part_ml = kv->part_ml;
  const size_t quad = 4 * type_bytes(dtype);
  a.vec = (uintptr_t)q % quad == 0 && (uintptr_t)out % quad == 0 && q_stride % 4 == 0 && out_stride % 4 == 0;
  // captured: later steps of these tokens may have more items, which the
  // work-groups then take in turn, and joins of the same rows
  auto grid = [&](size_t now, size_t most) {
    return (unsigned)std::min<size_t>(cap && now ? std::max(now, std::min<size_t>(most, KV_FEW_GROUPS)) : now, 1u << 20);
  };
  const size_t tiles = kv_max_items(kv->shape, ntok, kv->seqs.size()) - KV_MAX_PARTS;
  const size_t limit = kv_few_limit(kv->shape, kv->seqs, f32);
  bool few = false, many = false;
  for (const KvStepSeq& s : kv->seqs) (s.ntok * kv->shape.group() <= limit ? few : many) |= s.ntok > 0;
  for (int kind = 0; kind < 2; kind++) {
    if (!(kind ? many : few)) continue;
    const size_t nitems = (kind ? v.plan.many : v.plan.few).size(), njoins = (kind ? v.plan.many_joins : v.plan.few_joins).size();
    a.kind = kind;
    a.items = kind ? items + kv->at.many * 4 / sizeof(KvItem) : items;
    a.joins = kind ? joins + kv->at.many_joins * 4 / sizeof(KvJoin) : joins;
    a.nitems = cap ? 0xffffffffu : (unsigned)nitems;
    a.njoins = cap ? 0xffffffffu : (unsigned)njoins;
    const unsigned gi = grid(nitems, tiles + KV_MAX_PARTS), gj = cap ? (unsigned)std::min<size_t>(tiles, 256) : grid(njoins, 0);
    const unsigned rows = kind ? (unsigned)kv_many_rows(kv->shape.head_dim) : 16u * v.plan.cols;
    KV_LAUNCH(c, K_KV_ATTENTION, kind ? launch_kv_attend_many(a, gi, c->stream) : launch_kv_attend_few(a, v.plan.cols, gi, c->stream));
    unsigned parts = 0;  // of a row, now
    for (const KvJoin& j : kind ? v.plan.many_joins : v.plan.few_joins) parts = std::max(parts, j.parts);
    KV_LAUNCH(c, K_KV_ATTENTION, launch_kv_join(a, gj, rows, parts, c->stream));
  }
  return HALE_OK;
  KV_CATCH(c)
}

extern "C" int hale_kv_read_device(hale_kv_cache* kv, size_t layer, uint32_t seq, size_t first, size_t count, float* k,
                                   float* v) {
  if (!kv) return ctx_fail(nullptr, HALE_EINVAL, "kv_read: NULL argument");
  hale_ctx* c = kv->ctx;
  KV_TRY
  std::lock_guard<std::recursive_mutex> lk(c->mu);
  if (layer >= kv->layers) return ctx_fail(c, HALE_EINVAL, "kv_read: layer %zu of %zu", layer, kv->layers);
  size_t len = 0;
  std::string err;
  int rc = status(kv, "kv_read", kv->pages.len(seq, &len, &err), err);
  if (rc) return rc;
  if (first > len || count > len - first)
    return ctx_fail(c, HALE_EINVAL, "kv_read: positions %zu..%zu of %zu", first, first + count, len);
  if (count == 0) return HALE_OK;
  if (!k || !v || !aligned(k, HALE_F32) || !aligned(v, HALE_F32))
    return ctx_fail(c, HALE_EINVAL, "kv_read: outputs are NULL or not aligned");
  rc = moves_allowed(kv, "kv_read");
  if (rc) return rc;
  rc = send_pages(kv);
  if (rc) return rc;
  const size_t row = kv->shape.kv_heads * kv->shape.head_dim;
  for (size_t done = 0; done < count;) {
    const size_t n = kv_read_part(first + done, count - done);
    KV_LAUNCH(c, K_KV_READ, launch_kv_read(kv->geom, layer, seq, first + done, n, k + done * row, v + done * row, c->stream));
    done += n;
  }
  return HALE_OK;
  KV_CATCH(c)
}
