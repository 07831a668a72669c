// Runs the key/value cache's host side (hale-token_amd/csrc/kv.hip) over a HIP
// runtime in host memory (kv_fake_hip.h), under AddressSanitizer and
// UndefinedBehaviorSanitizer.  The argument names the check; exits 1 with a
// message where it fails.
#include "kv_fake_hip.h"

using namespace hale;

namespace {

struct Cache {
  hale_ctx c;
  hale_kv_cache* kv = nullptr;
  explicit Cache(size_t layers = 1, size_t heads = 4, size_t kv_heads = 2, size_t dim = 16, size_t pages = 64, size_t seqs = 8,
                 size_t max_len = 1024) {
    CHECK(hale_kv_create(&c, layers, heads, kv_heads, dim, pages, seqs, max_len, &kv) == HALE_OK);
  }
  ~Cache() { hale_kv_destroy(kv); }
  uint32_t seq() {
    uint32_t s = 0;
    CHECK(hale_kv_seq_create(kv, &s) == HALE_OK);
    return s;
  }
  int step(std::vector<uint32_t> seqs, std::vector<uint32_t> n) { return hale_kv_step(kv, seqs.size(), seqs.data(), n.data()); }
  int append(size_t ntok) {
    static float x[4];
    return hale_kv_append_device(kv, 0, HALE_F32, ntok, x, 1 << 20, x, 1 << 20);
  }
  int attend(size_t ntok, int dtype = HALE_F32, size_t window = 0) {
    static float x[4];
    return hale_kv_attention_device(kv, 0, dtype, ntok, x, 1 << 20, 1.0f, window, x, 1 << 20);
  }
  size_t len(uint32_t s) {
    size_t n = 0;
    CHECK(hale_kv_seq_len(kv, s, &n) == HALE_OK);
    return n;
  }
  size_t used() {
    size_t n = 0;
    CHECK(hale_kv_pages(kv, nullptr, &n) == HALE_OK);
    return n;
  }
};

// A step of one token and of a prompt's chunk, both behind long contexts, after
// four windows were attended over in both kinds of type: every list of
// every view has entries, and each arrives where the kernels read it.
void every_view() {
  const KvShape shape{32, 4, 128};
  const size_t windows[4] = {0, 1024, 2048, 4096}, lens[2] = {9000, 8000};
  const uint32_t ntok[2] = {1, 300};
  Cache w(1, 32, 4, 128, 300, 2, 12000);
  const uint32_t a = w.seq(), b = w.seq();
  CHECK(w.step({a, b}, {(uint32_t)lens[0], (uint32_t)lens[1]}) == HALE_OK);
  const size_t total = lens[0] + lens[1];
  for (int dtype : {HALE_F32, HALE_BF16})
    for (size_t window : windows) CHECK(w.attend(total, dtype, window) == HALE_OK);
  CHECK(w.step({a, b}, {ntok[0], ntok[1]}) == HALE_OK);
  CHECK(w.append(301) == HALE_OK);
  const std::vector<KvStepSeq> seqs = {{a, (uint32_t)lens[0], ntok[0], 0}, {b, (uint32_t)lens[1], ntok[1], 1}};
  int full = 0;
  for (int dtype : {HALE_F32, HALE_BF16})
    for (size_t window : windows) {
      fake.attends.clear();
      const int uploads = fake.uploads;
      CHECK(w.attend(301, dtype, window) == HALE_OK);
      CHECK(fake.uploads == uploads && fake.attends.size() == 2);
      KvPlan plan;
      kv_plan(shape, seqs, window, dtype == HALE_F32, &plan);
      full += !plan.few.empty() && !plan.many.empty() && !plan.few_joins.empty() && !plan.many_joins.empty();
      const uint32_t counts[4] = {(uint32_t)plan.few.size(), (uint32_t)plan.many.size(), (uint32_t)plan.few_joins.size(),
                                  (uint32_t)plan.many_joins.size()};
      for (int kind = 0; kind < 2; kind++) {
        const KvAttnArgs& at = fake.attends[kind];
        const auto& items = kind ? plan.many : plan.few;
        const auto& joins = kind ? plan.many_joins : plan.few_joins;
        CHECK(at.kind == kind && !memcmp(at.counts, counts, sizeof counts));
        CHECK(!memcmp(at.items, items.data(), items.size() * sizeof(KvItem)));
        CHECK(!memcmp(at.joins, joins.data(), joins.size() * sizeof(KvJoin)));
      }
    }
  CHECK(full == 8);
}

// Graphs keep the addresses that they were captured with: what a graph may still
// read stays until the context's last graph is gone.
void plan_behind_a_graph() {
  hale_ctx c;
  hale_kv_cache* kv = nullptr;
  const int32_t *old = nullptr, *grown = nullptr;
  CHECK(hale_kv_create(&c, 1, 4, 2, 16, 64, 8, 1024, &kv) == HALE_OK);
  CHECK(hale_kv_positions(kv, &old) == HALE_OK);
  const size_t before = fake.device.size();
  c.live_graphs = 1;
  CHECK(hale_kv_reserve(kv, 5000) == HALE_OK);
  CHECK(hale_kv_positions(kv, &grown) == HALE_OK && grown != old);
  CHECK(fake.device.size() == before + 1 && c.retired.size() == 1);
  volatile int32_t at = old[0];  // as a replay reads it
  (void)at;
  hale_kv_destroy(kv);
  at = old[0];
  at = grown[0];
  CHECK(c.retired.size() == 2 && fake.device.size() == 2);
  for (void* p : c.retired) (void)hipFree(p);  // as the last graph's end does
  // without a graph nothing is kept
  c.live_graphs = 0;
  c.retired.clear();
  CHECK(hale_kv_create(&c, 1, 4, 2, 16, 64, 8, 1024, &kv) == HALE_OK);
  CHECK(hale_kv_reserve(kv, 5000) == HALE_OK);
  CHECK(c.retired.empty() && fake.device.size() == before);
  hale_kv_destroy(kv);
}

// A captured rotation of the step's positions: replayed for any step, refused
// once the positions lie elsewhere.
void rotation_in_a_graph() {
  Cache w;
  const uint32_t a = w.seq();
  hale_rope_config config{};
  config.head_dim = config.rotary_dim = 16;
  config.base = 1e4;
  config.attention_factor = 1.0;
  hale_rope* rope = nullptr;
  CHECK(hale_rope_create(&w.c, &config, &rope) == HALE_OK);
  const int32_t* pos = nullptr;
  int32_t other[4] = {};
  float x[64];
  auto turn = [&](const int32_t* p) { return hale_rope_device(rope, HALE_F32, 2, p, x, 1, 16, x, 16, nullptr, 0, 0, nullptr, 0); };
  CHECK(hale_kv_positions(w.kv, &pos) == HALE_OK);
  CHECK(w.step({a}, {3}) == HALE_OK && turn(pos) == HALE_OK && w.c.kv_uses.empty());
  fake.capturing = true;
  CHECK(turn(other) == HALE_OK && w.c.kv_uses.empty());
  CHECK(turn(pos) == HALE_OK && turn(pos + 1) == HALE_OK && w.c.kv_uses.size() == 1);
  fake.capturing = false;
  std::vector<KvUse> uses = w.c.kv_uses;
  w.c.kv_uses.clear();
  CHECK(kv_check_replay(&w.c, uses) == HALE_OK);
  CHECK(w.step({a}, {5}) == HALE_OK && kv_check_replay(&w.c, uses) == HALE_OK);
  // with a store in the same graph, in either order, the step has to be of the same tokens
  for (int first = 0; first < 2; first++) {
    fake.capturing = true;
    CHECK((first ? turn(pos) : w.append(5)) == HALE_OK && (first ? w.append(5) : turn(pos)) == HALE_OK);
    fake.capturing = false;
    std::vector<KvUse> both;
    both.swap(w.c.kv_uses);
    CHECK(kv_check_replay(&w.c, both) == HALE_OK);
    CHECK(w.step({a}, {4}) == HALE_OK && kv_check_replay(&w.c, both) == HALE_EINVAL);
    CHECK(w.step({a}, {5}) == HALE_OK && kv_check_replay(&w.c, both) == HALE_OK);
  }
  CHECK(hale_kv_reserve(w.kv, 5000) == HALE_OK);
  CHECK(kv_check_replay(&w.c, uses) == HALE_EINVAL && w.c.err.find("grew") != std::string::npos);
  fake.capturing = true;
  CHECK(hale_kv_positions(w.kv, &pos) == HALE_OK && turn(pos) == HALE_OK);
  fake.capturing = false;
  uses.swap(w.c.kv_uses);
  CHECK(kv_check_replay(&w.c, uses) == HALE_OK);
  hale_kv_destroy(w.kv);
  w.kv = nullptr;
  CHECK(kv_check_replay(&w.c, uses) == HALE_EINVAL && w.c.err.find("gone") != std::string::npos);
  hale_rope_destroy(rope);
}

// What a caller can see of a cache: sequences, pages, the current step's plan as the
// kernels read it, and every position's page through the page table.
struct Seen {
  std::vector<size_t> lens;
  size_t used = 0;
  std::vector<std::vector<uint8_t>> plan;
  std::vector<uint8_t> contents;
  bool operator==(const Seen& o) const {
    return lens == o.lens && used == o.used && plan == o.plan && contents == o.contents;
  }
};
Seen look(Cache& w, const std::vector<uint32_t>& seqs, size_t tokens) {
  fake.allocs_until_failure = -1;
  Seen s;
  for (uint32_t q : seqs) s.lens.push_back(w.len(q));
  s.used = w.used();
  fake.attends.clear();
  fake.appends.clear();
  if (tokens) {
    CHECK(w.append(tokens) == HALE_OK);  // sends what the page table lacks
    for (size_t window : {0, 20}) CHECK(w.attend(tokens, HALE_F32, window) == HALE_OK);
    const KvAppendArgs& p = fake.appends[0];
    auto keep = [&](const void* at, size_t n) { s.plan.emplace_back((const uint8_t*)at, (const uint8_t*)at + n); };
    keep(&p.nblocks, 4);
    keep(p.blocks, p.nblocks * sizeof(KvBlock));
    for (const KvAttnArgs& a : fake.attends) {
      keep(a.counts, 16);
      keep(a.items, a.nitems * sizeof(KvItem));
      keep(a.joins, a.njoins * sizeof(KvJoin));
    }
    for (size_t i = 0; i < seqs.size(); i++)
      for (size_t j = 0; j * KV_PAGE < s.lens[i]; j++)
        s.contents.push_back(p.g.pool[p.g.table[seqs[i] * p.g.max_pages + j] * p.g.page_bytes]);
  }
  return s;
}
// A byte of each page, by which its copies are known.
void mark_pages(Cache& w) {
  fake.appends.clear();
  CHECK(w.append(430) == HALE_OK);
  const KvGeom& g = fake.appends[0].g;
  for (size_t p = 0; p < 64; p++) g.pool[p * g.page_bytes] = (uint8_t)(p + 1);
}

// Runs `call` with the first, second, .. allocation failing until none does: after
// each failure all that can be seen is as before.  Returns the failures.
template <typename F>
int without_memory(Cache& w, const std::vector<uint32_t>& seqs, size_t tokens, F call) {
  const Seen before = look(w, seqs, tokens);
  for (int k = 0;; k++) {
    CHECK(k < 1000);
    fake.allocs_until_failure = k;
    const int rc = call();
    fake.allocs_until_failure = -1;
    if (rc == HALE_OK) return k;
    CHECK(rc == HALE_ENOMEM);
    CHECK(look(w, seqs, tokens) == before);
  }
}

// Sequences of 300, 120 and 10 positions, the second's pages shared with a fork, and
// a hole in the pool; the step in progress has 430 tokens.
std::vector<uint32_t> furnish(Cache& w) {
  const uint32_t hole = w.seq(), a = w.seq(), b = w.seq(), c = w.seq();
  CHECK(w.step({hole}, {200}) == HALE_OK && w.attend(200) == HALE_OK && w.attend(200, HALE_F32, 20) == HALE_OK);
  CHECK(w.step({a, b, c}, {300, 120, 10}) == HALE_OK);
  CHECK(hale_kv_seq_free(w.kv, hole) == HALE_OK);
  uint32_t f = 0;
  CHECK(hale_kv_seq_fork(w.kv, b, 1, &f) == HALE_OK);
  mark_pages(w);
  return {a, b, c, f};
}

void step_without_memory() {
  for (uint32_t n : {1u, 3000u}) {  // within the plan's buffers, and growing them
    Cache w(1, 4, 2, 16, 64, 8, 4000);
    const std::vector<uint32_t> s = furnish(w);
    const uint32_t seqs[2] = {s[1], s[2]}, ntok[2] = {n, 70};
    CHECK(without_memory(w, s, 430, [&] { return hale_kv_step(w.kv, 2, seqs, ntok); }) > 0);
    const Seen after = look(w, s, n + 70);
    CHECK((after.lens == std::vector<size_t>{300, 120 + n, 80, 120}));
  }
}

// Sequences that can still be made (and are given back).
size_t free_sequences(Cache& w) {
  std::vector<uint32_t> made;
  uint32_t s = 0;
  while (hale_kv_seq_create(w.kv, &s) == HALE_OK) made.push_back(s);
  for (uint32_t m : made) CHECK(hale_kv_seq_free(w.kv, m) == HALE_OK);
  return made.size();
}

void copy_without_memory() {
  Cache w(1, 4, 2, 16, 64, 8, 4000);
  const std::vector<uint32_t> s = furnish(w);
  const size_t left = free_sequences(w);
  uint32_t out = 0;
  CHECK(without_memory(w, s, 430, [&] { return hale_kv_seq_copy(w.kv, s[0], &out); }) > 0);
  CHECK(free_sequences(w) == left - 1 && w.len(out) == 300);
  const uint32_t one[1] = {1}, both[2] = {s[0], out};
  CHECK(hale_kv_step(w.kv, 1, both + 1, one) == HALE_OK);  // sends the page table
  const Seen a = look(w, {s[0]}, 1), b = look(w, {out}, 1);
  CHECK(a.contents == b.contents && b.contents.size() == 5);
}

void compact_without_memory() {
  Cache w(1, 4, 2, 16, 64, 8, 4000);
  const std::vector<uint32_t> s = furnish(w);  // the first pages are free
  size_t moved = 99;
  CHECK(without_memory(w, s, 430, [&] { return hale_kv_compact(w.kv, &moved); }) > 0);
  CHECK(moved == 4);  // all of them by the call that succeeded
  CHECK(hale_kv_compact(w.kv, &moved) == HALE_OK && moved == 0);
  const Seen after = look(w, s, 430);
  CHECK(after.used == 8 && after.contents.size() == 10);
}

void others_without_memory() {
  Cache w(1, 4, 2, 16, 64, 8, 4000);
  const std::vector<uint32_t> s = furnish(w);
  const size_t left = free_sequences(w);
  static float x[4];
  for (size_t window : {40, 60}) {  // the third and the fourth one
    CHECK(without_memory(w, s, 430, [&] {
            return hale_kv_attention_device(w.kv, 0, HALE_F32, 430, x, 1 << 20, 1.0f, window, x, 1 << 20);
          }) > 0);
  }
  CHECK(w.attend(430, HALE_F32, 80) == HALE_EINVAL);
  uint32_t out[2] = {};
  CHECK(without_memory(w, s, 430, [&] { return hale_kv_seq_fork(w.kv, s[0], 2, out); }) > 0);
  CHECK(free_sequences(w) == left - 2 && w.len(out[0]) == 300 && w.len(out[1]) == 300);
  CHECK(without_memory(w, s, 430, [&] { return hale_kv_seq_truncate(w.kv, out[0], 70); }) >= 0);
  CHECK(without_memory(w, s, 430, [&] { return hale_kv_seq_free(w.kv, out[0]); }) >= 0);
  CHECK(without_memory(w, s, 430, [&] { return hale_kv_seq_create(w.kv, out); }) >= 0);
  CHECK(without_memory(w, s, 430, [&] { return hale_kv_resize(w.kv, 30); }) > 0);
  CHECK(without_memory(w, s, 430, [&] { return hale_kv_resize(w.kv, 50); }) > 0);
  const Seen resized = look(w, s, 430);
  CHECK(resized.contents.size() == 10);
  hale_rope_config config{};
  config.head_dim = config.rotary_dim = 16;
  config.base = 1e4;
  config.attention_factor = 1.0;
  hale_rope* rope = nullptr;
  const size_t device = fake.device.size();
  CHECK(without_memory(w, s, 430, [&] { return hale_rope_create(&w.c, &config, &rope); }) > 0);
  CHECK(fake.device.size() == device + 1);
  hale_rope_destroy(rope);
  hale_kv_cache* more = nullptr;
  const size_t host = fake.host.size();
  CHECK(without_memory(w, s, 430, [&] {
          const int rc = hale_kv_create(&w.c, 1, 4, 2, 16, 64, 8, 4000, &more);
          CHECK(rc == HALE_OK || (!more && fake.device.size() == device && w.c.kvs.size() == 1));
          return rc;
        }) > 0);
  CHECK(fake.host.size() == host + 1);
  hale_kv_destroy(more);
  // a graph's notes
  fake.capturing = true;
  for (int k = 0;; k++) {
    fake.allocs_until_failure = k;
    const int rc = hale_kv_append_device(w.kv, 0, HALE_F32, 430, x, 1 << 20, x, 1 << 20);
    fake.allocs_until_failure = -1;
    if (rc == HALE_OK) break;
    CHECK(rc == HALE_ENOMEM && w.c.kv_uses.empty());
  }
  fake.capturing = false;
  CHECK(w.c.kv_uses.size() == 1);
}

// A launch works on the step of its moment, which a graph inside another one
// would not see: refused while a capture goes on.
void launch_in_a_capture() {
  Cache w;
  const uint32_t a = w.seq();
  CHECK(w.step({a}, {3}) == HALE_OK && w.attend(3) == HALE_OK);
  fake.capturing = true;
  CHECK(w.attend(3) == HALE_OK);
  std::vector<KvUse> uses;
  uses.swap(w.c.kv_uses);
  uint32_t f = 0;
  CHECK(hale_kv_seq_fork(w.kv, a, 1, &f) == HALE_OK);  // a page table change to be sent
  CHECK(kv_check_replay(&w.c, uses) == HALE_EINVAL && w.c.err.find("captur") != std::string::npos);
  fake.capturing = false;
  CHECK(kv_check_replay(&w.c, uses) == HALE_OK);
}

// Reading goes in launches whose threads, 256 for each page, a grid's dimension can
// count, and whose positions lie one behind the other.
void long_reads() {
  const size_t most = (1u << 30);
  for (size_t first : {(size_t)0, (size_t)1, (size_t)63, (size_t)64, (size_t)5000})
    for (size_t count : {(size_t)1, (size_t)64, (size_t)1000, most - 64 - first, most - 63 - first, most - first}) {
      size_t at = first, launches = 0;
      while (at < first + count) {
        const size_t n = kv_read_part(at, first + count - at);
        CHECK(n >= 1 && at + n <= first + count);
        CHECK(((at + n - 1) / KV_PAGE - at / KV_PAGE + 1) * 256 < (size_t)1 << 32);
        at += n;
        launches++;
      }
      CHECK(at == first + count && launches <= 2);
    }
  Cache w;
  const uint32_t a = w.seq();
  CHECK(w.step({a}, {300}) == HALE_OK);
  float x[4];
  CHECK(hale_kv_read_device(w.kv, 0, a, 70, 200, x, x) == HALE_OK);
  CHECK(fake.read_counts == std::vector<size_t>{200});
}

}  // namespace

int main(int argc, char** argv) {
  const std::string what = argc > 1 ? argv[1] : "";
  if (what == "every_view")
    every_view();
  else if (what == "plan_behind_a_graph")
    plan_behind_a_graph();
  else if (what == "rotation_in_a_graph")
    rotation_in_a_graph();
  else if (what == "step_without_memory")
    step_without_memory();
  else if (what == "copy_without_memory")
    copy_without_memory();
  else if (what == "compact_without_memory")
    compact_without_memory();
  else if (what == "others_without_memory")
    others_without_memory();
  else if (what == "launch_in_a_capture")
    launch_in_a_capture();
  else if (what == "long_reads")
    long_reads();
  else
    return 2;
  CHECK(fake.device.empty() && fake.host.empty());
  return 0;
}
