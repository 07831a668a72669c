// Runs the host side of attention over shared prefixes (hale-token_amd/csrc/kv.hip) over a HIP
// runtime in host memory (kv_fake_hip.h), under AddressSanitizer and UndefinedBehaviorSanitizer.
// The argument names the check; exits 1 with a message where it fails.
#include "kv_fake_hip.h"

using namespace hale;

namespace {

struct Cache {
  hale_ctx c;
  hale_kv_cache* kv = nullptr;
  Cache(size_t heads, size_t kv_heads, size_t dim, size_t pages, size_t seqs, size_t max_len) {
    CHECK(hale_kv_create(&c, 1, heads, kv_heads, dim, pages, seqs, max_len, &kv) == HALE_OK);
  }
  ~Cache() { hale_kv_destroy(kv); }
  uint32_t seq(uint32_t len) {
    uint32_t s = 0;
    CHECK(hale_kv_seq_create(kv, &s) == HALE_OK && hale_kv_step(kv, 1, &s, &len) == HALE_OK);
    return s;
  }
  std::vector<uint32_t> fork(uint32_t s, size_t n) {
    std::vector<uint32_t> made(n);
    CHECK(hale_kv_seq_fork(kv, s, n, made.data()) == HALE_OK);
    return made;
  }
  size_t tokens = 0;
  void step(const std::vector<uint32_t>& seqs, const std::vector<uint32_t>& n) {
    CHECK(hale_kv_step(kv, seqs.size(), seqs.data(), n.data()) == HALE_OK);
    tokens = 0;
    for (uint32_t v : n) tokens += v;
  }
  // The attention's launches but for joins, captured or not.
  std::vector<KvAttnArgs> attend(bool captured, int dtype = HALE_BF16) {
    static float x[4];
    c.kv_uses.clear();  // another graph
    fake.capturing = captured;
    fake.attends.clear();
    CHECK(hale_kv_attention_device(kv, 0, dtype, tokens, x, 1 << 20, 1.0f, 0, x, 1 << 20) == HALE_OK);
    fake.capturing = false;
    return fake.attends;
  }
};

// A step whose tokens are all of one sequence has nobody to share with, now or when it is replayed:
// it is launched as without sharing.
void one_sequence() {
  for (size_t share : {0, 64}) {
    Cache w(64, 8, 16, 300, 4, 1 << 20);
    const uint32_t a = w.seq(5000), b = w.seq(100);
    CHECK(hale_kv_share_prefixes(w.kv, share) == HALE_OK);
    for (uint32_t n : {1, 8, 300}) {
      w.step({b, a}, {0, n});
      CHECK(w.attend(false).size() == 1);
      const auto got = w.attend(true);
      CHECK(got.size() == 1 && got[0].kind == (n == 300));
    }
  }
}

// Sequences of many rows only have no launch for few rows, whatever they come to share.
void many_rows() {
  Cache w(16, 2, 16, 300, 6, 8000);
  CHECK(hale_kv_share_prefixes(w.kv, 64) == HALE_OK);
  const auto seqs = w.fork(w.seq(5000), 3);
  w.step(seqs, {200, 300, 20});
  CHECK(w.attend(false).size() == 1);
  const auto got = w.attend(true);
  CHECK(got.size() == 1 && got[0].kind == 1);
  w.step(seqs, {200, 300, 1});
  CHECK(w.attend(true).size() == 2);
}

}  // namespace

int main(int argc, char** argv) {
  const std::string what = argc > 1 ? argv[1] : "";
  if (what == "one_sequence") one_sequence();
  else if (what == "many_rows") many_rows();
  else return 2;
  CHECK(fake.device.empty() && fake.host.empty());
  return 0;
}
