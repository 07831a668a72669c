// Checks that sharing pages is worth it where a plan shares them
// (hale-token_amd/csrc/kv_pages.cpp): a step never reads more pages than with each sequence
// by itself, whatever its numbers of rows.  The argument names the check; exits 1 with a
// message where it fails.
#include <stdio.h>
#include <stdlib.h>

#include <algorithm>
#include <random>
#include <string>

#include "kv_pages.h"

using namespace hale;

#define CHECK(cond)                                                    \
  do {                                                                 \
    if (!(cond)) {                                                     \
      fprintf(stderr, "line %d: %s does not hold\n", __LINE__, #cond); \
      exit(1);                                                         \
    }                                                                  \
  } while (0)

namespace {

std::string err;
std::vector<KvCopy> copies;

size_t reads(const KvPlan& p) {
  size_t n = 0;
  for (const KvItem& it : p.few) n += it.page1 - it.page0;
  for (const KvItem& it : p.many) n += it.page1 - it.page0;
  return n;
}

// A step of forks behind a prompt, ntok tokens each, and its plans apart and shared.
struct Step {
  std::vector<KvStepSeq> seqs;
  KvPlan apart, shared;
};
Step forks(const KvShape& s, uint32_t prompt, const std::vector<uint32_t>& ntok, bool f32, const std::vector<uint32_t>& tails = {}) {
  KvPages pages;
  pages.init(40000, ntok.size() + 1, prompt + 2000);
  uint32_t root;
  std::vector<uint32_t> made(ntok.size());
  CHECK(pages.create(&root, &err) == KvPages::OK && pages.step(1, &root, &prompt, nullptr, &copies, &err) == KvPages::OK);
  CHECK(pages.fork(root, made.size(), made.data(), &err) == KvPages::OK);
  if (!tails.empty()) CHECK(pages.step(made.size(), made.data(), tails.data(), nullptr, &copies, &err) == KvPages::OK);
  Step t;
  CHECK(pages.step(made.size(), made.data(), ntok.data(), &t.seqs, &copies, &err) == KvPages::OK);
  kv_plan(s, t.seqs, 0, f32, &t.apart);
  kv_plan_shared(s, t.seqs, pages, 1, f32, &t.shared);
  return t;
}
std::vector<uint32_t> each(size_t n, uint32_t v) { return std::vector<uint32_t>(n, v); }

void no_more_pages() {
  for (bool f32 : {false, true})
    for (size_t kv : {1, 4, 8})
      for (size_t group : {1, 4, 8, 16})
        for (size_t dim : {128, 256})
          for (uint32_t ntok : {1, 2, 3, 5, 10, 12, 20, 40, 75, 200, 600})
            for (uint32_t n : {2, 3, 8, 32})
              for (uint32_t prompt : {70u, 1000u, 9000u}) {
                const Step t = forks({kv * group, kv, dim}, prompt, each(n, ntok), f32);
                CHECK(reads(t.shared) <= reads(t.apart));
              }
  std::mt19937 rng(5);
  for (int k = 0; k < 400; k++) {  // of all kinds side by side
    std::vector<uint32_t> ntok, tails;
    for (size_t n = 2 + rng() % 30; ntok.size() < n;) {
      ntok.push_back(rng() % 6 == 0 ? rng() % 700 : rng() % 9 == 0 ? 0 : 1 + rng() % 12);
      tails.push_back(rng() % 400);
    }
    const size_t kv = 1 + rng() % 8, group = (size_t)1 << rng() % 5;
    const uint32_t prompt = rng() % 9000;
    const bool f32 = rng() % 2;
    const Step t = forks({kv * group, kv, 64u << rng() % 3}, prompt, ntok, f32, tails);
    CHECK(reads(t.shared) <= reads(t.apart));
    // two neighbours whose rows fit into one tile of the 16 that the kernel of few takes at least, in a step
    // that is long enough
    bool saves = false, long_one = false;
    size_t before = 1000;
    for (size_t i = 0; i < ntok.size(); i++)
      if (ntok[i]) {
        saves |= (ntok[i] + before) * group <= 16, before = ntok[i];
        long_one |= prompt + tails[i] + ntok[i] > 4 * KV_PAGE;
      }
    CHECK(!(saves && long_one && prompt >= KV_PAGE) || reads(t.shared) < reads(t.apart));
  }
}

// Sequences of many rows stay with the kernel of many, and share where that saves enough.
void many_rows() {
  const KvShape s{32, 4, 128};
  for (bool f32 : {false, true}) {
    const Step five = forks(s, 4000, each(8, 5), f32);  // 40 rows each: three tiles in place of eight
    CHECK(five.shared.few.empty() && !five.shared.many.empty() && reads(five.shared) * 2 < reads(five.apart));
    for (uint32_t ntok : {12, 40, 600}) {  // tiles that are full already, or nearly
      const Step t = forks(s, 4000, each(4, ntok), f32);
      CHECK(t.shared.few.empty() && reads(t.shared) == reads(t.apart) && t.shared.many.size() == t.apart.many.size());
    }
    // a prompt among decoding sequences: those on either side share, in tiles of few rows
    std::vector<uint32_t> ntok = each(21, 1);
    ntok[10] = 300;
    const Step t = forks(s, 4000, ntok, f32);
    size_t most = 0;
    for (const KvItem& it : t.shared.few) most = std::max<size_t>(most, it.rows);
    CHECK(most == 16 && reads(t.shared) < reads(t.apart));
    for (const KvItem& it : t.shared.many) CHECK(it.tok0 == t.seqs[10].tok0);
  }
}

// A plan says whether it shares any pages: without, each join has the one series of its row's own.
void nothing_shared() {
  for (uint32_t ntok : {1, 300})
    for (uint32_t pair : {0, 1}) {
      const KvShape s{32, 8, 128};
      KvPages pages;
      pages.init(4000, 40, 6000);
      std::vector<uint32_t> seqs(30), n(30);
      for (uint32_t k = 0; k < 30; k++) {
        CHECK(pages.create(&seqs[k], &err) == KvPages::OK);
        n[k] = 3900 + 7 * k;
      }
      CHECK(pages.step(30, seqs.data(), n.data(), nullptr, &copies, &err) == KvPages::OK);
      if (pair) {  // two forks beside them
        uint32_t made[2];
        CHECK(pages.fork(seqs[4], 2, made, &err) == KvPages::OK);
        seqs.insert(seqs.begin() + 5, made, made + 2);
      }
      n.assign(seqs.size(), ntok);
      std::vector<KvStepSeq> plan;
      CHECK(pages.step(seqs.size(), seqs.data(), n.data(), &plan, &copies, &err) == KvPages::OK);
      KvPlan p;
      kv_plan_shared(s, plan, pages, 1, false, &p);
      CHECK(p.alone == !(pair && ntok == 1));  // (tiles of 300 tokens are full already, and so many that none is divided)
      size_t most = 0;
      for (const KvShareJoin& j : p.share_joins) most = std::max<size_t>(most, j.n);
      CHECK(ntok == 1 ? p.alone == (most == 1) && most : most <= 1);
      kv_plan(s, plan, 0, false, &p);
      CHECK(!p.alone && !p.shared);
    }
}

// Where there is no room for the partial results of all levels, or of all runs, the others are shared.
void as_much_as_there_is_room_for() {
  const KvShape s{64, 8, 256};  // room for 81920 rows of partial results, 64 a token and part
  KvPages pages;
  pages.init(60000, 1100, 6000);
  auto check = [&](const std::vector<uint32_t>& seqs) {
    std::vector<KvStepSeq> plan;
    const std::vector<uint32_t> n(seqs.size(), 1);
    CHECK(pages.step(seqs.size(), seqs.data(), n.data(), &plan, &copies, &err) == KvPages::OK);
    KvPlan apart, shared;
    kv_plan(s, plan, 0, false, &apart);
    kv_plan_shared(s, plan, pages, 1, false, &shared);
    CHECK(shared.part_rows <= kv_part_rows(s.head_dim));
    return std::pair<size_t, KvPlan>(reads(apart) - reads(shared), shared);
  };
  // 20 talks of 30 behind one prompt: 38400 rows for each level and for the sequences' own pages
  uint32_t root;
  uint32_t len = 2000;
  CHECK(pages.create(&root, &err) == KvPages::OK && pages.step(1, &root, &len, nullptr, &copies, &err) == KvPages::OK);
  std::vector<uint32_t> talks(20), seqs;
  CHECK(pages.fork(root, 20, talks.data(), &err) == KvPages::OK);
  const std::vector<uint32_t> more(20, 640);
  CHECK(pages.step(20, talks.data(), more.data(), nullptr, &copies, &err) == KvPages::OK);
  for (uint32_t t : talks) {
    uint32_t made[30];
    CHECK(pages.fork(t, 30, made, &err) == KvPages::OK);
    seqs.insert(seqs.end(), made, made + 30);
  }
  auto got = check(seqs);
  // 31 pages of 8 heads, so many that they go to the kernel of many: tiles of 64 rows, 8 a sequence
  CHECK(got.first == (600 - 600 / 8) * 31u * 8);
  // two prompts with 500 answers each, 64000 rows of partial results each: the longer one's are shared
  for (uint32_t s : seqs) CHECK(pages.free(s, &err) == KvPages::OK);
  seqs.clear();
  for (uint32_t prompt : {1000u, 2000u}) {
    uint32_t a;
    std::vector<uint32_t> made(500);
    CHECK(pages.create(&a, &err) == KvPages::OK && pages.step(1, &a, &prompt, nullptr, &copies, &err) == KvPages::OK);
    CHECK(pages.fork(a, 500, made.data(), &err) == KvPages::OK);
    seqs.insert(seqs.end(), made.begin(), made.end());
  }
  got = check(seqs);
  CHECK(got.first == (500 - (500 + 7) / 8) * 31u * 8);
  for (const KvShareJoin& j : got.second.share_joins) CHECK(j.tok0 >= 500 && j.n == 2);
}

// 24 sequences of 16 rows each, whose shared pages go to the kernel of many rows and whose own, also where
// they have nothing in common, do not: what a captured step has to launch both kernels for.
void many_rows_by_sharing() {
  const KvShape s{128, 16, 32};
  for (bool f32 : {false, true}) {
    const Step t = forks(s, f32 ? 5700 : 3000, each(24, 2), f32);
    CHECK(!t.shared.many.empty() && !t.shared.few.empty() && t.apart.many.empty());
    CHECK(kv_share_may_many(s, t.seqs, 94, f32));
    KvPages pages;
    pages.init(400, 24, 6000);
    std::vector<uint32_t> seqs(24), n(24);
    for (uint32_t k = 0; k < 24; k++) {
      CHECK(pages.create(&seqs[k], &err) == KvPages::OK);
      n[k] = 30 * k;
    }
    CHECK(pages.step(24, seqs.data(), n.data(), nullptr, &copies, &err) == KvPages::OK);
    n = each(24, 2);
    std::vector<KvStepSeq> plan;
    CHECK(pages.step(24, seqs.data(), n.data(), &plan, &copies, &err) == KvPages::OK);
    KvPlan p;
    kv_plan_shared(s, plan, pages, 1, f32, &p);
    CHECK(p.many.empty() && p.alone && p.share_joins.empty());
  }
}

// Steps of short sequences, a few pages each, stay apart and need no joins; more or longer ones share.
void short_steps() {
  const KvShape s{32, 4, 128};
  for (bool f32 : {false, true}) {
    const Step a = forks(s, 200, each(8, 1), f32, each(8, 55));  // 256 positions with the new token
    CHECK(a.shared.alone && a.shared.share_joins.empty() && reads(a.shared) == reads(a.apart) && a.apart.few_joins.empty());
    std::vector<uint32_t> tails = each(8, 55);
    tails[3] = 56;
    const Step b = forks(s, 200, each(8, 1), f32, tails);  // one of 257
    CHECK(!b.shared.alone && reads(b.shared) < reads(b.apart));
    const Step c = forks(s, 200, each(200, 1), f32, each(200, 55));  // 800 tiles of four pages
    CHECK(!c.shared.alone && reads(c.shared) < reads(c.apart));
  }
}

// Rows of more parts than the join brings to LDS at once (256), over three levels of a long history.
void many_parts() {
  const KvShape s{2, 1, 16};
  KvPages pages;
  pages.init(1100, 8, 66000);
  uint32_t root, two[2], three[2], four;
  const auto step = [&](std::vector<uint32_t> seqs, std::vector<uint32_t> n, std::vector<KvStepSeq>* plan = nullptr) {
    CHECK(pages.step(seqs.size(), seqs.data(), n.data(), plan, &copies, &err) == KvPages::OK);
  };
  CHECK(pages.create(&root, &err) == KvPages::OK);
  step({root}, {337 * 64});
  CHECK(pages.fork(root, 2, two, &err) == KvPages::OK);
  step({two[1]}, {341 * 64});
  CHECK(pages.fork(two[1], 2, three, &err) == KvPages::OK);
  step({three[1]}, {341 * 64});
  CHECK(pages.fork(three[1], 1, &four, &err) == KvPages::OK);
  std::vector<KvStepSeq> plan;
  step({two[0], three[0], three[1], four}, each(4, 1), &plan);
  KvPlan p;
  kv_plan_shared(s, plan, pages, 1, true, &p);
  size_t most = 0;
  for (const KvShareJoin& j : p.share_joins) {
    size_t n = 0;
    for (uint32_t k = 0; k < j.n; k++) n += j.of[k].parts;
    most = std::max(most, n);
  }
  CHECK(most == 258);
}

}  // namespace

int main(int argc, char** argv) {
  const std::string what = argc > 1 ? argv[1] : "";
  if (what == "no_more_pages") no_more_pages();
  else if (what == "many_rows") many_rows();
  else if (what == "nothing_shared") nothing_shared();
  else if (what == "as_much_as_there_is_room_for") as_much_as_there_is_room_for();
  else if (what == "many_rows_by_sharing") many_rows_by_sharing();
  else if (what == "short_steps") short_steps();
  else if (what == "many_parts") many_parts();
  else return 2;
  return 0;
}
