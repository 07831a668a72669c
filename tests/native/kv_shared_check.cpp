// Checks the plans of steps whose sequences share pages
// (hale-token_amd/csrc/kv_pages.cpp) over random histories of forks, steps and
// truncations: every page that a row sees is attended over once, by an item whose
// page is the row's own, partial results lie apart, and a row's join takes
// exactly the parts that its items leave.  Exits 1 with a message where one
// of it fails.
#include <stdio.h>
#include <stdlib.h>

#include <algorithm>
#include <random>

#include "kv_pages.h"

using namespace hale;

#define CHECK(cond)                                                    \
  do {                                                                 \
    if (!(cond)) {                                                     \
      fprintf(stderr, "line %d: %s does not hold\n", __LINE__, #cond); \
      exit(1);                                                         \
    }                                                                  \
  } while (0)

// The pages that a plan reads, summed over its items.
static size_t check_plan(const KvShape& s, const KvPages& pages, const std::vector<KvStepSeq>& seqs, const KvPlan& plan) {
  const size_t group = s.group();
  size_t tokens = 0, read = 0;
  std::vector<const KvStepSeq*> of;  // token -> sequence
  for (const KvStepSeq& q : seqs)
    for (uint32_t t = 0; t < q.ntok; t++) of.push_back(&q), tokens++;
  CHECK(plan.shared && plan.few_joins.empty() && plan.many_joins.empty());
  CHECK(plan.few.size() <= kv_max_items(s, tokens, seqs.size()) && plan.many.size() <= kv_max_items(s, tokens, seqs.size()));
  CHECK(plan.share_joins.size() <= kv_max_items(s, tokens, seqs.size()) - KV_MAX_PARTS);
  CHECK(plan.part_rows <= kv_part_rows(s.head_dim));
  struct Row {
    std::vector<uint8_t> pages;  // how often each was attended over
    std::vector<uint32_t> parts;
    bool whole = false;
  };
  std::vector<Row> rows(tokens * group * s.kv_heads);
  std::vector<char> used(plan.part_rows, 0);
  for (int kind = 0; kind < 2; kind++)
    for (const KvItem& it : kind ? plan.many : plan.few) {
      CHECK(it.rows > 0 && it.page0 < it.page1 && it.head < s.kv_heads);
      CHECK(it.rows <= (kind ? kv_many_rows(s.head_dim) : 16 * (size_t)plan.cols));
      read += it.page1 - it.page0;
      for (uint32_t r = 0; r < it.rows; r++) {
        const size_t tok = it.tok0 + (it.row0 + r) / group;
        CHECK(tok < tokens);
        const KvStepSeq& q = *of[tok];
        const uint32_t pos = q.len0 + (uint32_t)(tok - q.tok0), item_pos = it.len0 + (it.row0 + r) / (uint32_t)group;
        Row& row = rows[(tok * group + (it.row0 + r) % group) * s.kv_heads + it.head];
        for (uint32_t p = it.page0; p < it.page1; p++) {
          if (p * KV_PAGE > pos) continue;  // hidden as the row's own mask says
          CHECK(pages.page_of(it.row, p * KV_PAGE) == pages.page_of(q.row, p * KV_PAGE));
          if (row.pages.size() <= p) row.pages.resize(p + 1);
          row.pages[p]++;
          // what the item's mask lets the row see of the page is what it holds
          const uint32_t last = std::min<uint32_t>(pos, p * KV_PAGE + KV_PAGE - 1), seen = std::min<uint32_t>(item_pos, p * KV_PAGE + KV_PAGE - 1);
          CHECK(last == seen);
          if (it.row != q.row) CHECK(p < q.len0 / KV_PAGE && p < pages.max_pages());
        }
        if (it.part == KV_WHOLE) {
          CHECK(!row.whole);
          row.whole = true;
        } else {
          CHECK(it.part + r < plan.part_rows && !used[it.part + r]);
          used[it.part + r] = 1;
          row.parts.push_back(it.part + r);
        }
      }
    }
  for (size_t tok = 0; tok < tokens; tok++)
    for (size_t x = 0; x < group * s.kv_heads; x++) {
      const Row& row = rows[tok * group * s.kv_heads + x];
      const uint32_t last = (of[tok]->len0 + (uint32_t)(tok - of[tok]->tok0)) / KV_PAGE;
      CHECK(row.pages.size() == last + 1);
      for (uint8_t n : row.pages) CHECK(n == 1);
      CHECK(row.whole == row.parts.empty());
    }
  std::vector<char> joined(rows.size(), 0);
  for (const KvShareJoin& j : plan.share_joins) {
    CHECK(j.n >= 1 && j.n <= KV_SHARE_LEVELS + 1 && j.rows <= kv_many_rows(s.head_dim));
    for (uint32_t r = 0; r < j.rows; r++) {
      const size_t tok = j.tok0 + (j.row0 + r) / group, at = (tok * group + (j.row0 + r) % group) * s.kv_heads + j.head;
      CHECK(tok < tokens && !joined[at]);
      joined[at] = 1;
      std::vector<uint32_t> parts;
      for (uint32_t k = 0; k < j.n; k++)
        for (uint32_t p = 0; p < j.of[k].parts; p++) parts.push_back(j.of[k].part0 + r + p * j.of[k].step);
      std::sort(parts.begin(), parts.end());
      std::sort(rows[at].parts.begin(), rows[at].parts.end());
      CHECK(parts.size() <= KV_SHARE_PARTS && parts == rows[at].parts);
    }
  }
  for (size_t k = 0; k < rows.size(); k++) CHECK(joined[k] == !rows[k].whole);
  return read;
}

int main() {
  std::mt19937 rng(7);
  auto below = [&](uint32_t n) { return (uint32_t)(rng() % n); };
  std::string err;
  std::vector<KvCopy> copies;
  size_t fewer = 0, rounds = 0;
  for (int trial = 0; trial < 60; trial++) {
    const size_t kv = 1 + below(4), group = 1 + below(8), dims[4] = {64, 128, 192, 256};
    const KvShape s{kv * group, kv, dims[below(4)]};
    KvPages pages;
    pages.init(6000, 40, 20000);
    std::vector<uint32_t> live;
    for (int k = 0; k < 3; k++) {
      uint32_t a;
      CHECK(pages.create(&a, &err) == KvPages::OK);
      live.push_back(a);
    }
    const uint32_t prompts[3] = {below(4000), below(600), 64 * below(20)};
    CHECK(pages.step(3, live.data(), prompts, nullptr, &copies, &err) == KvPages::OK);
    for (int turn = 0; turn < 12; turn++) {
      const uint32_t what = below(10);
      if (what < 3 && live.size() < 34) {
        uint32_t made[6];
        const size_t n = 1 + below(6);
        const size_t at = below((uint32_t)live.size());
        CHECK(pages.fork(live[at], n, made, &err) == KvPages::OK);
        live.insert(live.begin() + (long)at, made, made + n);  // beside their origin
      } else if (what == 3) {
        size_t len = 0;
        const uint32_t a = live[below((uint32_t)live.size())];
        CHECK(pages.len(a, &len, &err) == KvPages::OK);
        CHECK(pages.truncate(a, below((uint32_t)len + 1), &err) == KvPages::OK);
      } else if (what == 4 && live.size() > 4) {
        CHECK(pages.free(live.back(), &err) == KvPages::OK);
        live.pop_back();
      } else if (what == 5) {
        copies.clear();
        pages.compact(&copies);
      }
      // a step of some of them, most with a token or a few, some with a chunk
      std::vector<uint32_t> seqs, ntok;
      for (uint32_t a : live)
        if (below(8)) {
          seqs.push_back(a);
          ntok.push_back(below(16) == 0 ? below(700) : below(6) == 0 ? 0 : 1 + below(3));
        }
      std::vector<KvStepSeq> plan;
      copies.clear();
      if (pages.step(seqs.size(), seqs.data(), ntok.data(), &plan, &copies, &err) != KvPages::OK) continue;
      KvPlan shared, apart;
      const bool f32 = below(2);
      kv_plan_shared(s, plan, pages, 1 + below(6), f32, &shared);
      const size_t a = check_plan(s, pages, plan, shared);
      // what a captured launch may leave out
      const bool own = std::any_of(plan.begin(), plan.end(), [&](const KvStepSeq& q) { return q.ntok * s.group() > kv_few_limit(s, plan, f32); });
      CHECK(shared.many.empty() || own || kv_share_may_many(s, plan, pages.max_pages(), f32));
      kv_plan_shared(s, plan, pages, 1u << 20, f32, &apart);
      const size_t b = check_plan(s, pages, plan, apart);
      fewer += a < b;
      rounds++;
      // after pages moved the plan still holds
      copies.clear();
      pages.compact(&copies);
      check_plan(s, pages, plan, shared);
    }
  }
  fprintf(stderr, "%zu steps, %zu of them read less\n", rounds, fewer);
  CHECK(rounds > 300 && fewer > rounds / 4);
  // partial results beyond their room: the step is planned without sharing
  {
    const KvShape s{64, 1, 128};
    KvPages pages;
    pages.init(20000, 600, 8000);
    uint32_t root, made[500];
    std::vector<uint32_t> n(500, 4);
    CHECK(pages.create(&root, &err) == KvPages::OK);
    const uint32_t len = 4000;
    CHECK(pages.step(1, &root, &len, nullptr, &copies, &err) == KvPages::OK);
    CHECK(pages.fork(root, 500, made, &err) == KvPages::OK);
    std::vector<KvStepSeq> plan;
    CHECK(pages.step(500, made, n.data(), &plan, &copies, &err) == KvPages::OK);
    KvPlan p;
    kv_plan_shared(s, plan, pages, 1, false, &p);
    check_plan(s, pages, plan, p);
  }
  // few rows' kernel for short shared prompts, many rows' for long ones of many rows
  for (uint32_t len : {500u, 12000u}) {
    const KvShape s{64, 8, 128};
    KvPages pages;
    pages.init(20000, 110, 13000);
    uint32_t root, made[100];
    const std::vector<uint32_t> n(100, 1);
    CHECK(pages.create(&root, &err) == KvPages::OK && pages.step(1, &root, &len, nullptr, &copies, &err) == KvPages::OK);
    CHECK(pages.fork(root, 100, made, &err) == KvPages::OK);
    std::vector<KvStepSeq> plan;
    CHECK(pages.step(100, made, n.data(), &plan, &copies, &err) == KvPages::OK);
    KvPlan p;
    for (bool f32 : {false, true}) {
      kv_plan_shared(s, plan, pages, 1, f32, &p);
      CHECK(check_plan(s, pages, plan, p) > 0 && p.many.empty() == (len == 500));
      CHECK(kv_share_may_many(s, plan, pages.max_pages(), f32) && !kv_share_may_many(s, plan, 20, f32));
    }
  }
  // more sequences than are looked at
  {
    const KvShape s{2, 1, 64};
    KvPages pages;
    pages.init(8000, 1200, 1000);
    uint32_t root;
    std::vector<uint32_t> made(1100), n(1100, 1);
    CHECK(pages.create(&root, &err) == KvPages::OK);
    const uint32_t len = 500;
    CHECK(pages.step(1, &root, &len, nullptr, &copies, &err) == KvPages::OK);
    CHECK(pages.fork(root, 1100, made.data(), &err) == KvPages::OK);
    std::vector<KvStepSeq> plan;
    KvPlan p;
    for (size_t count : {KV_SHARE_SEQS, KV_SHARE_SEQS + 1}) {
      CHECK(pages.step(count, made.data(), n.data(), &plan, &copies, &err) == KvPages::OK);
      kv_plan_shared(s, plan, pages, 1, true, &p);
      const size_t read = check_plan(s, pages, plan, p);
      CHECK(count > KV_SHARE_SEQS ? read == count * 8 : read < count * 2);
    }
  }
  return 0;
}
