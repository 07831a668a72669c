// Runs the page bookkeeping and the step plans of the key/value cache
// (hale-token_amd/csrc/kv_pages.cpp) against a plain model: random creates,
// forks, copies, cuts, frees, steps and compactions over small pools, with every
// page's contents tracked as the copies move them.  Built with
// AddressSanitizer and UndefinedBehaviorSanitizer by tests/test_kv_pages.py.
// Prints "<operations> <refusals>"; exits 1 with a message on a difference.
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>

#include <algorithm>
#include <map>
#include <set>
#include <string>
#include <vector>

#include "kv_pages.h"

using namespace hale;

namespace {

uint64_t rng_state = 0x9E3779B97F4A7C15ull;
uint64_t next() {  // xorshift64*
  rng_state ^= rng_state >> 12;
  rng_state ^= rng_state << 25;
  rng_state ^= rng_state >> 27;
  return rng_state * 0x2545F4914F6CDD1Dull;
}
size_t below(size_t n) { return (size_t)(next() >> 11) % n; }

#define CHECK(cond)                                                 \
  do {                                                              \
    if (!(cond)) {                                                  \
      fprintf(stderr, "line %d: %s does not hold\n", __LINE__, #cond); \
      exit(1);                                                      \
    }                                                               \
  } while (0)

// A pool whose positions hold token numbers, and the model: each sequence's tokens.
struct World {
  KvPages p;
  std::vector<std::vector<uint64_t>> pool;
  std::vector<uint32_t> table;
  std::map<uint32_t, std::vector<uint64_t>> want;
  uint64_t token = 1;
  long refusals = 0;

  World(size_t pages, size_t seqs, size_t max_len) {
    p.init(pages, seqs, max_len);
    pool.assign(pages, std::vector<uint64_t>(KV_PAGE, 0));
    table.assign(seqs * p.max_pages(), 0);
  }
  // copies as one launch makes them: all sources read before any is written
  // must equal all at once, so no destination is a source or written twice
  void apply(const std::vector<KvCopy>& copies) {
    std::set<uint32_t> dst, src;
    for (const KvCopy& c : copies) {
      CHECK(c.src < pool.size() && c.dst < pool.size());
      CHECK(dst.insert(c.dst).second);
      src.insert(c.src);
    }
    for (uint32_t d : dst) CHECK(!src.count(d));
    for (const KvCopy& c : copies) pool[c.dst] = pool[c.src];
  }
  void send() {
    for (uint32_t i : p.dirty) table[i] = p.entry(i);
    p.dirty.clear();
  }
  void compare() {
    send();
    std::vector<uint32_t> refs(pool.size(), 0);
    for (auto& kv : want) {
      std::string err;
      size_t n = 0;
      CHECK(p.len(kv.first, &n, &err) == KvPages::OK && n == kv.second.size());
      for (size_t i = 0; i < n; i++) {
        const uint32_t page = table[kv.first * p.max_pages() + i / KV_PAGE];
        CHECK(page == p.page_of(kv.first, i));
        CHECK(pool[page][i % KV_PAGE] == kv.second[i]);
        if (i % KV_PAGE == 0) refs[page]++;
      }
    }
    size_t used = 0;
    for (size_t i = 0; i < pool.size(); i++) {
      CHECK(refs[i] == p.refs((uint32_t)i));
      used += refs[i] != 0;
    }
    CHECK(used == p.used());
  }
  uint32_t any() {
    auto it = want.begin();
    std::advance(it, below(want.size()));
    return it->first;
  }
};

void random_walk(size_t pages, size_t seqs, size_t max_len, long steps, long* ops, long* refusals) {
  World w(pages, seqs, max_len);
  std::string err;
  for (long k = 0; k < steps; k++) {
    const int what = (int)below(16);
    ++*ops;
    if (w.want.empty() || what == 0) {
      uint32_t s = 0;
      if (w.p.create(&s, &err) == KvPages::OK) {
        CHECK(!w.want.count(s) && s < seqs);
        w.want[s] = {};
      } else {
        CHECK(w.want.size() == seqs);
        ++*refusals;
      }
    } else if (what == 1) {
      const uint32_t s = w.any();
      CHECK(w.p.free(s, &err) == KvPages::OK);
      CHECK(w.p.free(s, &err) == KvPages::BAD);
      w.want.erase(s);
    } else if (what == 2) {
      const uint32_t s = w.any();
      const size_t n = below(4);
      uint32_t out[4];
      if (w.p.fork(s, n, out, &err) == KvPages::OK) {
        for (size_t i = 0; i < n; i++) {
          CHECK(!w.want.count(out[i]));
          w.want[out[i]] = w.want[s];
        }
      } else {
        CHECK(w.want.size() + n > seqs);
        ++*refusals;
      }
    } else if (what == 3) {
      const uint32_t s = w.any();
      uint32_t out = 0;
      std::vector<KvCopy> c;
      if (w.p.copy(s, &out, &c, &err) == KvPages::OK) {
        w.apply(c);
        w.want[out] = w.want[s];
      } else {
        CHECK(c.empty());
        ++*refusals;
      }
    } else if (what == 4) {
      const uint32_t s = w.any();
      const size_t n = below(w.want[s].size() + 1);
      CHECK(w.p.truncate(s, w.want[s].size() + 1, &err) == KvPages::BAD);
      CHECK(w.p.truncate(s, n, &err) == KvPages::OK);
      w.want[s].resize(n);
    } else if (what == 5) {
      std::vector<KvCopy> c;
      w.p.compact(&c);
      w.apply(c);
      for (size_t i = 0; i < pages; i++) CHECK((w.p.refs((uint32_t)i) != 0) == (i < w.p.used()));
    } else {
      std::vector<uint32_t> ids, n;
      for (auto& kv : w.want)
        if (below(2)) {
          ids.push_back(kv.first);
          n.push_back((uint32_t)(below(4) ? below(20) : below(200)));
        }
      std::vector<KvStepSeq> plan;
      std::vector<KvCopy> c;
      const KvPages::Status can = w.p.check_step(ids.size(), ids.data(), n.data(), &err);
      const KvPages::Status st = w.p.step(ids.size(), ids.data(), n.data(), &plan, &c, &err);
      CHECK(can == st);
      if (st == KvPages::OK) {
        w.apply(c);
        w.send();
        uint32_t tok = 0;
        for (size_t i = 0; i < ids.size(); i++) {
          CHECK(plan[i].row == ids[i] && plan[i].len0 == w.want[ids[i]].size() && plan[i].ntok == n[i] && plan[i].tok0 == tok);
          for (uint32_t t = 0; t < n[i]; t++) {
            const size_t pos = w.want[ids[i]].size();
            const uint32_t page = w.table[ids[i] * w.p.max_pages() + pos / KV_PAGE];
            CHECK(w.p.refs(page) == 1);  // nobody else sees what the step stores
            w.pool[page][pos % KV_PAGE] = w.token;
            w.want[ids[i]].push_back(w.token++);
          }
          tok += n[i];
        }
      } else {
        CHECK(c.empty());
        ++*refusals;
      }
    }
    w.compare();
  }
}

// Every row of every sequence meets every page that it sees exactly once, and
// the counts stay within what the buffers are sized for.
void plans() {
  for (int k = 0; k < 3000; k++) {
    KvShape s{};
    s.kv_heads = 1 + below(8);
    s.heads = s.kv_heads * (1 + below(below(4) ? 8 : 40));
    s.head_dim = 16 * (1 + below(16));
    std::vector<KvStepSeq> seqs(below(below(3) ? 4 : 40));
    uint32_t tok = 0;
    for (auto& q : seqs) {
      q = {(uint32_t)(&q - seqs.data()), (uint32_t)(below(3) ? below(3000) : below(200000)), (uint32_t)(below(2) ? below(8) : below(400)), tok};
      tok += q.ntok;
    }
    const size_t window = below(2) ? 0 : 1 + below(below(2) ? 100 : 5000);
    KvPlan plan;
    const bool f32 = below(2);
    kv_plan(s, seqs, window, f32, &plan);
    const size_t limit = kv_few_limit(s, seqs, f32);
    CHECK(limit >= 16 && limit <= 64 && (s.head_dim <= 128 || limit == 16));
    CHECK(plan.cols >= 1 && 16 * (size_t)plan.cols <= kv_few_rows(s.head_dim));
    CHECK(plan.few.size() + plan.many.size() <= kv_max_items(s, tok, seqs.size()));
    CHECK(plan.few_joins.size() + plan.many_joins.size() + KV_MAX_PARTS <= kv_max_items(s, tok, seqs.size()));
    CHECK(plan.part_rows <= kv_part_rows(s.head_dim));
    // every new token is in one block, at its position, and no other is
    std::vector<KvBlock> blocks;
    const size_t max_pages = 4096;
    kv_blocks(seqs, max_pages, &blocks);
    CHECK(blocks.size() <= kv_max_blocks(tok, seqs.size()));
    std::vector<int> seen(tok, 0);
    for (const KvBlock& b : blocks) {
      const KvStepSeq& q = seqs[b.entry / max_pages];
      CHECK(b.block < 4 && b.old < b.end && b.end <= KV_BLOCK);
      const size_t pos = b.entry % max_pages * KV_PAGE + b.block * KV_BLOCK;
      CHECK(b.old == (q.len0 > pos ? q.len0 - pos : 0));
      for (int j = b.old; j < b.end; j++) {
        const long long t = (long long)b.tok + j;
        CHECK(t == (long long)q.tok0 + (long long)(pos + j) - q.len0 && t >= q.tok0 && t < (long long)q.tok0 + q.ntok);
        seen[t]++;
      }
    }
    for (int n : seen) CHECK(n == 1);
    std::map<std::pair<std::pair<uint32_t, uint32_t>, uint32_t>, std::vector<const KvItem*>> tiles;
    for (int kind = 0; kind < 2; kind++)
      for (const KvItem& it : kind ? plan.many : plan.few) {
        CHECK(it.row < seqs.size() && it.len0 == seqs[it.row].len0 && it.tok0 == seqs[it.row].tok0);
        const size_t all = seqs[it.row].ntok * s.group(), tile = kind ? kv_many_rows(s.head_dim) : 16 * (size_t)plan.cols;
        CHECK((all > limit) == (kind == 1));
        CHECK(it.head < s.kv_heads && it.rows >= 1 && it.rows <= tile);
        CHECK(it.row0 % tile == 0 && it.row0 + it.rows <= all && (it.rows == tile || it.row0 + it.rows == all));
        CHECK(it.page0 < it.page1);
        tiles[{{it.row, it.head}, it.row0}].push_back(&it);
      }
    size_t want = 0;
    for (auto& q : seqs) {
      const size_t all = q.ntok * s.group(), tile = all > limit ? kv_many_rows(s.head_dim) : kv_few_rows(s.head_dim);
      want += (all + tile - 1) / tile * s.kv_heads;
    }
    CHECK(tiles.size() == want);
    std::vector<char> taken(plan.part_rows, 0);  // rows of partial results, each written by one item
    std::map<uint32_t, const KvJoin*> joins;
    for (int kind = 0; kind < 2; kind++)
    for (const KvJoin& j : kind ? plan.many_joins : plan.few_joins) {
      CHECK(j.step == (kind ? kv_many_rows(s.head_dim) : 16 * (size_t)plan.cols));
      CHECK(j.parts > 1 && j.parts <= 2 * KV_FEW_GROUPS && j.parts <= 2 * KV_MANY_GROUPS && j.rows <= j.step);
      joins[j.part0] = &j;
    }
    size_t divided = 0;
    for (auto& t : tiles) {
      auto& v = t.second;
      const KvStepSeq& q = seqs[v[0]->row];
      std::sort(v.begin(), v.end(), [](const KvItem* a, const KvItem* b) { return a->page0 < b->page0; });
      const size_t low = q.len0 + v[0]->row0 / s.group(), high = q.len0 + (v[0]->row0 + v[0]->rows - 1) / s.group();
      CHECK(v.back()->page1 == high / KV_PAGE + 1);
      CHECK(v[0]->page0 == (window && low + 1 > window ? (low + 1 - window) / KV_PAGE : 0));
      const KvJoin* j = v.size() > 1 ? joins.at(v[0]->part) : nullptr;
      if (j) {
        divided++;
        CHECK(j->parts == v.size() && j->tok0 == v[0]->tok0 && j->head == v[0]->head && j->row0 == v[0]->row0 && j->rows == v[0]->rows);
      }
      for (size_t i = 0; i < v.size(); i++) {
        if (i) CHECK(v[i]->page0 == v[i - 1]->page1);
        if (!j) {
          CHECK(v[i]->part == KV_WHOLE);
          continue;
        }
        CHECK(v[i]->part == j->part0 + i * j->step && v[i]->part + v[i]->rows <= plan.part_rows);
        for (uint32_t r = 0; r < v[i]->rows; r++) CHECK(!taken[v[i]->part + r]++);
      }
    }
    CHECK(divided == plan.few_joins.size() + plan.many_joins.size());
  }
}

void refusals() {
  KvPages p;
  p.init(4, 2, 200);
  std::string err;
  uint32_t a = 9, b = 9, c = 9, out[2];
  CHECK(p.create(&a, &err) == KvPages::OK && p.create(&b, &err) == KvPages::OK);
  CHECK(p.create(&c, &err) == KvPages::FULL && !err.empty());
  CHECK(p.free(7, &err) == KvPages::BAD && p.truncate(7, 0, &err) == KvPages::BAD && p.fork(7, 1, out, &err) == KvPages::BAD);
  CHECK(p.fork(a, 1, out, &err) == KvPages::FULL);
  CHECK(p.copy(a, out, nullptr, &err) == KvPages::FULL);
  std::vector<KvStepSeq> plan;
  std::vector<KvCopy> copies;
  const uint32_t twice[2] = {a, a}, both[2] = {a, b}, one[2] = {1, 1}, over[2] = {1, 201}, many[2] = {100, 200};
  CHECK(p.step(2, twice, one, &plan, &copies, &err) == KvPages::BAD);
  CHECK(p.step(2, both, over, &plan, &copies, &err) == KvPages::BAD);
  CHECK(p.step(2, both, many, &plan, &copies, &err) == KvPages::FULL && p.used() == 0);
  const uint32_t gone[1] = {5};
  CHECK(p.step(1, gone, one, &plan, &copies, &err) == KvPages::BAD);
  CHECK(p.step(2, both, one, &plan, &copies, &err) == KvPages::OK && p.used() == 2);
  CHECK(p.free(b, &err) == KvPages::OK && p.fork(a, 1, out, &err) == KvPages::OK);
  // three pages are free: both sharers growing over a page needs the copy and two more
  const uint32_t sharers[2] = {a, out[0]}, wide[2] = {100, 100}, wider[2] = {120, 130};
  CHECK(p.step(2, sharers, wider, &plan, &copies, &err) == KvPages::FULL && p.refs(0) == 2);
  CHECK(p.step(2, sharers, wide, &plan, &copies, &err) == KvPages::OK && copies.size() == 1 && p.used() == 4);
}

}  // namespace

// Forks that are freed again without a step between do not pile up changes.
void forks_without_steps() {
  KvPages p;
  p.init(64, 8, 64 * KV_PAGE);
  std::string err;
  std::vector<KvCopy> copies;
  uint32_t a = 0, f = 0;
  CHECK(p.create(&a, &err) == KvPages::OK);
  const uint32_t n = 60 * KV_PAGE;
  CHECK(p.step(1, &a, &n, nullptr, &copies, &err) == KvPages::OK);
  for (int k = 0; k < 20000; k++) {
    CHECK(p.fork(a, 1, &f, &err) == KvPages::OK);
    if (k < 19999) CHECK(p.free(f, &err) == KvPages::OK);
    CHECK(p.dirty.size() <= 200000);
  }
  std::vector<char> said(8 * 64, 0);  // every entry that holds a page is among the changes
  for (uint32_t d : p.dirty) said[d] = 1;
  for (uint32_t j = 0; j < 60; j++) CHECK(said[a * 64 + j] && said[f * 64 + j]);
}

int main() {
  long ops = 0, refused = 0;
  refusals();
  forks_without_steps();
  plans();
  random_walk(12, 6, 300, 6000, &ops, &refused);
  random_walk(40, 9, 1000, 6000, &ops, &refused);
  random_walk(3, 5, 70, 6000, &ops, &refused);
  printf("%ld %ld\n", ops, refused);
  return 0;
}
