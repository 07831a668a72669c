// kv_pages.cpp -- page bookkeeping and step plans of the key/value cache.
#include "kv_pages.h"

#include <algorithm>
#include <cstdio>

namespace hale {

namespace {

KvPages::Status refuse(std::string* err, KvPages::Status s, const char* fmt, size_t a, size_t b = 0, size_t c = 0) {
  char buf[192];
  std::snprintf(buf, sizeof buf, fmt, a, b, c);
  *err = buf;
  return s;
}

size_t ceil_div(size_t a, size_t b) { return (a + b - 1) / b; }

}  // namespace

void KvPages::init(size_t pages, size_t max_seqs, size_t max_len) {
  max_len_ = max_len;
  max_pages_ = ceil_div(max_len, KV_PAGE);
  refs_.assign(pages, 0);
  free_.resize(pages);
  for (size_t i = 0; i < pages; i++) free_[i] = (uint32_t)(pages - 1 - i);  // the lowest is taken first
  seqs_.resize(max_seqs);
  for (Seq& s : seqs_) s.pages.reserve(max_pages_ < 64 ? max_pages_ : 64);
  free_seqs_.resize(max_seqs);
  for (size_t i = 0; i < max_seqs; i++) free_seqs_[i] = (uint32_t)(max_seqs - 1 - i);
  mark_.assign(max_seqs, 0);
}

KvPages::Status KvPages::find(uint32_t seq, std::string* err) const {
  if (live(seq)) return OK;
  return refuse(err, BAD, "no sequence %zu", seq);
}

uint32_t KvPages::take() {
  const uint32_t p = free_.back();
  free_.pop_back();
  refs_[p] = 1;
  return p;
}

void KvPages::drop(uint32_t page) {
  if (--refs_[page] == 0) free_.push_back(page);
}

void KvPages::set(uint32_t seq, size_t index) { dirty.push_back((uint32_t)(seq * max_pages_ + index)); }

KvPages::Status KvPages::create(uint32_t* seq, std::string* err) {
  if (free_seqs_.empty()) return refuse(err, FULL, "all %zu sequences are in use", seqs_.size());
  *seq = free_seqs_.back();
  free_seqs_.pop_back();
  Seq& s = seqs_[*seq];
  s.live = true;
  s.len = 0;
  s.pages.clear();
  return OK;
}

KvPages::Status KvPages::free(uint32_t seq, std::string* err) {
  const Status st = find(seq, err);
  if (st) return st;
  free_seqs_.push_back(seq);  // reserved at init: holds every sequence
  Seq& s = seqs_[seq];
  for (uint32_t p : s.pages) drop(p);
  s.pages.clear();
  s.live = false;
  s.len = 0;
  return OK;
}

KvPages::Status KvPages::fork(uint32_t seq, size_t n, uint32_t* out, std::string* err) {
  const Status st = find(seq, err);
  if (st) return st;
  if (n > free_seqs_.size()) return refuse(err, FULL, "%zu forks, but only %zu of %zu sequences are free", n, free_seqs_.size(), seqs_.size());
  const size_t np = seqs_[seq].pages.size();
  dirty.reserve(dirty.size() + n * np);
  for (size_t i = 0; i < n; i++) seqs_[free_seqs_[free_seqs_.size() - 1 - i]].pages.reserve(np);
  if (dirty.size() > settled_) {  // forks without a step between: each entry once
    std::sort(dirty.begin(), dirty.end());
    dirty.erase(std::unique(dirty.begin(), dirty.end()), dirty.end());
    settled_ = 2 * dirty.size() + 65536;
  }
  for (size_t i = 0; i < n; i++) {
    uint32_t id = 0;
    (void)create(&id, err);
    Seq& s = seqs_[id];
    s.pages = seqs_[seq].pages;
    s.len = seqs_[seq].len;
    for (size_t j = 0; j < np; j++) {
      refs_[s.pages[j]]++;
      set(id, j);
    }
    out[i] = id;
  }
  return OK;
}

KvPages::Status KvPages::copy(uint32_t seq, uint32_t* out, std::vector<KvCopy>* copies, std::string* err) {
  const Status st = find(seq, err);
  if (st) return st;
  const size_t np = seqs_[seq].pages.size();
  if (np > free_.size()) return refuse(err, FULL, "a copy of %zu pages, but only %zu of %zu are free", np, free_.size(), refs_.size());
  if (free_seqs_.empty()) return refuse(err, FULL, "all %zu sequences are in use", seqs_.size());
  dirty.reserve(dirty.size() + np);
  copies->reserve(copies->size() + np);
  seqs_[free_seqs_.back()].pages.reserve(np);
  (void)create(out, err);
  Seq& s = seqs_[*out];
  s.len = seqs_[seq].len;
  for (size_t j = 0; j < np; j++) {
    const uint32_t p = take();
    s.pages.push_back(p);
    copies->push_back({seqs_[seq].pages[j], p});
    set(*out, j);
  }
  return OK;
}

KvPages::Status KvPages::truncate(uint32_t seq, size_t len, std::string* err) {
  const Status st = find(seq, err);
  if (st) return st;
  Seq& s = seqs_[seq];
  if (len > s.len) return refuse(err, BAD, "sequence %zu holds %zu positions, not %zu", seq, s.len, len);
  while (s.pages.size() > ceil_div(len, KV_PAGE)) {
    drop(s.pages.back());
    s.pages.pop_back();
  }
  s.len = len;
  return OK;
}

KvPages::Status KvPages::len(uint32_t seq, size_t* len, std::string* err) const {
  const Status st = find(seq, err);
  if (st) return st;
  *len = seqs_[seq].len;
  return OK;
}

KvPages::Status KvPages::check_step(size_t nseq, const uint32_t* seqs, const uint32_t* ntok, std::string* err) {
  if (++stamp_ == 0) {  // wrapped: no mark may equal the new stamp
    std::fill(mark_.begin(), mark_.end(), 0u);
    stamp_ = 1;
  }
  need_ = copies_ = 0;
  for (size_t i = 0; i < nseq; i++) {
    const Status st = find(seqs[i], err);
    if (st) return st;
    if (mark_[seqs[i]] == stamp_) return refuse(err, BAD, "sequence %zu twice in one step", seqs[i]);
    mark_[seqs[i]] = stamp_;
    const Seq& s = seqs_[seqs[i]];
    if (ntok[i] > max_len_ - s.len)
      return refuse(err, BAD, "sequence %zu: context overflow, %zu positions needed, at most %zu", seqs[i], s.len + ntok[i], max_len_);
    need_ += ceil_div(s.len + ntok[i], KV_PAGE) - s.pages.size();
  }
  // Shared pages that are written to.  Of k sequences of this step on a page
  // that r sequences hold, k copy it where r > k; where r == k the last one
  // writes in place.  Counted by taking the references off and putting them back.
  for (size_t i = 0; i < nseq; i++) {
    const Seq& s = seqs_[seqs[i]];
    if (ntok[i] && s.len % KV_PAGE && refs_[s.pages.back()] > 1) {
      refs_[s.pages.back()]--;
      copies_++;
      mark_[seqs[i]] = 0;  // copies
    }
  }
  for (size_t i = 0; i < nseq; i++)
    if (mark_[seqs[i]] == 0) refs_[seqs_[seqs[i]].pages.back()]++;
  need_ += copies_;
  if (need_ > free_.size()) return refuse(err, FULL, "%zu pages needed, but only %zu of %zu are free", need_, free_.size(), refs_.size());
  return OK;
}

void KvPages::preview(size_t nseq, const uint32_t* seqs, const uint32_t* ntok, std::vector<KvStepSeq>* plan) const {
  plan->resize(nseq);
  uint32_t tok0 = 0;
  for (size_t i = 0; i < nseq; i++) {
    (*plan)[i] = {seqs[i], (uint32_t)seqs_[seqs[i]].len, ntok[i], tok0};
    tok0 += ntok[i];
  }
}

void KvPages::reserve_step(size_t nseq, const uint32_t* seqs, const uint32_t* ntok, std::vector<KvCopy>* copies) {
  copies->reserve(copies->size() + copies_);
  dirty.reserve(dirty.size() + need_);
  for (size_t i = 0; i < nseq; i++) {
    Seq& s = seqs_[seqs[i]];
    s.pages.reserve(ceil_div(s.len + ntok[i], KV_PAGE));
  }
}

KvPages::Status KvPages::step(size_t nseq, const uint32_t* seqs, const uint32_t* ntok, std::vector<KvStepSeq>* plan,
                              std::vector<KvCopy>* copies, std::string* err) {
  const Status st = check_step(nseq, seqs, ntok, err);
  if (st) return st;
  if (plan) preview(nseq, seqs, ntok, plan);
  reserve_step(nseq, seqs, ntok, copies);
  for (size_t i = 0; i < nseq; i++) {
    Seq& s = seqs_[seqs[i]];
    if (mark_[seqs[i]] == 0) {
      const uint32_t p = take();
      copies->push_back({s.pages.back(), p});
      refs_[s.pages.back()]--;  // others hold it: it never becomes free here
      s.pages.back() = p;
      set(seqs[i], s.pages.size() - 1);
    }
    s.len += ntok[i];
    while (s.pages.size() * KV_PAGE < s.len) {
      s.pages.push_back(take());
      set(seqs[i], s.pages.size() - 1);
    }
  }
  return OK;
}

void KvPages::compact_size(size_t* moved, size_t* entries) const {
  const size_t n = used();
  *moved = *entries = 0;
  for (size_t p = n; p < refs_.size(); p++) *moved += refs_[p] != 0;
  if (*moved == 0) return;
  for (const Seq& s : seqs_)
    for (uint32_t p : s.pages) *entries += p >= n;
}

void KvPages::compact(std::vector<KvCopy>* copies) {
  const size_t n = used();
  std::vector<uint32_t> to(refs_.size());
  size_t hole = 0, moved = 0, entries = 0;
  compact_size(&moved, &entries);
  copies->reserve(copies->size() + moved);
  dirty.reserve(dirty.size() + entries);
  for (size_t p = n; p < refs_.size(); p++) {
    if (!refs_[p]) continue;
    while (refs_[hole]) hole++;
    to[p] = (uint32_t)hole;
    copies->push_back({(uint32_t)p, (uint32_t)hole});
    refs_[hole] = refs_[p];
    refs_[p] = 0;
  }
  for (uint32_t id = 0; id < seqs_.size(); id++)
    for (size_t j = 0; j < seqs_[id].pages.size(); j++)
      if (seqs_[id].pages[j] >= n) {
        seqs_[id].pages[j] = to[seqs_[id].pages[j]];
        set(id, j);
      }
  free_.clear();  // keeps its room
  for (size_t p = refs_.size(); p > n; p--) free_.push_back((uint32_t)(p - 1));
}

void KvPages::resize(size_t pages) {
  const size_t n = used();
  std::vector<uint32_t> refs(pages, 0), rest;
  rest.reserve(pages);  // drop() never allocates
  std::copy(refs_.begin(), refs_.begin() + n, refs.begin());
  for (size_t p = pages; p > n; p--) rest.push_back((uint32_t)(p - 1));
  refs_.swap(refs);
  free_.swap(rest);
}

namespace {

struct Tile {
  const KvStepSeq* q;
  uint32_t head, row0, rows, page0, page1;
};

// Tiles into items of at most `each` pages, and the joins of those divided.
void divide(const std::vector<Tile>& tiles, size_t each, size_t step, std::vector<KvItem>* items, std::vector<KvJoin>* joins,
            uint32_t* part_rows) {
  for (const Tile& t : tiles) {
    const size_t n = t.page1 - t.page0, parts = ceil_div(n, each);
    if (parts > 1)
      joins->push_back({t.q->tok0, (uint16_t)t.head, (uint16_t)t.rows, t.row0, *part_rows, (uint32_t)parts, (uint32_t)step, {0, 0}});
    for (size_t k = 0; k < parts; k++) {
      items->push_back({t.q->row, t.q->len0, t.q->tok0, (uint16_t)t.head, (uint16_t)t.rows, t.row0,
                        (uint32_t)(t.page0 + n * k / parts), (uint32_t)(t.page0 + n * (k + 1) / parts),
                        parts > 1 ? *part_rows : KV_WHOLE});
      if (parts > 1) *part_rows += (uint32_t)step;
    }
  }
}

size_t count_pages(const std::vector<Tile>& tiles) {
  size_t total = 0;
  for (const Tile& t : tiles) total += t.page1 - t.page0;
  return total;
}

// Most pages of an item of many rows.  The work-groups that run at once take the
// items in rounds; with the longest tile cut into 1, 2, .. parts, the time is about
// the rounds times an item's mean pages (at least the longest item), and a
// part costs about four pages for its partial result.  The cut of the least time
// (4 heads of 128, bf16: 300 tokens behind 8000 67.6 us, uncut 214.6; 64 behind 16000 39.4,
// uncut 404.9; 2048 behind 4000 are not cut).
size_t many_each(const std::vector<Tile>& tiles) {
  const size_t total = count_pages(tiles), least = ceil_div(total, KV_MANY_GROUPS);
  size_t longest = 0, best = 0;
  for (const Tile& t : tiles) longest = std::max<size_t>(longest, t.page1 - t.page0);
  double best_time = 0;
  for (size_t cut = 1; cut <= 64; cut++) {
    const size_t each = std::max<size_t>(4, ceil_div(longest, cut));
    if (cut > 1 && each < least) break;
    size_t items = 0, parts = 0;
    for (const Tile& t : tiles) {
      const size_t n = ceil_div(t.page1 - t.page0, each);
      items += n;
      parts += n > 1 ? n : 0;
    }
    if (parts > 2 * KV_MANY_GROUPS) break;
    const double mean = (double)(total + 4 * parts) / (double)items;
    const double time = std::max((double)each, (double)ceil_div(items, KV_MANY_GROUPS) * mean) + (parts ? 4 : 0);
    if (cut == 1 || time < best_time) {
      best = each;
      best_time = time;
    }
    if (each == 4) break;
  }
  return best;
}

// Work-group i runs on accelerator die i % 8, each of which has its own L2: the
// items of one sequence and head, which read the same pages, go to one die (or
// as few as keep all eight busy), the longest first.  That holds while all eight lists have
// items: for 1, 2, 4 or a multiple of 8 streams of as many items.  Where lists are empty or
// run out, the rest of the others goes over all dies, still the longest first, which keeps
// the dies equally busy (bf16, 4 heads of 128: 2048 tokens
// behind 4000 192 us, 225 in the order of the tiles; two prompts of 1000 36.5, 45.1).
void spread(std::vector<KvItem>* items) {
  constexpr size_t DIES = 8;
  if (items->size() < 2 * DIES) return;
  size_t streams = 0;
  std::vector<std::vector<KvItem>> die(DIES);
  std::vector<size_t> first;  // items of a stream lie one behind the other
  for (size_t i = 0; i < items->size(); i++)
    if (i == 0 || (*items)[i].tok0 != (*items)[i - 1].tok0 || (*items)[i].head != (*items)[i - 1].head) {
      streams++;
      first.push_back(i);
    }
  first.push_back(items->size());
  const size_t share = streams < DIES ? DIES / streams : 1;  // dies per stream
  for (size_t s = 0; s < streams; s++)
    for (size_t i = first[s]; i < first[s + 1]; i++) die[(s * share + (i - first[s]) % share) % DIES].push_back((*items)[i]);
  for (auto& d : die) {
    std::stable_sort(d.begin(), d.end(), [](const KvItem& a, const KvItem& b) { return a.page1 - a.page0 > b.page1 - b.page0; });
    // all of them running at once, two to a compute unit: a long one beside a short one
    if (d.size() <= KV_MANY_GROUPS / DIES) std::reverse(d.begin() + (d.size() + 1) / 2, d.end());
  }
  size_t n = 0;
  for (size_t k = 0; n < items->size(); k++)
    for (auto& d : die)
      if (k < d.size()) (*items)[n++] = d[k];
}

}  // namespace

// A work-group of few rows reads its pages for up to 32 rows, one of many for up to 128, of
// which the missing ones cost as much; but few rows run on four times as many pages at
// once.  So few rows while their tiles leave compute units idle (4 heads of 128, 8
// rows a token, few / many: bf16 of 64 rows, 1 sequence of 8000 = 8 tiles 15.5 / 21.9 us,
// 2 of 4000 15.8 / 16.9, 4 of 4000 = 32 tiles 27.2 / 20.4; 24 rows, 4 of 4000 16.3 / 19.0,
// 8 of 4000 26.4 / 21.1, 32 of 2000 42.1 / 26.4).  In f32, whose products are doubled,
// the missing rows cost more: 32 rows at any number (8 of 4000 33.2 / 39.5), 64 as
// above (2 of 4000 17.4 / 22.3, 4 31.1 / 25.5).
size_t kv_few_limit(const KvShape& s, const std::vector<KvStepSeq>& seqs, bool f32) {
  const size_t group = s.group(), rows = kv_few_rows(s.head_dim);
  if (rows == 16) return 16;
  size_t tiles = 0;
  for (const KvStepSeq& q : seqs)
    if (q.ntok * group <= 64) tiles += ceil_div(q.ntok * group, rows) * s.kv_heads;
  return tiles < 32 ? 64 : f32 ? 32 : 16;
}

void kv_plan(const KvShape& s, const std::vector<KvStepSeq>& seqs, size_t window, bool f32, KvPlan* out) {
  out->few.clear();
  out->many.clear();
  out->few_joins.clear();
  out->many_joins.clear();
  out->part_rows = 0;
  const size_t group = s.group(), few_rows = kv_few_rows(s.head_dim), many_rows = kv_many_rows(s.head_dim);
  const size_t limit = kv_few_limit(s, seqs, f32);
  size_t most = 0;
  for (const KvStepSeq& q : seqs)
    if (q.ntok * group <= limit) most = std::max(most, q.ntok * group);
  // a second group of 16 rows costs though it be empty: 32 bf16 sequences of 4000, 8 rows
  // each, 33.6 us with one, 44.0 with two
  out->cols = most <= 16 ? 1 : 2;
  std::vector<Tile> few, many;
  for (const KvStepSeq& q : seqs) {
    const bool is_few = q.ntok * group <= limit;
    const size_t rows = is_few ? few_rows : many_rows;
    for (uint32_t h = 0; h < s.kv_heads; h++)
      // the rows with the most pages first, so that the last work-groups are short
      for (size_t t = ceil_div(q.ntok * group, rows); t-- > 0;) {
        const size_t r = t * rows, n = std::min(rows, q.ntok * group - r);
        const size_t low = q.len0 + r / group, high = q.len0 + (r + n - 1) / group;
        const size_t page0 = window && low + 1 > window ? (low + 1 - window) / KV_PAGE : 0;
        (is_few ? few : many).push_back({&q, h, (uint32_t)r, (uint32_t)n, (uint32_t)page0, (uint32_t)(high / KV_PAGE + 1)});
      }
  }
  // few rows: a work-group's waves take a page each, fewer than four leave some idle; eight
  // pages at least instead of four take longer (1 x 4096 f32 12.9 us for 11.2), as do
  // 256 or 1024 groups for 512 (32 of 200 to 8000 40.7 and 41.5 us for 39.5, one of
  // 131000 30.0 and 38.2 for 31.1)
  divide(few, std::max<size_t>(4, ceil_div(count_pages(few), KV_FEW_GROUPS)), 16 * (size_t)out->cols, &out->few, &out->few_joins,
         &out->part_rows);
  if (!many.empty()) divide(many, many_each(many), many_rows, &out->many, &out->many_joins, &out->part_rows);
  spread(&out->many);
}

void kv_blocks(const std::vector<KvStepSeq>& seqs, size_t max_pages, std::vector<KvBlock>* out) {
  out->clear();
  for (const KvStepSeq& q : seqs) {
    if (!q.ntok) continue;
    const uint32_t end = q.len0 + q.ntok;
    for (uint32_t b = q.len0 / KV_BLOCK; b * KV_BLOCK < end; b++) {
      const uint32_t pos = b * KV_BLOCK;
      out->push_back({(uint32_t)(q.row * max_pages + pos / KV_PAGE), (int32_t)(q.tok0 + pos - q.len0),
                      (uint8_t)(pos % KV_PAGE / KV_BLOCK), (uint8_t)(q.len0 > pos ? q.len0 - pos : 0),
                      (uint8_t)(end - pos < KV_BLOCK ? end - pos : KV_BLOCK), 0, 0});
    }
  }
}

size_t kv_max_items(const KvShape& s, size_t tokens, size_t nseq) {
  // tiles of 16 rows or more, one more per sequence for the last, and the further parts of divided ones
  return (tokens * s.group() / 16 + nseq) * s.kv_heads + KV_MAX_PARTS;
}

}  // namespace hale
