// kv_pages.h -- the pages of a key/value cache and the plan of one step over
// it: which page holds which positions of which sequence, how many sequences
// share it, and how the attention of a step is divided.  Host-only C++: no
// entry here touches the device; what has to move there is returned as lists.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <string>
#include <vector>

#include "../../include/hale_moe.h"

namespace hale {

constexpr size_t KV_PAGE = 64;   // positions per page (HALE_KV_PAGE)
constexpr size_t KV_BLOCK = 16;  // positions per scale (HALE_KV_BLOCK)

// One sequence's share of a step, as the kernels read it.
struct KvStepSeq {
  uint32_t row;    // its row of the page table
  uint32_t len0;   // positions held before the step
  uint32_t ntok;   // new tokens
  uint32_t tok0;   // the first one's index among the step's tokens
};

// A block of 16 positions that the step's tokens touch: positions old .. end -
// 1 of it are new, the one at j is token tok + j.
struct KvBlock {
  uint32_t entry;  // of its page in the page table
  int32_t tok;     // may be negative
  uint8_t block;   // of the page: 0..3
  uint8_t old, end, pad;
  uint32_t pad2;
};

// One work-group's share of the attention: rows row0 .. row0 + rows - 1 of a
// sequence's queries of one key/value head (row r is token r / group, head
// r % group of the group) over pages page0 .. page1 - 1.
struct KvItem {
  uint32_t row;    // of the page table
  uint32_t len0, tok0;  // as in KvStepSeq
  uint16_t head, rows;
  uint32_t row0;
  uint32_t page0, page1;
  uint32_t part;  // the first of its rows among the partial results, or KV_WHOLE
};
constexpr uint32_t KV_WHOLE = 0xffffffffu;

// Partial results of `rows` rows to be joined: `parts` of them, part0, part0 +
// step, .. their first rows.
struct KvJoin {
  uint32_t tok0;
  uint16_t head, rows;
  uint32_t row0;
  uint32_t part0, parts, step;
  uint32_t pad[2];
};

// The attention of a step under one window: sequences of few rows (the waves of
// a work-group share their pages) and of many (the waves share their rows).
struct KvPlan {
  int cols = 1;  // few: groups of 16 rows per work-group, 1 or 2
  std::vector<KvItem> few, many;
  std::vector<KvJoin> few_joins, many_joins;
  uint32_t part_rows = 0;
};

struct KvCopy {
  uint32_t src, dst;
};

// The plans that a cache keeps: of each window, for f32 and for the half types.
constexpr int KV_MAX_VIEWS = 2 * HALE_KV_MAX_WINDOWS;
// Pieces that a step's upload is put together from, at most: its counts, positions and
// blocks, and the counts, items and joins (of few and of many rows) of each view.
constexpr int KV_STEP_PIECES = 3, KV_VIEW_PIECES = 5;
constexpr int KV_MAX_PIECES = KV_STEP_PIECES + KV_MAX_VIEWS * KV_VIEW_PIECES;

struct KvShape {
  size_t heads, kv_heads, head_dim;
  size_t group() const { return heads / kv_heads; }
};

// Work-groups that a step's attention is divided into where its length allows,
// for few and for many rows apart.  A tile of pages that is divided has more
// than total / groups of them, so there are at most twice as many parts.
constexpr size_t KV_FEW_GROUPS = 512, KV_MANY_GROUPS = 512;
constexpr size_t KV_MAX_PARTS = 2 * (KV_FEW_GROUPS + KV_MANY_GROUPS);

// Rows per work-group of the kernel of few rows, at most, and of that of many.
inline size_t kv_few_rows(size_t head_dim) { return head_dim <= 128 ? 32 : 16; }
inline size_t kv_many_rows(size_t head_dim) { return head_dim <= 128 ? 128 : 64; }
inline size_t kv_part_rows(size_t head_dim) {
  return 2 * KV_FEW_GROUPS * kv_few_rows(head_dim) + 2 * KV_MANY_GROUPS * kv_many_rows(head_dim);
}

// Most rows of a sequence that the kernel of few rows takes in this step (f32: type of
// queries and results).  Of tokens per sequence only, so that a captured launch
// holds for all later steps of as many.
size_t kv_few_limit(const KvShape& s, const std::vector<KvStepSeq>& seqs, bool f32);

// Divides the attention of a step: tiles of rows, and few enough pages each
// that all compute units take part.  Window 0 sees every earlier position.
void kv_plan(const KvShape& s, const std::vector<KvStepSeq>& seqs, size_t window, bool f32, KvPlan* out);

// Positions that one launch of the reading kernel takes of those first .. first + count - 1: its
// grid has a work-group of 256 threads per page, and counts threads in 32 bits.
inline size_t kv_read_part(size_t first, size_t count) {
  constexpr size_t pages = (1u << 24) - 1;
  const size_t most = (first / KV_PAGE + pages) * KV_PAGE - first;
  return count < most ? count : most;
}

// The blocks that a step's tokens touch.
void kv_blocks(const std::vector<KvStepSeq>& seqs, size_t max_pages, std::vector<KvBlock>* out);

// Most items (of both kinds together) and blocks that a plan of so many tokens and
// sequences can have.
size_t kv_max_items(const KvShape& s, size_t tokens, size_t nseq);
inline size_t kv_max_blocks(size_t tokens, size_t nseq) { return tokens / KV_BLOCK + 2 * nseq; }

// The pool's pages, their owners and the sequences.
class KvPages {
 public:
  // Throws std::bad_alloc.
  void init(size_t pages, size_t max_seqs, size_t max_len);

  size_t pages() const { return refs_.size(); }
  size_t used() const { return refs_.size() - free_.size(); }
  size_t max_seqs() const { return seqs_.size(); }
  size_t max_pages() const { return max_pages_; }  // a page table row's entries
  size_t max_len() const { return max_len_; }

  // Every call either succeeds or leaves everything as it was, with a message.
  enum Status { OK, BAD, FULL };
  Status create(uint32_t* seq, std::string* err);
  Status free(uint32_t seq, std::string* err);
  // n new sequences that share the pages of `seq`
  Status fork(uint32_t seq, size_t n, uint32_t* out, std::string* err);
  // one new sequence with pages of its own; copies: what they are filled from
  Status copy(uint32_t seq, uint32_t* out, std::vector<KvCopy>* copies, std::string* err);
  Status truncate(uint32_t seq, size_t len, std::string* err);
  Status len(uint32_t seq, size_t* len, std::string* err) const;
  // Whether step() would succeed, and a message if not.
  Status check_step(size_t nseq, const uint32_t* seqs, const uint32_t* ntok, std::string* err);
  // After check_step(): what the step would be, and the page table changes and
  // page copies that it would make.
  void preview(size_t nseq, const uint32_t* seqs, const uint32_t* ntok, std::vector<KvStepSeq>* plan) const;
  // and room for what step() adds, so that it throws nothing.  Throws std::bad_alloc.
  void reserve_step(size_t nseq, const uint32_t* seqs, const uint32_t* ntok, std::vector<KvCopy>* copies);
  size_t step_changes() const { return need_; }
  size_t step_copies() const { return copies_; }
  // Room for ntok[i] more positions of seqs[i]: new pages, and copies of
  // shared, partly filled pages that the step writes to.  plan (may be null): as preview().
  Status step(size_t nseq, const uint32_t* seqs, const uint32_t* ntok, std::vector<KvStepSeq>* plan,
              std::vector<KvCopy>* copies, std::string* err);
  // What compact() would move: pages, and page table entries that change.
  void compact_size(size_t* moved, size_t* entries) const;
  // Moves the pages behind the first used() into the holes before.
  void compact(std::vector<KvCopy>* copies);
  // Another number of pages, at least used(), of a compacted pool.  Throws
  // std::bad_alloc, leaving everything as it was.
  void resize(size_t pages);

  // The page that holds a sequence's position (which it holds).
  uint32_t page_of(uint32_t seq, size_t pos) const { return seqs_[seq].pages[pos / KV_PAGE]; }
  bool live(uint32_t seq) const { return seq < seqs_.size() && seqs_[seq].live; }
  uint32_t refs(uint32_t page) const { return refs_[page]; }

  // Page table entries (row * max_pages + index) that changed since they were
  // last sent, some perhaps several times, and an entry's page now (0 where the
  // sequence has none there).
  std::vector<uint32_t> dirty;
  uint32_t entry(uint32_t index) const {
    const Seq& s = seqs_[index / max_pages_];
    return index % max_pages_ < s.pages.size() ? s.pages[index % max_pages_] : 0;
  }

 private:
  struct Seq {
    bool live = false;
    size_t len = 0;
    std::vector<uint32_t> pages;
  };
  Status find(uint32_t seq, std::string* err) const;
  uint32_t take();
  void drop(uint32_t page);
  void set(uint32_t seq, size_t index);
  std::vector<uint32_t> refs_, free_;
  std::vector<Seq> seqs_;
  std::vector<uint32_t> free_seqs_;
  // check_step(): what it saw of each sequence in its last call, and its counts
  std::vector<uint32_t> mark_;
  size_t settled_ = 65536;  // changes from which on fork() looks for repeated ones
  uint32_t stamp_ = 0;
  size_t need_ = 0, copies_ = 0;
  size_t max_len_ = 0, max_pages_ = 0;
};

}  // namespace hale
