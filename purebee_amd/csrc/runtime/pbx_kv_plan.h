// pbx_kv_plan.h -- the paged KV cache's bookkeeping on the host: which pages a
// sequence holds, and the work lists of a batch that the kernels of pbx_kv.hip
// run over.  No HIP calls, so every page id and index that reaches a kernel
// can be checked without a GPU.
#ifndef PBX_KV_PLAN_H
#define PBX_KV_PLAN_H

#include <stdint.h>
#include <stdio.h>

#include <algorithm>
#include <string>
#include <vector>

#include "pbx.h"

struct kv_seq {
  int len = 0;
  uint64_t met = 0;    // the last call that named it (kv_pages::batches)
  uint64_t moved = 0;  // the last call that dropped its positions, or moved them or their
  int moved_at = 0;    // pages, from position moved_at on
  std::vector<int32_t> pages;
};

struct kv_pages {
  int page_tokens = 0, max_seq = 0;
  uint64_t batches = 0;  // planned so far, refused ones too (and forks and compactions)
  uint64_t forks = 0;    // forks so far: pages that a sequence had alone may be shared since
  std::vector<int32_t> free_list;  // handed out from the back
  std::vector<int32_t> refs;       // sequences that hold a page
  std::vector<kv_seq> seqs;

  void init(int page_tokens_, int n_pages, int max_seqs, int max_seq_) {
    page_tokens = page_tokens_;
    max_seq = max_seq_;
    free_list.resize(n_pages);
    for (int i = 0; i < n_pages; ++i) free_list[i] = n_pages - 1 - i;
    refs.assign(n_pages, 0);
    seqs.assign(max_seqs, kv_seq());
  }
  // A page for one sequence (the caller has seen that there is one), and one that a
  // sequence lets go of; untake and ungive take the last such call back.  None of
  // them allocates: the free list never holds more than it did at first.
  int32_t take() {
    const int32_t p = free_list.back();
    free_list.pop_back();
    refs[p] = 1;
    return p;
  }
  void give(int32_t p) {
    if (!--refs[p]) free_list.push_back(p);
  }
  void untake(int32_t p) {
    refs[p] = 0;
    free_list.push_back(p);
  }
  void ungive(int32_t p) {
    if (!refs[p]++) free_list.pop_back();
  }
  int pages_of(int tokens) const { return (int)(((int64_t)tokens + page_tokens - 1) / page_tokens); }

  int truncate(int seq, int n, std::string *why) {
    char buf[160];
    if (seq < 0 || seq >= (int)seqs.size()) {
      snprintf(buf, sizeof buf, "sequence %d outside [0, %d)", seq, (int)seqs.size());
    } else if (n < 0 || n > seqs[seq].len) {
      snprintf(buf, sizeof buf, "sequence %d holds %d positions, not %d", seq, seqs[seq].len, n);
    } else {
      kv_seq &s = seqs[seq];
      s.len = n;
      while ((int)s.pages.size() > pages_of(n)) {
        give(s.pages.back());
        s.pages.pop_back();
      }
      return PBX_OK;
    }
    *why = buf;
    return PBX_EINVAL;
  }

  // Sequence dsts[i] comes to hold the first lens[i] positions (lens == NULL: all)
  // that srcs[i] held before the call, in the same pages.
  int fork(int n, const int32_t *dsts, const int32_t *srcs, const int32_t *lens, std::string *why) {
    char buf[160];
    ++batches;
    std::vector<std::vector<int32_t>> held(n);
    std::vector<int> len(n);
    for (int i = 0; i < n; ++i) {
      const int d = dsts[i], s = srcs[i], known = (int)seqs.size();
      buf[0] = 0;
      if (d < 0 || d >= known || s < 0 || s >= known)
        snprintf(buf, sizeof buf, "sequence %d outside [0, %d)", d < 0 || d >= known ? d : s, known);
      else if (seqs[d].met == batches)
        snprintf(buf, sizeof buf, "sequence %d twice among those that are made", d);
      else if (lens && (lens[i] < 0 || lens[i] > seqs[s].len))
        snprintf(buf, sizeof buf, "sequence %d holds %d positions, not %d", s, seqs[s].len, lens[i]);
      if (buf[0]) {
        *why = buf;
        return PBX_EINVAL;
      }
      seqs[d].met = batches;
      len[i] = lens ? lens[i] : seqs[s].len;
      held[i].assign(seqs[s].pages.begin(), seqs[s].pages.begin() + pages_of(len[i]));
    }
    ++forks;
    for (auto &h : held)
      for (int32_t p : h) ++refs[p];
    for (int i = 0; i < n; ++i) {
      kv_seq &d = seqs[dsts[i]];
      for (int32_t p : d.pages) give(p);
      d.pages.swap(held[i]);
      d.len = len[i];
      d.moved = batches;
      d.moved_at = dsts[i] == srcs[i] ? len[i] : 0;
    }
    return PBX_OK;
  }
};

// One block of PBX_KV_BLOCK positions that a batch's rows touch (append, read).
struct kv_block_item {
  int32_t page, sub;    // the page and the block's place in it
  int32_t pos0;         // the block's first position
  int32_t start, count; // the sequence's rows of the batch: positions and
  int32_t row0;         // first packed row
  int32_t pad[2];
};
// Query rows 16 u tile .. of a sequence ((row, head of the KV group) pairs, the
// head fastest) over its blocks blk0..blk1 - 1: u 16-row tiles, 1, 2, 4 or 8 (the kernels have 4 at most).
struct kv_attn_item {
  int32_t start, count, row0;
  int32_t tile;
  int32_t blk0, blk1;
  int32_t tab;       // the sequence's page ids, from here on in the page table
  int32_t part, parts;  // this item's place among those of its rows
  int32_t slot;      // the first part's partial result, in units of 16 rows (parts > 1)
  int32_t join;      // which rows these are among those that are split (parts > 1)
  int32_t pad;
  int32_t pages[4];  // the pages from block blk0 on (as far as blk1 needs them)
};

// A page of a sequence that grows in it while others hold it too: the sequence gets
// a copy of its filled blocks, in every layer.
struct kv_page_copy {
  int32_t from, to, blocks, pad;
};
struct kv_own_page {  // where such a copy took its place
  int32_t seq, index;
};

struct kv_batch_plan {
  int n_rows = 0;
  bool last = true;  // the rows are the last of their sequences
  std::vector<int32_t> seqs, starts, counts;
  std::vector<int32_t> had;  // the sequences' lengths before
  std::vector<kv_page_copy> copies;
  std::vector<kv_own_page> owned;  // [copies]
  // work lists, in the order they lie in device memory
  std::vector<kv_block_item> blocks;
  std::vector<kv_attn_item> attn;  // those of u 1, then 2, 4, 8
  std::vector<int32_t> row_pos;  // position of every packed row
  std::vector<int32_t> last_rows;  // the last row of each sequence that has any
  std::vector<int32_t> table;    // page ids, sequence by sequence
  int n_attn[4] = {0, 0, 0, 0};
  int n_slots = 0, n_joins = 0;

  // the memory of another plan's lists, to be filled again
  void take_lists(kv_batch_plan *p) {
    blocks.swap(p->blocks);
    attn.swap(p->attn);
    row_pos.swap(p->row_pos);
    last_rows.swap(p->last_rows);
    table.swap(p->table);
  }
};

// Checks a batch and, if it holds, takes its pages and fills the plan; refused
// batches change nothing.  Costs what the batch is, however many sequences the
// cache could hold.
inline int kv_plan_rows(kv_pages *kv, int n, const int32_t *seqs, const int32_t *starts,
                        const int32_t *counts, kv_batch_plan *p, std::string *why) {
  char buf[200];
  ++kv->batches;
  int64_t rows = 0, need = 0;
  // Pages that the batch's sequences will have left to others, taken off their
  // counts while the batch is looked over: the last holder needs no copy.
  struct Left {
    kv_pages *kv;
    std::vector<int32_t> pages;
    ~Left() {
      for (int32_t p : pages) ++kv->refs[p];
    }
  };
  kv_batch_plan q;
  {
  Left left{kv, {}};
  for (int i = 0; i < n; ++i) {
    const int s = seqs[i];
    buf[0] = 0;
    if (s < 0 || s >= (int)kv->seqs.size()) {
      snprintf(buf, sizeof buf, "sequence %d outside [0, %d)", s, (int)kv->seqs.size());
    } else if (kv->seqs[s].met == kv->batches) {
      snprintf(buf, sizeof buf, "sequence %d twice in one batch", s);
    } else if (counts[i] < 0) {
      snprintf(buf, sizeof buf, "sequence %d: %d rows", s, counts[i]);
    } else {
      const int len = kv->seqs[s].len, at = starts ? starts[i] : len;
      if (at < 0 || at > len)
        snprintf(buf, sizeof buf, "sequence %d holds %d positions: rows cannot start at %d", s, len, at);
      else if ((int64_t)at + counts[i] > kv->max_seq)
        snprintf(buf, sizeof buf, "sequence %d: positions [%d, %lld) exceed max_seq %d", s, at,
                 (long long)at + counts[i], kv->max_seq);
      else
        need += std::max(0, kv->pages_of(at + counts[i]) - (int)kv->seqs[s].pages.size());
      const std::vector<int32_t> &held = kv->seqs[s].pages;
      for (int j = at / kv->page_tokens; !buf[0] && at + counts[i] > len && j < (int)held.size(); ++j)
        if (kv->refs[held[j]] > 1) {
          left.pages.push_back(held[j]);
          --kv->refs[held[j]];
          q.owned.push_back({s, j});
          ++need;
        }
    }
    if (buf[0]) {
      *why = buf;
      return PBX_EINVAL;
    }
    kv->seqs[s].met = kv->batches;
    rows += counts[i];
  }
  if (rows > (1 << 26)) {
    snprintf(buf, sizeof buf, "%lld rows in one batch", (long long)rows);
    *why = buf;
    return PBX_ENOTSUP;
  }
  if (need > (int64_t)kv->free_list.size()) {
    snprintf(buf, sizeof buf, "%lld pages wanted, %d free", (long long)need, (int)kv->free_list.size());
    *why = buf;
    return PBX_ENOMEM;
  }
  }
  for (int i = 0; i < n; ++i) {
    kv_seq &s = kv->seqs[seqs[i]];
    q.seqs.push_back(seqs[i]);
    q.starts.push_back(starts ? starts[i] : s.len);
    q.counts.push_back(counts[i]);
    q.had.push_back(s.len);
    s.pages.reserve(kv->pages_of(q.starts[i] + counts[i]));
  }
  q.n_rows = (int)rows;
  q.copies.reserve(q.owned.size());
  // nothing below allocates on behalf of a sequence: the pages change hands whole
  for (const kv_own_page &o : q.owned) {
    kv_seq &s = kv->seqs[o.seq];
    const int32_t from = s.pages[o.index], to = kv->take();
    const int filled = std::min(kv->page_tokens, s.len - o.index * kv->page_tokens);
    q.copies.push_back({from, to, (filled + PBX_KV_BLOCK - 1) / PBX_KV_BLOCK, 0});
    kv->give(from);
    s.pages[o.index] = to;
    if (s.moved != kv->batches) s.moved_at = o.index * kv->page_tokens;
    s.moved = kv->batches;
  }
  for (int i = 0; i < n; ++i) {
    kv_seq &s = kv->seqs[seqs[i]];
    const int end = q.starts[i] + counts[i];
    while ((int)s.pages.size() < kv->pages_of(end)) s.pages.push_back(kv->take());
    s.len = std::max(s.len, end);
  }
  std::swap(*p, q);
  return PBX_OK;
}

// Takes a planned batch back (before another one is planned): the lengths and
// pages are as they were.
inline void kv_plan_undo(kv_pages *kv, const kv_batch_plan &p) {
  std::string why;
  for (size_t i = p.seqs.size(); i-- > 0;) kv->truncate(p.seqs[i], p.had[i], &why);
  for (size_t i = p.copies.size(); i-- > 0;) {
    kv->seqs[p.owned[i].seq].pages[p.owned[i].index] = p.copies[i].from;
    kv->ungive(p.copies[i].from);
    kv->untake(p.copies[i].to);
  }
}

// One block that a compaction fills: rows of the sequence's old positions, coded
// anew, or (raw) the old block as it is.
struct kv_pack_item {
  int32_t page, sub;   // where it goes
  int32_t pos0, rows;  // its first (new) position, and its rows
  int32_t at;          // its rows, from here on in the list
  int32_t raw;         // the page of the old block to be copied as it is, or -1
  int32_t pad[2];
};
struct kv_pack_row {
  int32_t page, pos;  // a row's old page and position
};
struct kv_pack_plan {
  std::vector<kv_pack_item> items;
  std::vector<int32_t> launches;  // items of each launch: later ones fill pages that earlier ones emptied
  std::vector<kv_pack_row> rows;
  std::vector<int32_t> seqs;
  std::vector<int32_t> log;  // pages taken (p) and given back (-1 - p), in order
  std::vector<kv_seq> was;
};

inline void kv_pack_undo(kv_pages *kv, kv_pack_plan *p) {
  for (size_t i = p->log.size(); i-- > 0;) {
    const int32_t x = p->log[i];
    if (x >= 0)
      kv->untake(x);
    else
      kv->ungive(-1 - x);
  }
  for (size_t i = 0; i < p->was.size(); ++i) {
    kv->seqs[p->seqs[i]].len = p->was[i].len;
    kv->seqs[p->seqs[i]].pages.swap(p->was[i].pages);
  }
  p->log.clear();
  p->was.clear();
}

// Where a compaction ends with some of its launches missing, after others wrote pages that
// were given back before: neither the old rows nor the new ones are whole, and the sequences
// are cut to the positions before those that move.
inline void kv_pack_cut(kv_pages *kv, const kv_pack_plan &p) {
  std::string why;
  for (int32_t s : p.seqs) kv->truncate(s, std::min(kv->seqs[s].len, kv->seqs[s].moved_at), &why);
}

// Sequence seqs[i] keeps counts[i] of its positions (rising; `positions` holds them
// one sequence after the other), which move together to 0 .. counts[i] - 1.  Pages
// whose rows all stay are kept; the rest goes to fresh pages, so that no block is
// read after it was written over.  Positions only move down: once a page of new rows
// is filled, as many old pages have been read for good, so a pool with few free pages
// takes several launches (each fills pages that are free before it).
inline int kv_plan_pack(kv_pages *kv, int n, const int32_t *seqs, const int32_t *counts, const int32_t *positions,
                        kv_pack_plan *p, std::string *why) {
  char buf[200];
  ++kv->batches;
  int64_t at = 0, all = 0, rows = 0;
  for (int i = 0; i < n; ++i) {
    const int s = seqs[i], known = (int)kv->seqs.size(), len = s < 0 || s >= known ? 0 : kv->seqs[s].len;
    buf[0] = 0;
    if (s < 0 || s >= known)
      snprintf(buf, sizeof buf, "sequence %d outside [0, %d)", s, known);
    else if (kv->seqs[s].met == kv->batches)
      snprintf(buf, sizeof buf, "sequence %d twice", s);
    else if (counts[i] < 0 || counts[i] > len)
      snprintf(buf, sizeof buf, "sequence %d holds %d positions, %d are to stay", s, len, counts[i]);
    const int32_t *pos = positions + at;
    bool rise = true;  // (all of them, without a branch, and the first that does not only then)
    for (int j = 1; !buf[0] && j < counts[i]; ++j) rise &= pos[j] > pos[j - 1];
    if (!buf[0] && counts[i]) rise &= pos[0] >= 0 && pos[counts[i] - 1] < len;
    for (int j = 0; !buf[0] && !rise && j < counts[i]; ++j)
      if (pos[j] < 0 || pos[j] >= len || (j && pos[j] <= pos[j - 1]))
        snprintf(buf, sizeof buf, "sequence %d: positions have to rise within [0, %d) (%d at place %d)", s, len,
                 pos[j], j);
    if (buf[0]) {
      *why = buf;
      return PBX_EINVAL;
    }
    kv->seqs[s].met = kv->batches;
    at += counts[i];
    all += (int64_t)kv->seqs[s].pages.size();
    rows += counts[i];
  }
  if (rows > (1 << 26) || all > (1 << 26)) {
    *why = "more than 2^26 positions in one call";
    return PBX_ENOTSUP;
  }
  const int T = kv->page_tokens, per_page = T / PBX_KV_BLOCK;
  // everything that may throw comes first (the log and the lists cannot grow past these);
  // a plan that was used before gives its memory
  p->log.clear();
  p->launches.clear();
  p->items.clear();
  p->seqs.assign(seqs, seqs + n);
  p->was.resize(n);
  p->log.reserve(2 * all + 2);
  p->launches.reserve(all + 1);
  p->items.reserve(all * per_page);
  p->rows.resize(rows);
  std::vector<std::vector<int32_t>> made(n);
  std::vector<int> first(n), read(n);  // first page that is replaced, and old pages that are given back
  std::vector<int> from(n);            // positions from which rows or pages move
  at = 0;
  for (int i = 0; i < n; ++i) {
    int same = 0;
    while (same < counts[i] && positions[at + same] == same) ++same;
    first[i] = same == counts[i] ? kv->pages_of(same) : same / T;
    read[i] = first[i];
    from[i] = same == counts[i] ? same : first[i] * T;
    made[i].reserve(kv->pages_of(counts[i]));
    at += counts[i];
  }
  for (int i = 0; i < n; ++i) {
    kv_seq &s = kv->seqs[seqs[i]];
    p->was[i].len = s.len;
    p->was[i].pages = s.pages;
  }
  size_t launched = 0;
  auto give = [&](int i, int upto) {
    for (; read[i] < upto; ++read[i]) {
      kv->give(p->was[i].pages[read[i]]);
      p->log.push_back(-1 - p->was[i].pages[read[i]]);
    }
  };
  at = 0;
  int shift = 0, listed = 0;
  while (1 << shift < T) ++shift;  // (pages are a power of two)
  int done = 0;  // sequences whose old pages were given back
  std::vector<int> need(n, 0);  // old pages that the pages planned so far have read for good
  for (int i = 0; i < n; ++i) {
    const std::vector<int32_t> &old = p->was[i].pages;
    const int base = first[i] * T, list = listed;
    made[i].assign(old.begin(), old.begin() + first[i]);
    const int32_t *pages = old.data(), *pos = positions + at;
    kv_pack_row *out = p->rows.data() + listed;
    for (int j = base; j < counts[i]; ++j) out[j - base] = {pages[(unsigned)pos[j] >> shift], pos[j]};
    listed += std::max(0, counts[i] - base);
    need[i] = first[i];
    for (int j = first[i]; j < kv->pages_of(counts[i]); ++j) {
      if (kv->free_list.empty()) {
        if (p->items.size() > launched) p->launches.push_back((int32_t)(p->items.size() - launched));
        launched = p->items.size();
        for (; done < i; ++done) give(done, (int)p->was[done].pages.size());
        give(i, need[i]);
        if (kv->free_list.empty()) {
          kv_pack_undo(kv, p);
          snprintf(buf, sizeof buf, "no free page to move positions of sequence %d to", seqs[i]);
          *why = buf;
          return PBX_ENOMEM;
        }
      }
      const int32_t page = kv->take();
      p->log.push_back(page);
      made[i].push_back(page);
      for (int b = 0; b < per_page && j * T + b * PBX_KV_BLOCK < counts[i]; ++b) {
        const int pos0 = j * T + b * PBX_KV_BLOCK, m = std::min(PBX_KV_BLOCK, counts[i] - pos0);
        const bool stays = positions[at + pos0 + m - 1] == pos0 + m - 1;
        p->items.push_back({page, b, pos0, m, list + pos0 - base, stays ? old[j] : -1, {0, 0}});
      }
      const int next = (j + 1) * T;
      need[i] = next < counts[i] ? positions[at + next] / T : (int)old.size();
    }
    at += counts[i];
  }
  p->rows.resize(listed);
  if (p->items.size() > launched) p->launches.push_back((int32_t)(p->items.size() - launched));
  for (int i = 0; i < n; ++i) give(i, (int)p->was[i].pages.size());
  for (int i = 0; i < n; ++i) {
    kv_seq &s = kv->seqs[seqs[i]];
    s.len = counts[i];
    s.pages.swap(made[i]);
    s.moved = kv->batches;
    s.moved_at = from[i];
  }
  return PBX_OK;
}

#define KV_MAX_PARTS 64

// The work lists of a planned batch: `groups` = n_heads / n_kv_heads query
// heads a KV head, `kv_heads` KV heads (each item runs once per KV head),
// `max_u` 16-row tiles of the widest kernel for this head size, `want`
// workgroups that fill the GPU.
inline void kv_plan_work(const kv_pages &kv, int groups, int kv_heads, int max_u, int want, kv_batch_plan *p) {
  const int n = (int)p->seqs.size();
  p->blocks.clear();
  p->attn.clear();
  p->row_pos.clear();
  p->last_rows.clear();
  p->table.clear();
  p->n_slots = p->n_joins = 0;
  for (int &x : p->n_attn) x = 0;
  p->last = true;
  // log2 u of each sequence: the narrowest kernel that holds its rows, or the
  // widest there is
  std::vector<int> width(n, 0);
  for (int i = 0; i < n; ++i)
    while (2 << width[i] <= max_u && (int64_t)p->counts[i] * groups > 16 << width[i]) ++width[i];
  auto tiles_of = [&](int i) {
    const int t = 16 << width[i];
    return (int)(((int64_t)p->counts[i] * groups + t - 1) / t);
  };
  auto blocks_of = [&](int i, int tile) {  // visible to the tile's last row
    const unsigned rows = (unsigned)p->counts[i] * groups;  // (at most 2^20 rows of 2^10 heads)
    const unsigned last = std::min(rows, (unsigned)(16 << width[i]) * (tile + 1u)) - 1;
    return (int)((p->starts[i] + last / (unsigned)groups) / PBX_KV_BLOCK + 1);
  };
  // Where the tiles are few (one and a half a CU: `want` is two), narrower ones:
  // half as many rows a workgroup make twice as many workgroups (one sequence of
  // 36 rows on 6,000 positions, 9 / 3 heads of 64: 22.8 -> 10.7 us; 17 of 6 to 34
  // rows, 32 / 8 heads of 64: 7.9 -> 6.0, and at two a CU as many got slower).
  auto workgroups = [&]() {
    int64_t g = 0;
    for (int i = 0; i < n; ++i) g += tiles_of(i);
    return g * kv_heads;
  };
  for (int w = 3; w > 0 && workgroups() < 3 * want / 4; --w)
    for (int i = 0; i < n; ++i) width[i] = std::min(width[i], w - 1);
  // Each width is a launch of its own, one after the other.  One whose blocks do
  // not fill the GPU (16 a workgroup) is little but latency and joins the next
  // wider one that there is (33 sequences of 1 to 9 rows: 17.6 -> 12 us).
  const int64_t least = 16;
  for (int w = 0; w < 3; ++w) {
    int64_t here = 0;
    int wider = 4;
    for (int i = 0; i < n; ++i) {
      if (width[i] > w && p->counts[i]) wider = std::min(wider, width[i]);
      for (int t = 0, tiles = width[i] == w ? tiles_of(i) : 0; t < tiles; ++t) here += blocks_of(i, t);
    }
    if (wider == 4 || here * kv_heads >= least * want) continue;
    for (int i = 0; i < n; ++i)
      if (width[i] == w) width[i] = wider;
  }
  int64_t total = 0;  // blocks that the tiles visit
  std::vector<int32_t> seen;  // by each
  for (int i = 0; i < n; ++i)
    for (int t = 0, tiles = tiles_of(i); t < tiles; ++t) {
      seen.push_back(blocks_of(i, t));
      total += seen.back();
    }
  // an item: at least 16 blocks (four a wave), and about `want` workgroups in all;
  // wide tiles that fill the GPU as they are, longest first, are split only where
  // one is far longer than that: their partial results cost more than the
  // better balance brings (a 1,000-token prompt 32 -> 23 us)
  const int64_t even = std::max<int64_t>(least, (total * kv_heads + want - 1) / want);
  const int64_t wide = workgroups() < want / 2 ? even : 4 * even;
  const int per_page = kv.page_tokens / PBX_KV_BLOCK;
  // Items in order of log2 u, then the ones with the most blocks first (so that none of
  // them is the last to start), else as they come: counted by u and length, then each
  // written to its place.
  const unsigned chunks[2] = {(unsigned)std::min<int64_t>(even, 1 << 20), (unsigned)std::min<int64_t>(wide, 1 << 20)};
  auto parts_of = [&](int nb, int lu) {  // (a sequence has 2^15 blocks at most)
    const unsigned chunk = chunks[lu > 0];
    return nb <= (int)chunk ? 1 : (int)std::min<unsigned>(KV_MAX_PARTS, (nb + chunk - 1) / chunk);
  };
  int most = 0;
  int64_t n_blocks = 0, n_table = 0;
  for (int i = 0; i < n; ++i) {
    if (!p->counts[i]) continue;
    const int end = p->starts[i] + p->counts[i];
    most = std::max(most, (end - 1) / PBX_KV_BLOCK + 1);
    n_blocks += (end - 1) / PBX_KV_BLOCK + 1 - p->starts[i] / PBX_KV_BLOCK;
    n_table += kv.pages_of(end);
  }
  std::vector<int32_t> place((size_t)4 * (most + 1), 0);  // [u][most - length]
  const int32_t *nbs = seen.data();
  for (int i = 0; i < n; ++i) {
    const int lu = width[i], tiles = tiles_of(i);
    int32_t *at = place.data() + (size_t)lu * (most + 1) + most;
    for (int t = 0; t < tiles; ++t) {
      const int nb = *nbs++, parts = parts_of(nb, lu);
      p->n_attn[lu] += parts;
      if (parts == 1) {
        ++at[-nb];
        continue;
      }
      const int each = nb / parts, more = nb % parts;  // lengths differ by one at most
      at[-each] += parts - more;
      if (more) at[-each - 1] += more;
    }
  }
  int32_t sum = 0;
  for (int32_t &x : place) {
    const int32_t here = x;
    x = sum;
    sum += here;
  }
  p->attn.resize(sum);
  p->blocks.reserve(n_blocks);
  p->table.reserve(n_table);
  p->row_pos.resize(p->n_rows);
  int row0 = 0, page_shift = 0;
  while (1 << page_shift < per_page) ++page_shift;
  nbs = seen.data();
  for (int i = 0; i < n; ++i) {
    const kv_seq &s = kv.seqs[p->seqs[i]];
    const int start = p->starts[i], count = p->counts[i], tab = (int)p->table.size(), lu = width[i];
    if (!count) continue;
    if (start + count != s.len) p->last = false;
    const int used = kv.pages_of(start + count);
    p->table.insert(p->table.end(), s.pages.begin(), s.pages.begin() + used);
    for (int b = start / PBX_KV_BLOCK; b * PBX_KV_BLOCK < start + count; ++b)
      p->blocks.push_back({s.pages[b / per_page], b % per_page, b * PBX_KV_BLOCK, start, count, row0, {0, 0}});
    for (int t = 0; t < count; ++t) p->row_pos[row0 + t] = start + t;
    int32_t *at = place.data() + (size_t)lu * (most + 1) + most;
    const int tiles = tiles_of(i);
    for (int t = 0; t < tiles; ++t) {
      const int nb = *nbs++, parts = parts_of(nb, lu);
      for (int k = 0, blk0 = 0; k < parts; ++k) {
        const int blk1 = parts == 1 ? nb : nb * (k + 1) / parts;
        const int first = blk0 >> page_shift, last = (blk1 - 1) >> page_shift;
        kv_attn_item &x = p->attn[at[blk0 - blk1]++];
        x = {start, count, row0, t, blk0, blk1, tab, k, parts, p->n_slots, p->n_joins, 0, {0, 0, 0, 0}};
        for (int j = 0; j < 4; ++j) x.pages[j] = s.pages[std::min(first + j, last)];
        blk0 = blk1;
      }
      if (parts > 1) {
        p->n_slots += parts << lu;
        ++p->n_joins;
      }
    }
    row0 += count;
    p->last_rows.push_back(row0 - 1);
  }
}

// Whether the batch has rows of sequence seq from position n on.
inline bool kv_plan_reaches(const kv_batch_plan &p, int seq, int n) {
  for (size_t i = 0; i < p.seqs.size(); ++i)
    if (p.seqs[i] == seq) return p.counts[i] && p.starts[i] + p.counts[i] > n;
  return false;
}

// Whether the batch runs over positions that the last call (a fork, a compaction, a
// batch that took pages of its own) dropped or moved.
inline bool kv_plan_moved(const kv_pages &kv, const kv_batch_plan &p) {
  for (size_t i = 0; i < p.seqs.size(); ++i) {
    const kv_seq &s = kv.seqs[p.seqs[i]];
    if (p.counts[i] && s.moved == kv.batches && p.starts[i] + p.counts[i] > s.moved_at) return true;
  }
  return false;
}

#endif
