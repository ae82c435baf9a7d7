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
  uint64_t met = 0;  // the last batch that named it (kv_pages::batches)
  std::vector<int32_t> pages;
};

struct kv_pages {
  int page_tokens = 0, max_seq = 0;
  uint64_t batches = 0;  // planned so far, refused ones too
  std::vector<int32_t> free_list;  // handed out from the back
  std::vector<kv_seq> seqs;

  void init(int page_tokens_, int n_pages, int max_seqs, int max_seq_) {
    page_tokens = page_tokens_;
    max_seq = max_seq_;
    free_list.resize(n_pages);
    for (int i = 0; i < n_pages; ++i) free_list[i] = n_pages - 1 - i;
    seqs.assign(max_seqs, kv_seq());
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
        free_list.push_back(s.pages.back());
        s.pages.pop_back();
      }
      return PBX_OK;
    }
    *why = buf;
    return PBX_EINVAL;
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

struct kv_batch_plan {
  int n_rows = 0;
  bool last = true;  // the rows are the last of their sequences
  std::vector<int32_t> seqs, starts, counts;
  std::vector<int32_t> had;  // the sequences' lengths before
  // work lists, in the order they lie in device memory
  std::vector<kv_block_item> blocks;
  std::vector<kv_attn_item> attn;  // those of u 1, then 2, 4, 8
  std::vector<int32_t> row_pos;  // position of every packed row
  std::vector<int32_t> last_rows;  // the last row of each sequence that has any
  std::vector<int32_t> table;    // page ids, sequence by sequence
  int n_attn[4] = {0, 0, 0, 0};
  int n_slots = 0, n_joins = 0;
};

// Checks a batch and, if it holds, takes its pages and fills the plan; refused
// batches change nothing.  Costs what the batch is, however many sequences the
// cache could hold.
inline int kv_plan_rows(kv_pages *kv, int n, const int32_t *seqs, const int32_t *starts,
                        const int32_t *counts, kv_batch_plan *p, std::string *why) {
  char buf[200];
  ++kv->batches;
  int64_t rows = 0, need = 0;
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
  kv_batch_plan q;
  for (int i = 0; i < n; ++i) {
    kv_seq &s = kv->seqs[seqs[i]];
    q.seqs.push_back(seqs[i]);
    q.starts.push_back(starts ? starts[i] : s.len);
    q.counts.push_back(counts[i]);
    q.had.push_back(s.len);
    s.pages.reserve(kv->pages_of(q.starts[i] + counts[i]));
  }
  q.n_rows = (int)rows;
  q.row_pos.reserve(rows);
  // nothing below allocates on behalf of a sequence: the pages change hands whole
  for (int i = 0; i < n; ++i) {
    kv_seq &s = kv->seqs[seqs[i]];
    const int end = q.starts[i] + counts[i];
    while ((int)s.pages.size() < kv->pages_of(end)) {
      s.pages.push_back(kv->free_list.back());
      kv->free_list.pop_back();
    }
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
    const int64_t rows = (int64_t)p->counts[i] * groups;
    const int64_t last = std::min<int64_t>(rows, (16 << width[i]) * ((int64_t)tile + 1)) - 1;
    return (int)((p->starts[i] + last / groups) / PBX_KV_BLOCK + 1);
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
      for (int t = 0; width[i] == w && t < tiles_of(i); ++t) here += blocks_of(i, t);
    }
    if (wider == 4 || here * kv_heads >= least * want) continue;
    for (int i = 0; i < n; ++i)
      if (width[i] == w) width[i] = wider;
  }
  int64_t total = 0;  // blocks that the tiles visit
  for (int i = 0; i < n; ++i)
    for (int t = 0; t < tiles_of(i); ++t) total += blocks_of(i, t);
  // an item: at least 16 blocks (four a wave), and about `want` workgroups in all;
  // wide tiles that fill the GPU as they are, longest first, are split only where
  // one is far longer than that: their partial results cost more than the
  // better balance brings (a 1,000-token prompt 32 -> 23 us)
  const int64_t even = std::max<int64_t>(least, (total * kv_heads + want - 1) / want);
  const int64_t wide = workgroups() < want / 2 ? even : 4 * even;
  const int per_page = kv.page_tokens / PBX_KV_BLOCK;
  std::vector<kv_attn_item> by_u[4];
  int row0 = 0;
  for (int i = 0; i < n; ++i) {
    const kv_seq &s = kv.seqs[p->seqs[i]];
    const int start = p->starts[i], count = p->counts[i], tab = (int)p->table.size(), lu = width[i];
    if (!count) continue;
    if (start + count != s.len) p->last = false;
    const int used = kv.pages_of(start + count);
    p->table.insert(p->table.end(), s.pages.begin(), s.pages.begin() + used);
    for (int b = start / PBX_KV_BLOCK; b * PBX_KV_BLOCK < start + count; ++b)
      p->blocks.push_back({s.pages[b / per_page], b % per_page, b * PBX_KV_BLOCK, start, count, row0, {0, 0}});
    for (int t = 0; t < count; ++t) p->row_pos.push_back(start + t);
    for (int t = 0; t < tiles_of(i); ++t) {
      const int nb = blocks_of(i, t);
      const int64_t chunk = lu ? wide : even;
      const int parts = (int)std::min<int64_t>(KV_MAX_PARTS, (nb + chunk - 1) / chunk);
      for (int k = 0; k < parts; ++k) {
        kv_attn_item x = {start, count, row0, t, (int)((int64_t)nb * k / parts), (int)((int64_t)nb * (k + 1) / parts),
                          tab, k, parts, p->n_slots, p->n_joins, 0, {0, 0, 0, 0}};
        for (int j = 0; j < 4; ++j) x.pages[j] = s.pages[std::min(x.blk0 / per_page + j, (x.blk1 - 1) / per_page)];
        by_u[lu].push_back(x);
      }
      if (parts > 1) {
        p->n_slots += parts << lu;
        ++p->n_joins;
      }
    }
    row0 += count;
    p->last_rows.push_back(row0 - 1);
  }
  for (int c = 0; c < 4; ++c) {
    // the items with the most blocks first, so that none of them is the last to start
    std::stable_sort(by_u[c].begin(), by_u[c].end(), [](const kv_attn_item &x, const kv_attn_item &y) {
      return x.blk1 - x.blk0 > y.blk1 - y.blk0;
    });
    p->attn.insert(p->attn.end(), by_u[c].begin(), by_u[c].end());
    p->n_attn[c] = (int)by_u[c].size();
  }
}

// Whether the batch has rows of sequence seq from position n on.
inline bool kv_plan_reaches(const kv_batch_plan &p, int seq, int n) {
  for (size_t i = 0; i < p.seqs.size(); ++i)
    if (p.seqs[i] == seq) return p.counts[i] && p.starts[i] + p.counts[i] > n;
  return false;
}

#endif
