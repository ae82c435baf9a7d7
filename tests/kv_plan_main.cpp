// Random batches, truncations and refusals over the paged KV cache's host
// bookkeeping (purebee_amd/csrc/runtime/pbx_kv_plan.h): every page, row, block
// and partial result that the kernels would address is checked.
#include "pbx_kv_plan.h"

#include <stdlib.h>

#include <map>
#include <random>
#include <set>

#define CHECK(x)                                                  \
  do {                                                            \
    if (!(x)) {                                                   \
      fprintf(stderr, "line %d: %s\n", __LINE__, #x);             \
      exit(1);                                                    \
    }                                                             \
  } while (0)

static std::mt19937 rng(7);
static int pick(int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); }

static void check_pages(const kv_pages &kv, int n_pages) {
  std::set<int> all(kv.free_list.begin(), kv.free_list.end());
  CHECK(all.size() == kv.free_list.size());
  for (const kv_seq &s : kv.seqs) {
    CHECK((int)s.pages.size() == kv.pages_of(s.len));
    for (int p : s.pages) CHECK(all.insert(p).second);
  }
  CHECK((int)all.size() == n_pages && *all.begin() == 0 && *all.rbegin() == n_pages - 1);
}

static void check_work(const kv_pages &kv, const kv_batch_plan &p, int groups) {
  const int per_page = kv.page_tokens / PBX_KV_BLOCK;
  CHECK((int)p.row_pos.size() == p.n_rows);
  size_t bi = 0, ai = 0, ji = 0;
  int row0 = 0, tab = 0;
  std::set<int> slots;
  for (size_t i = 0; i < p.seqs.size(); ++i) {
    const kv_seq &s = kv.seqs[p.seqs[i]];
    const int start = p.starts[i], count = p.counts[i], end = start + count;
    CHECK(end <= s.len);
    if (!count) continue;
    for (int t = 0; t < count; ++t) CHECK(p.row_pos[row0 + t] == start + t);
    const int used = kv.pages_of(end);
    for (int k = 0; k < used; ++k) CHECK(p.table[tab + k] == s.pages[k]);
    // every touched block once
    for (int b = start / PBX_KV_BLOCK; b <= (end - 1) / PBX_KV_BLOCK; ++b, ++bi) {
      const kv_block_item &x = p.blocks[bi];
      CHECK(x.page == s.pages[b / per_page] && x.sub == b % per_page && x.pos0 == b * PBX_KV_BLOCK);
      CHECK(x.start == start && x.count == count && x.row0 == row0);
    }
    // every row in a tile, and every position that it sees in one of the tile's items
    int tiles = 0, row = 0;
    while (row < count * groups) {
      const int last = std::min(count * groups, row + 16) - 1;
      const int seen = start + last / groups + 1;  // positions
      int blk = 0, parts = 0;
      const size_t first = ai;
      while (ai < p.attn.size() && p.attn[ai].row0 == row0 && p.attn[ai].tile == tiles) {
        const kv_attn_item &x = p.attn[ai++];
        CHECK(x.start == start && x.count == count && x.tab == tab);
        CHECK(x.blk0 == blk && x.blk1 > x.blk0 && (x.blk1 - 1) / per_page < used);
        blk = x.blk1;
        ++parts;
        if (x.slot >= 0) CHECK(x.slot < p.n_slots && slots.insert(x.slot).second);
      }
      CHECK(blk == (seen + PBX_KV_BLOCK - 1) / PBX_KV_BLOCK);
      if (parts > 1) {
        const kv_join_item &j = p.joins[ji++];
        CHECK(j.row0 == row0 && j.tile == tiles && j.count == count && j.n == parts);
        for (int k = 0; k < parts; ++k) CHECK(p.attn[first + k].slot == j.slot + k);
      } else {
        CHECK(p.attn[first].slot == -1);
      }
      row += 16;
      ++tiles;
    }
    row0 += count;
    tab += used;
  }
  CHECK(bi == p.blocks.size() && ai == p.attn.size() && ji == p.joins.size());
  CHECK((int)slots.size() == p.n_slots && row0 == p.n_rows && tab == (int)p.table.size());
}

int main() {
  int taken = 0, refused = 0;
  for (int round = 0; round < 300; ++round) {
    const int page = PBX_KV_BLOCK << pick(0, 5), n_pages = pick(1, 60), n_seqs = pick(1, 9);
    const int max_seq = pick(1, 3000), groups = pick(1, 40), heads = pick(1, 12);
    kv_pages kv;
    kv.init(page, n_pages, n_seqs, max_seq);
    for (int step = 0; step < 40; ++step) {
      std::string why;
      if (pick(0, 3) == 0) {
        const int s = pick(-1, n_seqs), had = s >= 0 && s < n_seqs ? kv.seqs[s].len : 0;
        const int n = pick(-1, had + 1);
        const int rc = kv.truncate(s, n, &why);
        CHECK((rc == PBX_OK) == (s >= 0 && s < n_seqs && n >= 0 && n <= had));
        CHECK((rc == PBX_OK) == why.empty());
        check_pages(kv, n_pages);
        continue;
      }
      std::vector<int> seqs, starts, counts;
      for (int s = 0; s < n_seqs; ++s)
        if (pick(0, 2)) seqs.push_back(pick(0, 40) ? s : pick(-1, n_seqs));
      std::shuffle(seqs.begin(), seqs.end(), rng);
      bool fits = true;
      std::set<int> once;
      const bool at_end = pick(0, 1);
      for (int s : seqs) {
        const bool known = s >= 0 && s < n_seqs;
        fits = fits && known && once.insert(s).second;
        const int len = known ? kv.seqs[s].len : 0;
        starts.push_back(at_end ? len : pick(0, 30) ? pick(0, len) : pick(-2, len + 2));
        counts.push_back(pick(0, 4) ? pick(0, 300) : pick(-1, 2));
        fits = fits && starts.back() >= 0 && starts.back() <= len && counts.back() >= 0 &&
               starts.back() + counts.back() <= max_seq;
      }
      const std::vector<kv_seq> before = kv.seqs;
      const std::vector<int> free_before = kv.free_list;
      kv_batch_plan p;
      const int rc = kv_plan_rows(&kv, (int)seqs.size(), seqs.data(), at_end ? nullptr : starts.data(),
                                  counts.data(), &p, &why);
      if (!fits) CHECK(rc == PBX_EINVAL);
      if (rc) {
        CHECK(rc == PBX_EINVAL ? !fits : rc == PBX_ENOMEM);
        CHECK(kv.free_list == free_before && !why.empty());
        for (int s = 0; s < n_seqs; ++s) CHECK(kv.seqs[s].len == before[s].len && kv.seqs[s].pages == before[s].pages);
        ++refused;
      } else {
        for (size_t i = 0; i < seqs.size(); ++i)
          CHECK(kv.seqs[seqs[i]].len == std::max(before[seqs[i]].len, starts[i] + counts[i]));
        kv_plan_work(kv, groups, heads, pick(1, 2000), &p);
        check_work(kv, p, groups);
        bool last = true;
        for (size_t i = 0; i < seqs.size(); ++i) {
          last = last && (!counts[i] || starts[i] + counts[i] == kv.seqs[seqs[i]].len);
          CHECK(kv_plan_reaches(p, seqs[i], starts[i] + counts[i] - 1) == (counts[i] > 0));
          CHECK(!kv_plan_reaches(p, seqs[i], starts[i] + counts[i]));
        }
        CHECK(p.last == last);
        ++taken;
      }
      check_pages(kv, n_pages);
    }
  }
  printf("taken %d refused %d\n", taken, refused);
  return 0;
}
