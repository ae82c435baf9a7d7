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

static void check_work(const kv_pages &kv, const kv_batch_plan &p, int groups, int max_u) {
  const int per_page = kv.page_tokens / PBX_KV_BLOCK;
  CHECK((int)p.row_pos.size() == p.n_rows);
  CHECK(p.n_attn[0] + p.n_attn[1] + p.n_attn[2] + p.n_attn[3] == (int)p.attn.size());
  // the items of a tile, by (first row, tile)
  std::map<std::pair<int, int>, std::vector<std::pair<kv_attn_item, int>>> items;
  int at = 0;
  for (int c = 0; c < 4; ++c)
    for (int k = 0; k < p.n_attn[c]; ++k, ++at) {
      CHECK(!k || p.attn[at - 1].blk1 - p.attn[at - 1].blk0 >= p.attn[at].blk1 - p.attn[at].blk0);
      items[{p.attn[at].row0, p.attn[at].tile}].push_back({p.attn[at], 1 << c});
    }
  size_t bi = 0, used_items = 0, last = 0;
  int row0 = 0, tab = 0;
  std::set<int> slots, joins;
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
      CHECK(items.count({row0, tiles}));
      auto list = items[{row0, tiles}];
      std::sort(list.begin(), list.end(), [](auto &x, auto &y) { return x.first.part < y.first.part; });
      const int u16 = list[0].second, parts = (int)list.size();
      CHECK(u16 <= max_u && parts <= KV_MAX_PARTS);
      const int bottom = std::min(count * groups, row + 16 * u16) - 1;
      const int seen = start + bottom / groups + 1;  // positions
      int blk = 0;
      for (int k = 0; k < parts; ++k) {
        const kv_attn_item &x = list[k].first;
        CHECK(list[k].second == u16 && x.part == k && x.parts == parts);
        CHECK(x.start == start && x.count == count && x.tab == tab);
        CHECK(x.blk0 == blk && x.blk1 > x.blk0 && (x.blk1 - 1) / per_page < used);
        for (int b = x.blk0; b < std::min(x.blk1, x.blk0 + 4); ++b)
          CHECK(x.pages[b / per_page - x.blk0 / per_page] == s.pages[b / per_page]);
        blk = x.blk1;
        CHECK(x.slot == list[0].first.slot && x.join == list[0].first.join);
        for (int u = 0; parts > 1 && u < u16; ++u)
          CHECK(x.slot + k * u16 + u < p.n_slots && slots.insert(x.slot + k * u16 + u).second);
      }
      CHECK(blk == (seen + PBX_KV_BLOCK - 1) / PBX_KV_BLOCK);
      if (parts > 1) CHECK(list[0].first.join < p.n_joins && joins.insert(list[0].first.join).second);
      used_items += parts;
      row += 16 * u16;
      ++tiles;
    }
    row0 += count;
    tab += used;
    CHECK(last < p.last_rows.size() && p.last_rows[last] == row0 - 1);
    ++last;
  }
  CHECK(last == p.last_rows.size());
  CHECK(bi == p.blocks.size() && used_items == p.attn.size() && (int)joins.size() == p.n_joins);
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
        const int max_u = 1 << pick(0, 3);
        kv_plan_work(kv, groups, heads, max_u, pick(1, 2000), &p);
        check_work(kv, p, groups, max_u);
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
