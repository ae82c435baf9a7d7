// Random batches, forks, compactions and truncations over the paged KV cache's host
// bookkeeping (purebee_amd/csrc/runtime/pbx_kv_plan.h), with what the kernels would do
// played on rows of numbers: every sequence has to hold its own rows at every step,
// and pages have to add up.
#include "pbx_kv_plan.h"

#include <stdlib.h>

#include <random>

#define CHECK(x)                                                  \
  do {                                                            \
    if (!(x)) {                                                   \
      fprintf(stderr, "line %d: %s\n", __LINE__, #x);             \
      exit(1);                                                    \
    }                                                             \
  } while (0)

static std::mt19937 rng(11);
static int pick(int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); }

struct World {
  kv_pages kv;
  int n_pages;
  std::vector<std::vector<int>> pool;  // [page][slot]: a row's number
  std::vector<std::vector<int>> want;  // [sequence]: its rows

  void check() {
    std::vector<int> refs(n_pages, 0);
    for (size_t s = 0; s < kv.seqs.size(); ++s) {
      const kv_seq &q = kv.seqs[s];
      CHECK(q.len == (int)want[s].size() && (int)q.pages.size() == kv.pages_of(q.len));
      for (int32_t p : q.pages) ++refs[p];
      for (int t = 0; t < q.len; ++t) CHECK(pool[q.pages[t / kv.page_tokens]][t % kv.page_tokens] == want[s][t]);
    }
    for (int32_t p : kv.free_list) CHECK(refs[p] == 0);
    int used = 0;
    for (int p = 0; p < n_pages; ++p) {
      CHECK(kv.refs[p] == refs[p]);
      used += refs[p] > 0;
    }
    CHECK(used + (int)kv.free_list.size() == n_pages);
  }
};

static bool same(const World &w, const std::vector<kv_seq> &seqs, const std::vector<int32_t> &free_list,
                 const std::vector<int32_t> &refs) {
  for (size_t s = 0; s < seqs.size(); ++s)
    if (seqs[s].len != w.kv.seqs[s].len || seqs[s].pages != w.kv.seqs[s].pages) return false;
  return free_list == w.kv.free_list && refs == w.kv.refs;
}

int main() {
  int grown = 0, copies = 0, packs = 0, many = 0, refused = 0, forks = 0, row = 0;
  for (int round = 0; round < 400; ++round) {
    World w;
    const int page = PBX_KV_BLOCK << pick(0, 3), n_seqs = pick(1, 8), max_seq = pick(40, 2000);
    w.n_pages = pick(1, 40);
    w.kv.init(page, w.n_pages, n_seqs, max_seq);
    w.pool.assign(w.n_pages, std::vector<int>(page, -1));
    w.want.assign(n_seqs, {});
    for (int step = 0; step < 60; ++step) {
      std::string why;
      const std::vector<kv_seq> seqs0 = w.kv.seqs;
      const std::vector<int32_t> free0 = w.kv.free_list, refs0 = w.kv.refs;
      std::vector<int> seqs;
      for (int s = 0; s < n_seqs; ++s)
        if (pick(0, 1)) seqs.push_back(s);
      std::shuffle(seqs.begin(), seqs.end(), rng);
      const int n = (int)seqs.size(), what = pick(0, 5);
      if (what == 0) {
        const int s = pick(0, n_seqs - 1), to = pick(0, w.kv.seqs[s].len);
        CHECK(w.kv.truncate(s, to, &why) == PBX_OK);
        w.want[s].resize(to);
      } else if (what <= 2) {  // forks
        std::vector<int> srcs, lens;
        bool ok = true;
        for (int i = 0; i < n; ++i) {
          srcs.push_back(pick(0, 60) ? pick(0, n_seqs - 1) : pick(-1, n_seqs));
          const bool known = srcs[i] >= 0 && srcs[i] < n_seqs;
          lens.push_back(known ? pick(0, 60) ? pick(0, w.kv.seqs[srcs[i]].len) : w.kv.seqs[srcs[i]].len + 1 : 0);
          ok = ok && known && lens[i] <= w.kv.seqs[srcs[i]].len;
        }
        const bool all = pick(0, 1);
        if (all) {
          ok = true;
          for (int s : srcs) ok = ok && s >= 0 && s < n_seqs;
        }
        if (n && !pick(0, 30)) {
          seqs.push_back(seqs[0]);
          srcs.push_back(0);
          lens.push_back(0);
          ok = false;
        }
        const int rc = w.kv.fork((int)seqs.size(), seqs.data(), srcs.data(), all ? nullptr : lens.data(), &why);
        CHECK((rc == PBX_OK) == ok && (rc == PBX_OK) == why.empty());
        if (rc) {
          CHECK(rc == PBX_EINVAL && same(w, seqs0, free0, refs0));
          ++refused;
        } else {
          const auto had = w.want;
          for (int i = 0; i < n; ++i) {
            w.want[seqs[i]] = had[srcs[i]];
            if (!all) w.want[seqs[i]].resize(lens[i]);
          }
          ++forks;
        }
      } else if (what == 3) {  // a compaction
        std::vector<int> counts, at;
        bool ok = true;
        for (int s : seqs) {
          const int len = w.kv.seqs[s].len, begin = (int)at.size();
          const int lead = pick(0, 2) ? pick(0, len) : 0, odds = pick(1, 6);
          for (int t = 0; t < len; ++t)
            if (t < lead || pick(1, odds) == 1) at.push_back(t);
          if (!pick(0, 60) && (int)at.size() > begin + 1) {
            std::swap(at[begin], at.back());
            ok = false;
          }
          if (!pick(0, 60) && (int)at.size() > begin) {
            at.back() = len;
            ok = false;
          }
          counts.push_back((int)at.size() - begin);
        }
        kv_pack_plan p;
        const int rc = kv_plan_pack(&w.kv, n, seqs.data(), counts.data(), at.data(), &p, &why);
        if (!ok) CHECK(rc == PBX_EINVAL);
        if (rc) {
          CHECK((rc == PBX_EINVAL) == !ok && (ok ? rc == PBX_ENOMEM : true) && !why.empty());
          CHECK(same(w, seqs0, free0, refs0));
          ++refused;
        } else if (!pick(0, 9)) {
          kv_pack_undo(&w.kv, &p);
          CHECK(same(w, seqs0, free0, refs0));
        } else {
          size_t k = 0;
          for (int32_t m : p.launches) {
            CHECK(m > 0);
            const auto before = w.pool;  // a launch's blocks run in any order
            std::vector<char> written(w.n_pages, 0);
            for (int32_t i = 0; i < m; ++i) written[p.items[k + i].page] = 1;
            for (int32_t i = 0; i < m; ++i, ++k) {
              const kv_pack_item &x = p.items[k];
              CHECK(x.rows > 0 && x.rows <= PBX_KV_BLOCK && x.pos0 % PBX_KV_BLOCK == 0);
              CHECK(x.at >= 0 && x.at + x.rows <= (int)p.rows.size());
              for (int t = 0; t < x.rows; ++t) {
                const int pos = p.rows[x.at + t].pos, from = p.rows[x.at + t].page;
                CHECK(from >= 0 && from < w.n_pages && !written[from]);
                CHECK(pos >= x.pos0 + t && (x.raw < 0 || (x.raw == from && pos == x.pos0 + t)));
                w.pool[x.page][x.sub * PBX_KV_BLOCK + t] = before[from][pos % page];
              }
            }
          }
          CHECK(k == p.items.size());
          int c = 0;
          for (int i = 0; i < n; ++i) {
            std::vector<int> made;
            for (int t = 0; t < counts[i]; ++t) made.push_back(w.want[seqs[i]][at[c++]]);
            w.want[seqs[i]] = made;
          }
          ++packs;
          many += p.launches.size() > 1;
        }
      } else {  // a batch
        std::vector<int> starts, counts;
        const bool at_end = pick(0, 2);
        for (int s : seqs) {
          const int len = w.kv.seqs[s].len;
          starts.push_back(at_end ? len : pick(0, len));
          counts.push_back(std::min(max_seq - starts.back(), pick(0, 1) ? pick(0, 3) : pick(0, 150)));
        }
        kv_batch_plan p;
        const int rc = kv_plan_rows(&w.kv, n, seqs.data(), starts.data(), counts.data(), &p, &why);
        if (rc) {
          CHECK(rc == PBX_ENOMEM && same(w, seqs0, free0, refs0) && !why.empty());
          ++refused;
        } else if (!pick(0, 9)) {
          kv_plan_undo(&w.kv, p);
          std::vector<int32_t> f = w.kv.free_list, g = free0;
          std::sort(f.begin(), f.end());
          std::sort(g.begin(), g.end());
          CHECK(f == g && w.kv.refs == refs0);
        } else {
          for (const kv_page_copy &x : p.copies) {
            CHECK(x.from != x.to && x.blocks > 0 && x.blocks * PBX_KV_BLOCK <= page);
            for (int t = 0; t < x.blocks * PBX_KV_BLOCK; ++t) w.pool[x.to][t] = w.pool[x.from][t];
            ++copies;
          }
          for (int i = 0; i < n; ++i) {
            const int s = seqs[i], end = starts[i] + counts[i], had = (int)w.want[s].size();
            if (end <= had) continue;  // (rows that were there: such a batch only reads here)
            w.want[s].resize(end);
            for (int t = starts[i]; t < end; ++t) {
              const int at = w.kv.seqs[s].pages[t / page];
              CHECK(w.kv.refs[at] == 1);
              w.want[s][t] = w.pool[at][t % page] = ++row;
            }
            ++grown;
          }
        }
      }
      w.check();
    }
  }
  printf("grown %d copies %d packs %d launches %d refused %d forks %d\n", grown, copies, packs, many, refused, forks);
  return 0;
}
