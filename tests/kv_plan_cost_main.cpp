// The cost of planning a small batch beside the number of sequences that the
// cache could hold, and a plan that is taken back
// (purebee_amd/csrc/runtime/pbx_kv_plan.h).
#include "pbx_kv_plan.h"

#include <stdlib.h>

#include <chrono>

#define CHECK(x)                                                  \
  do {                                                            \
    if (!(x)) {                                                   \
      fprintf(stderr, "line %d: %s\n", __LINE__, #x);             \
      exit(1);                                                    \
    }                                                             \
  } while (0)

// Nanoseconds of planning and taking back a batch of two sequences, the least of many.
static double cost(int max_seqs) {
  kv_pages kv;
  kv.init(64, 64, max_seqs, 4096);
  const int32_t seqs[2] = {max_seqs - 1, 3}, counts[2] = {1, 70};
  std::string why;
  double least = 1e30;
  for (int i = 0; i < 300; ++i) {
    const auto a = std::chrono::steady_clock::now();
    kv_batch_plan p;
    CHECK(kv_plan_rows(&kv, 2, seqs, nullptr, counts, &p, &why) == PBX_OK);
    CHECK(kv.seqs[3].len == 70 && kv.seqs[max_seqs - 1].len == 1 && kv.free_list.size() == 61);
    kv_plan_undo(&kv, p);
    const auto b = std::chrono::steady_clock::now();
    CHECK(kv.seqs[3].len == 0 && kv.seqs[max_seqs - 1].len == 0 && kv.free_list.size() == 64);
    least = std::min(least, std::chrono::duration<double, std::nano>(b - a).count());
  }
  return least;
}

int main() {
  // taken back: a sequence that grew over a page, one that did not, one whose rows lay inside it
  kv_pages kv;
  kv.init(32, 10, 4, 1000);
  std::string why;
  const int32_t seqs[3] = {2, 0, 1}, first[3] = {40, 5, 64}, more[3] = {30, 0, 10}, starts[3] = {40, 5, 3};
  kv_batch_plan p;
  CHECK(kv_plan_rows(&kv, 3, seqs, nullptr, first, &p, &why) == PBX_OK);
  const std::vector<kv_seq> held = kv.seqs;
  const std::vector<int32_t> free_pages = kv.free_list;
  CHECK(kv_plan_rows(&kv, 3, seqs, starts, more, &p, &why) == PBX_OK);
  CHECK(kv.seqs[2].len == 70 && kv.seqs[2].pages.size() == 3);
  kv_plan_undo(&kv, p);
  for (int s = 0; s < 4; ++s) CHECK(kv.seqs[s].len == held[s].len && kv.seqs[s].pages == held[s].pages);
  CHECK(kv.free_list == free_pages);
  // a sequence twice is refused in one batch, and in one after the other is not
  const int32_t twice[2] = {1, 1}, ones[2] = {1, 1};
  for (int i = 0; i < 3; ++i) {
    CHECK(kv_plan_rows(&kv, 2, twice, nullptr, ones, &p, &why) == PBX_EINVAL);
    CHECK(kv_plan_rows(&kv, 1, twice, nullptr, ones, &p, &why) == PBX_OK);
  }
  CHECK(kv.seqs[1].len == 67);
  const double few = cost(64), many = cost(1 << 20);
  printf("ns %.0f %.0f\n", few, many);
  return 0;
}
