// The paged KV cache's calls (purebee_amd/csrc/runtime/pbx_kv.cpp) with a GPU that only counts
// launches, and refuses one where it is told to: what errors leave of sequences and batches.
#include "pbx_internal.h"

#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <functional>
#include <new>
#include <string>
#include <vector>

#define CHECK(x)                                                  \
  do {                                                            \
    if (!(x)) {                                                   \
      fprintf(stderr, "line %d: %s (%s)\n", __LINE__, #x, said);  \
      exit(1);                                                    \
    }                                                             \
  } while (0)

static char said[512];
static int packs = 0, refuse_pack = -1;  // launches of compactions so far, and the one that fails
static bool capturing = false;

static int left = -1;  // allocations that succeed, -1: all
void *operator new(size_t n) {
  if (left >= 0 && left-- == 0) {
    left = 0;
    throw std::bad_alloc();
  }
  void *p = malloc(n ? n : 1);
  if (!p) throw std::bad_alloc();
  return p;
}
void operator delete(void *p) noexcept { free(p); }
void operator delete(void *p, size_t) noexcept { free(p); }

extern "C" {
hipError_t hipMalloc(void **p, size_t n) { return (*p = calloc(1, n ? n : 1)) ? hipSuccess : hipErrorOutOfMemory; }
hipError_t hipFree(void *p) { return free(p), hipSuccess; }
hipError_t hipHostFree(void *p) { return free(p), hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipMemcpyAsync(void *, const void *, size_t, hipMemcpyKind, hipStream_t) { return hipSuccess; }
hipError_t hipMemsetAsync(void *, int, size_t, hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *s) {
  *s = capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
  return hipSuccess;
}
hipError_t hipEventCreateWithFlags(hipEvent_t *e, unsigned) { return *e = (hipEvent_t)1, hipSuccess; }
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
}

int pbx_fail(pbx_ctx *, int code, const char *fmt, ...) {
  va_list a;
  va_start(a, fmt);
  vsnprintf(said, sizeof said, fmt, a);
  va_end(a);
  return code;
}
hipFunction_t pbx_kernel_by_name(pbx_ctx *, const std::string &) { return (hipFunction_t)1; }
int pbx_launch(pbx_ctx *, int, dim3, dim3, void **, hipStream_t) { return PBX_OK; }
int pbx_launch_fn(pbx_ctx *c, hipFunction_t, const char *name, dim3, dim3, void **, hipStream_t) {
  if (!strcmp(name, "pbx_kv_pack") && packs++ == refuse_pack) return pbx_fail(c, PBX_EHIP, "refused");
  return PBX_OK;
}
static int ensure(void **p, size_t *cap, size_t need) {
  if (*cap >= need) return PBX_OK;
  free(*p);
  *p = calloc(1, need);
  *cap = need;
  return PBX_OK;
}
int pbx_ensure_dev(pbx_ctx *, void **p, size_t *cap, size_t need) { return ensure(p, cap, need); }
int pbx_ensure_mapped(pbx_ctx *, void **h, void **d, size_t *cap, size_t need) {
  const int rc = ensure(h, cap, need);
  *d = *h;
  return rc;
}

struct Cache {
  pbx_ctx c;
  pbx_kv *kv = nullptr;

  explicit Cache(int pages) {
    pbx_kv_config g{};
    g.n_layers = 1, g.n_heads = g.n_kv_heads = 1, g.head_dim = 32, g.page_tokens = 32;
    g.n_pages = pages, g.max_seqs = 4, g.max_seq = 4096, g.rope_style = PBX_ROPE_NONE;
    CHECK(pbx_kv_create(&c, &g, &kv) == PBX_OK);
  }
  ~Cache() { pbx_kv_release_all(&c); }
  pbx_kv_batch *batch(int32_t seq, int32_t start, int32_t count) {
    pbx_kv_batch *b = nullptr;
    CHECK(pbx_kv_batch_create(kv, &b) == PBX_OK);
    CHECK(pbx_kv_batch_set(b, 1, &seq, &start, &count) == PBX_OK);
    return b;
  }
  int length(int seq) {
    int n = -1;
    CHECK(pbx_kv_length(kv, seq, &n) == PBX_OK);
    return n;
  }
  int free_pages() {
    int n = -1;
    CHECK(pbx_kv_info(kv, &n, nullptr) == PBX_OK);
    return n;
  }
  int compact(int32_t seq, const std::vector<int32_t> &kept) {
    const int32_t count = (int32_t)kept.size();
    packs = 0;
    return pbx_kv_compact(kv, 1, &seq, &count, kept.data());
  }
};

static int read(pbx_kv_batch *b) {
  static float4 out[8 * 256];
  return pbx_kv_read_dev(b, 0, (float *)out, 0, nullptr, 0);
}

// Positions but those from `at` on, `n` of them.
static std::vector<int32_t> without(int len, int at, int n) {
  std::vector<int32_t> kept;
  for (int i = 0; i < len; ++i)
    if (i < at || i >= at + n) kept.push_back(i);
  return kept;
}

// A compaction in a pool with one free page takes a launch a page, of which one fails.
static void failed_compactions() {
  for (int fails = 0; fails < 3; ++fails) {
    Cache k(6);
    k.batch(1, 0, 20);
    pbx_kv_batch *all = k.batch(0, 0, 128), *first = k.batch(0, 0, 32), *other = k.batch(1, 0, 20);
    CHECK(k.free_pages() == 1);
    refuse_pack = fails;
    CHECK(k.compact(0, without(128, 40, 3)) == PBX_EHIP);
    refuse_pack = -1;
    CHECK(packs == fails + 1);
    CHECK(read(first) == PBX_OK && read(other) == PBX_OK);  // what did not move is still there
    CHECK(k.length(1) == 20);
    if (fails < 2) {  // nothing was written but the page that was free
      CHECK(k.length(0) == 128 && k.free_pages() == 1 && read(all) == PBX_OK);
    } else {  // positions that moved are partly in pages that were given back
      CHECK(k.length(0) == 32 && k.free_pages() == 4);
      CHECK(read(all) == PBX_EINVAL && strstr(said, "dropped or moved"));
    }
    CHECK(k.compact(0, without(k.length(0), 3, 1)) == PBX_OK && k.length(0) == (fails < 2 ? 127 : 31));
  }
}

// A batch that is refused, because a captured graph reads a page that its sequence would
// leave, stays what it was.
static void refused_sets() {
  Cache k(8);
  pbx_kv_batch *b = k.batch(0, 0, 50), *reads = nullptr;
  const int32_t one = 1, zero = 0, more = 2;
  CHECK(pbx_kv_fork(k.kv, 1, &one, &zero, nullptr) == PBX_OK);
  b = k.batch(1, 0, 50);
  reads = k.batch(1, 0, 50);
  capturing = true;
  CHECK(read(reads) == PBX_OK);
  CHECK(pbx_kv_batch_set(b, 1, &one, nullptr, &more) == PBX_EINVAL);  // (inside a capture none is set)
  capturing = false;
  int rows = 0;
  for (int again = 0; again < 2; ++again) {
    CHECK(pbx_kv_batch_set(b, 1, &one, nullptr, &more) == PBX_EINVAL && strstr(said, "captured graph"));
    CHECK(k.length(1) == 50 && k.free_pages() == 6);
    CHECK(pbx_kv_batch_rows(b, &rows) == PBX_OK && rows == 50 && read(b) == PBX_OK && read(reads) == PBX_OK);
  }
  CHECK(pbx_kv_batch_free(reads) == PBX_OK);
  CHECK(pbx_kv_batch_set(b, 1, &one, nullptr, &more) == PBX_OK && k.length(1) == 52 && k.free_pages() == 5);
}

// Every call with one allocation more each time, until it succeeds: until then it changes nothing.
static void memory_runs_out() {
  int refused = 0;
  Cache k(60);
  pbx_kv_batch *grown = k.batch(3, 0, 1), *kept = k.batch(0, 0, 700);
  auto until_done = [&](int expected, const std::function<int()> &call) {
    for (int n = 0;; ++n) {
      int had[4];
      for (int s = 0; s < 4; ++s) had[s] = k.length(s);
      const int pages = k.free_pages();
      left = n;
      const int rc = call();
      left = -1;
      if (rc == expected) break;
      CHECK(rc == PBX_ENOMEM && n < 200);
      ++refused;
      for (int s = 0; s < 4; ++s) CHECK(k.length(s) == had[s]);
      CHECK(k.free_pages() == pages && read(kept) == PBX_OK);
    }
  };
  const int32_t all[] = {1, 2, 3}, from[] = {0, 0, 0}, lens[] = {700, 50, 333}, rows[] = {40, 1, 90};
  until_done(PBX_OK, [&] { return pbx_kv_fork(k.kv, 3, all, from, lens); });
  CHECK(k.length(2) == 50 && k.free_pages() == 60 - 22);
  until_done(PBX_OK, [&] { return pbx_kv_batch_set(grown, 3, all, nullptr, rows); });
  CHECK(k.length(3) == 423 && read(grown) == PBX_OK);
  std::vector<int32_t> at = without(740, 100, 17);
  for (int32_t p : without(423, 0, 50)) at.push_back(p);
  const int32_t two[] = {1, 3}, counts[] = {723, 373};
  until_done(PBX_OK, [&] { return pbx_kv_compact(k.kv, 2, two, counts, at.data()); });
  CHECK(k.length(1) == 723 && k.length(3) == 373 && read(grown) == PBX_EINVAL);
  until_done(PBX_EINVAL, [&] { return pbx_kv_truncate(k.kv, 1, 1000); });
  until_done(PBX_EINVAL, [&] { return pbx_kv_truncate(k.kv, 7, 0); });
  for (int s = 0; s < 4; ++s) CHECK(pbx_kv_truncate(k.kv, s, 0) == PBX_OK);
  CHECK(k.free_pages() == 60 && refused > 30);
}

int main(int argc, char **argv) {
  const std::string what = argc > 1 ? argv[1] : "";
  if (what == "failed_compactions") failed_compactions();
  else if (what == "refused_sets") refused_sets();
  else if (what == "memory_runs_out") memory_runs_out();
  else return 2;
  return 0;
}
