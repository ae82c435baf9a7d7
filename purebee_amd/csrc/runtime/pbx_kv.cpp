// pbx_kv.cpp -- the paged 8-bit KV cache of include/pbx.h: pool, batches and
// the launches of pbx_kv.hip.

#include "pbx_internal.h"
#include "pbx_kv_plan.h"

#include <math.h>
#include <string.h>

#include <new>

#define PBX_KV_MAGIC 0x5042584Bu        // "PBXK"
#define PBX_KV_BATCH_MAGIC 0x50425842u  // "PBXB"

struct KvArgsHost {  // KvArgs in pbx_kv.hip
  uint8_t *codes;    // of the layer
  float *scales;
  int kv_heads, groups, head_dim, page_shift;
};

struct KvRopeHost {  // KvRope in pbx_kv.hip
  const double *table;
  int style, dim;
};

// Lists that a call makes on the host: written to coherent pinned memory, from where a
// kernel copies them to the device, in order with the context's other work (setting a
// small batch took 17.6 us with a copy operation of the runtime, 14.2 so).
struct kv_lists {
  int32_t *host = nullptr, *mapped = nullptr, *dev = nullptr;
  size_t host_cap = 0, dev_cap = 0;
  hipEvent_t copied = nullptr;

  int make() { return hipEventCreateWithFlags(&copied, hipEventDisableTiming) == hipSuccess ? PBX_OK : PBX_EHIP; }
  void release() {
    if (dev) hipFree(dev);
    if (host) hipHostFree(host);
    if (copied) hipEventDestroy(copied);
  }
};

struct pbx_kv {
  uint32_t magic = PBX_KV_MAGIC;
  pbx_ctx *c = nullptr;
  pbx_kv_config cfg;
  int hdp = 0;         // head_dim padded to the kernels' width
  int page_shift = 0;  // log2 of the blocks of a page
  kv_pages pages;
  uint8_t *codes = nullptr;  // [layer][page][kv head][block][keys 32 hdp | values 32 hdp]
  float *scales = nullptr;   // [layer][page][kv head][block][key, value]
  double *rope = nullptr;    // [max_seq][rope_dim / 2][cos, sin]
  size_t layer_codes = 0, layer_scales = 0, bytes = 0;
  // the kernels for this head size; attention by log2 of the query tiles (4 at most)
  hipFunction_t append = nullptr, read = nullptr, pack = nullptr, attn[3] = {};
  std::vector<pbx_kv_batch *> batches;
  kv_lists lists;        // of a compaction
  kv_pack_plan packing;  // the last one, whose memory the next one uses
};

struct pbx_kv_batch {
  uint32_t magic = PBX_KV_BATCH_MAGIC;
  pbx_kv *kv = nullptr;
  kv_batch_plan plan;
  bool set = false;
  bool stale = false;     // positions of it were dropped or moved
  bool captured = false;  // a graph may hold its calls
  bool appends = false;   // appends among them
  uint64_t alone = 0;     // forks after which its rows' pages were seen to be its sequences' alone, and one
  // the plan on the device: blocks, attention items, row positions, last rows, page ids
  // and page copies
  kv_lists lists;
  size_t at_attn = 0, at_pos = 0, at_last = 0, at_table = 0, at_copies = 0;
  float *part = nullptr;  // partial results of split rows
  size_t part_cap = 0;
  // [split rows][KV head][32] parts done so far (zero between launches), each count in a
  // cache line of its own: atomics on one line queue up
  unsigned *arrived = nullptr;
  size_t arrived_cap = 0;
};

static bool kv_ok(const pbx_kv *kv) { return kv && kv->magic == PBX_KV_MAGIC; }
static bool batch_ok(const pbx_kv_batch *b) { return b && b->magic == PBX_KV_BATCH_MAGIC; }

// Padded head dims that the kernels are built for.
static int kv_padded(int hd) {
  for (int w : {32, 64, 96, 128, 192, 256})
    if (hd <= w) return w;
  return 0;
}

// Threads of the append and read workgroups (append_threads of pbx_kv.hip).
static int kv_threads(int hdp) { return hdp <= 64 ? 256 : 4 * hdp; }

static int pack_threads(int hdp) { return hdp <= 64 ? 256 : 2 * hdp; }  // likewise

// 16-row query tiles of the widest attention kernel for a head size.
static int kv_max_tiles(int hdp) { return hdp <= 64 ? 4 : 2; }

static int kv_launch(pbx_ctx *c, hipFunction_t f, const char *name, int64_t grid, int block, void **args) {
  if (grid > 0x7fffffff) return pbx_fail(c, PBX_ENOTSUP, "kv: %lld workgroups", (long long)grid);
  return pbx_launch_fn(c, f, name, dim3((unsigned)grid), dim3(block), args, c->stream);
}

// Items of a launch at most, where each is a workgroup (of up to 512 threads) a layer and
// KV head: a grid holds less than 2^32 threads.
static int kv_items_a_launch(const pbx_kv_config &g) {
  return (int)std::max<int64_t>(1, (1 << 22) / ((int64_t)g.n_kv_heads * g.n_layers));
}

// Room for n words of lists, whose last ones the device has read.
static int lists_room(pbx_ctx *c, kv_lists *l, size_t n, const char *who) {
  if (hipEventSynchronize(l->copied) != hipSuccess)
    return pbx_fail(c, PBX_EHIP, "%s: waiting for the last lists failed", who);
  const size_t bytes = (n * 4 + 15) / 16 * 16;
  const int rc = pbx_ensure_mapped(c, (void **)&l->host, (void **)&l->mapped, &l->host_cap, bytes);
  return rc ? rc : pbx_ensure_dev(c, (void **)&l->dev, &l->dev_cap, bytes);
}
static int lists_send(pbx_ctx *c, kv_lists *l, size_t n, const char *who) {
  int64_t n16 = (int64_t)(n + 3) / 4;
  void *args[] = {&l->mapped, &l->dev, &n16};
  const int rc = pbx_launch(c, PBX_K_COPY16, dim3((unsigned)std::min<int64_t>((n16 + 255) / 256, 1024)), dim3(256), args);
  if (rc) return rc;
  return hipEventRecord(l->copied, c->stream) == hipSuccess ? PBX_OK
                                                            : pbx_fail(c, PBX_EHIP, "%s: event record failed", who);
}

bool pbx_capturing(pbx_ctx *c) {
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  return hipStreamIsCapturing(c->stream, &st) != hipSuccess || st != hipStreamCaptureStatusNone;
}

// Creating and freeing wait for the stream, which would end a capture.
int pbx_not_capturing(pbx_ctx *c, const char *who) {
  return pbx_capturing(c) ? pbx_fail(c, PBX_EINVAL, "%s: the context's stream is being captured", who) : PBX_OK;
}

static void batch_release(pbx_kv_batch *b) {
  b->lists.release();
  if (b->part) hipFree(b->part);
  if (b->arrived) hipFree(b->arrived);
  b->magic = 0;
  delete b;
}

static void kv_release(pbx_kv *kv) {
  for (pbx_kv_batch *b : kv->batches) batch_release(b);
  for (void *p : {(void *)kv->codes, (void *)kv->scales, (void *)kv->rope})
    if (p) hipFree(p);
  kv->lists.release();
  kv->magic = 0;
  delete kv;
}

void pbx_kv_release_all(pbx_ctx *c) {
  auto *list = (std::vector<pbx_kv *> *)c->kvs;
  if (!list) return;
  for (pbx_kv *kv : *list) kv_release(kv);
  delete list;
  c->kvs = nullptr;
}

static int kv_check(pbx_ctx *c, const pbx_kv_config &g) {
  if (g.n_layers <= 0 || g.n_heads <= 0 || g.n_kv_heads <= 0 || g.n_pages <= 0 || g.max_seqs <= 0 ||
      g.max_seq <= 0)
    return pbx_fail(c, PBX_EINVAL, "pbx_kv_create: every size must be positive");
  if (g.n_heads % g.n_kv_heads)
    return pbx_fail(c, PBX_EINVAL, "pbx_kv_create: need n_kv_heads | n_heads");
  if (g.head_dim % 4 || g.head_dim < 32 || g.head_dim > 256)
    return pbx_fail(c, PBX_ENOTSUP, "pbx_kv_create: head_dim %d unsupported (32..256, %%4)", g.head_dim);
  if (g.page_tokens < PBX_KV_BLOCK || g.page_tokens > 1024 || (g.page_tokens & (g.page_tokens - 1)))
    return pbx_fail(c, PBX_EINVAL, "pbx_kv_create: page_tokens %d (32, 64, .. 1024)", g.page_tokens);
  if (g.max_seq > (1 << 20) || g.n_kv_heads > 65535 || g.n_heads > 1024 || g.max_seqs > (1 << 20) || g.n_pages > (1 << 26))
    return pbx_fail(c, PBX_ENOTSUP, "pbx_kv_create: max_seq %d, n_heads %d, max_seqs %d or n_pages %d too large",
                    g.max_seq, g.n_heads, g.max_seqs, g.n_pages);
  if (g.rope_style != PBX_ROPE_NONE && g.rope_style != PBX_ROPE_PAIRS && g.rope_style != PBX_ROPE_HALVES)
    return pbx_fail(c, PBX_EINVAL, "pbx_kv_create: rope_style %d", g.rope_style);
  if (g.rope_style == PBX_ROPE_NONE) return PBX_OK;
  if (g.rope_dim < 0 || g.rope_dim > g.head_dim || g.rope_dim % 4)
    return pbx_fail(c, PBX_EINVAL, "pbx_kv_create: rope_dim %d (a multiple of 4 up to head_dim)", g.rope_dim);
  if (!(g.rope_theta > 0) || !(g.rope_scale > 0) || !isfinite(g.rope_theta) || !isfinite(g.rope_scale))
    return pbx_fail(c, PBX_EINVAL, "pbx_kv_create: rope_theta and rope_scale must be positive");
  const int rd = g.rope_dim ? g.rope_dim : g.head_dim;
  for (int i = 0; g.rope_factors && i < rd / 2; ++i)
    if (!(g.rope_factors[i] > 0) || !isfinite(g.rope_factors[i]))
      return pbx_fail(c, PBX_EINVAL, "pbx_kv_create: rope_factors[%d] must be positive", i);
  return PBX_OK;
}

static int kv_make(pbx_ctx *c, const pbx_kv_config &g, pbx_kv *kv) {
  kv->c = c;
  kv->cfg = g;
  kv->hdp = kv_padded(g.head_dim);
  if (g.rope_style == PBX_ROPE_NONE)
    kv->cfg.rope_dim = 0;
  else if (!g.rope_dim)
    kv->cfg.rope_dim = g.head_dim;
  const int per_page = g.page_tokens / PBX_KV_BLOCK;
  while ((1 << kv->page_shift) < per_page) ++kv->page_shift;
  kv->pages.init(g.page_tokens, g.n_pages, g.max_seqs, g.max_seq);
  // (sizes that overflow would pass for small ones)
  if ((double)g.n_layers * g.n_pages * g.n_kv_heads * g.page_tokens * kv->hdp > 0x1p46)
    return pbx_fail(c, PBX_ENOMEM, "pbx_kv_create: a pool of more than 2^47 bytes");
  const size_t blocks = (size_t)g.n_pages * g.n_kv_heads * per_page;
  kv->layer_codes = blocks * 2 * PBX_KV_BLOCK * kv->hdp;
  kv->layer_scales = blocks * 2;
  const int half = kv->cfg.rope_dim / 2;
  const size_t codes = kv->layer_codes * g.n_layers, scales = kv->layer_scales * g.n_layers * 4;
  const size_t table = (size_t)g.max_seq * half * 16;
  std::vector<double> freq(half + 1);
  for (int i = 0; i < half; ++i)
    freq[i] = pow(g.rope_theta, -2.0 * i / kv->cfg.rope_dim) / g.rope_scale /
              (g.rope_factors ? (double)g.rope_factors[i] : 1.0);
  kv->cfg.rope_factors = nullptr;  // the caller's array need not outlive the call
  if (hipSetDevice(c->device) != hipSuccess)
    return pbx_fail(c, PBX_EHIP, "pbx_kv_create: hipSetDevice failed");
  const std::string hdp = std::to_string(kv->hdp);
  kv->append = pbx_kernel_by_name(c, "pbx_kv_append_" + hdp);
  kv->read = pbx_kernel_by_name(c, "pbx_kv_read_" + hdp);
  kv->pack = pbx_kernel_by_name(c, "pbx_kv_pack_" + hdp);
  bool found = kv->append && kv->read && kv->pack;
  for (int k = 0; 1 << k <= kv_max_tiles(kv->hdp); ++k) {
    kv->attn[k] = pbx_kernel_by_name(c, "pbx_kv_attn_" + hdp + "_" + std::to_string(1 << k));
    found = found && kv->attn[k];
  }
  if (!found) return pbx_fail(c, PBX_ELOAD, "pbx_kv_create: kernels for head_dim %d not found", g.head_dim);
  if (kv->lists.make())
    return pbx_fail(c, PBX_EHIP, "pbx_kv_create: event creation failed");
  double *dfreq = nullptr;
  if (hipMalloc((void **)&kv->codes, codes) != hipSuccess ||
      hipMalloc((void **)&kv->scales, scales) != hipSuccess ||
      (half && (hipMalloc((void **)&kv->rope, table) != hipSuccess ||
                hipMalloc((void **)&dfreq, half * 8) != hipSuccess))) {
    (void)hipGetLastError();
    return pbx_fail(c, PBX_ENOMEM, "pbx_kv_create: %zu bytes of device memory", codes + scales + table);
  }
  kv->bytes = codes + scales + table;
  int rc = PBX_OK;
  if (hipMemsetAsync(kv->codes, 0x80, codes, c->stream) != hipSuccess ||  // code 0
      hipMemsetAsync(kv->scales, 0, scales, c->stream) != hipSuccess)
    rc = pbx_fail(c, PBX_EHIP, "pbx_kv_create: clearing the pool failed");
  if (!rc && half) {
    if (hipMemcpyAsync(dfreq, freq.data(), half * 8, hipMemcpyHostToDevice, c->stream) != hipSuccess)
      rc = pbx_fail(c, PBX_EHIP, "pbx_kv_create: frequency copy failed");
    const int64_t n = (int64_t)g.max_seq * half;
    void *args[] = {&dfreq, &kv->rope, (void *)&half, (void *)&n};
    if (!rc) rc = kv_launch(c, c->fn[PBX_K_KV_ROPE_TABLE], "pbx_kv_rope_table", (n + 255) / 256, 256, args);
  }
  if (hipStreamSynchronize(c->stream) != hipSuccess && !rc)
    rc = pbx_fail(c, PBX_EHIP, "pbx_kv_create: initialisation failed");
  if (dfreq) hipFree(dfreq);
  return rc;
}

extern "C" int pbx_kv_create(pbx_ctx *c, const pbx_kv_config *cfg, pbx_kv **out) {
  if (!c) return pbx_fail(nullptr, PBX_EINVAL, "pbx_kv_create: ctx is NULL");
  if (!cfg || !out) return pbx_fail(c, PBX_EINVAL, "pbx_kv_create: NULL argument");
  *out = nullptr;
  int rc = kv_check(c, *cfg);
  if (rc || (rc = pbx_not_capturing(c, "pbx_kv_create"))) return rc;
  pbx_kv *kv = nullptr;
  try {
    kv = new pbx_kv();
    if (!c->kvs) c->kvs = new std::vector<pbx_kv *>();
    auto *list = (std::vector<pbx_kv *> *)c->kvs;
    list->reserve(list->size() + 1);
    if (!(rc = kv_make(c, *cfg, kv))) {
      list->push_back(kv);
      *out = kv;
      return PBX_OK;
    }
  } catch (const std::bad_alloc &) {
    rc = pbx_fail(c, PBX_ENOMEM, "pbx_kv_create: out of host memory");
  }
  if (kv) kv_release(kv);
  return rc;
}

extern "C" int pbx_kv_free(pbx_kv *kv) {
  if (!kv) return PBX_OK;
  if (!kv_ok(kv)) return pbx_fail(nullptr, PBX_EINVAL, "pbx_kv_free: not a live cache");
  pbx_ctx *c = kv->c;
  if (const int rc = pbx_not_capturing(c, "pbx_kv_free")) return rc;
  hipSetDevice(c->device);
  hipStreamSynchronize(c->stream);
  auto *list = (std::vector<pbx_kv *> *)c->kvs;
  list->erase(std::remove(list->begin(), list->end(), kv), list->end());
  kv_release(kv);
  return PBX_OK;
}

extern "C" int pbx_kv_info(const pbx_kv *kv, int *free_pages, size_t *device_bytes) {
  if (!kv_ok(kv)) return pbx_fail(nullptr, PBX_EINVAL, "pbx_kv_info: not a live cache");
  if (free_pages) *free_pages = (int)kv->pages.free_list.size();
  if (device_bytes) *device_bytes = kv->bytes;
  return PBX_OK;
}

extern "C" int pbx_kv_length(const pbx_kv *kv, int seq, int *n) {
  if (!kv_ok(kv)) return pbx_fail(nullptr, PBX_EINVAL, "pbx_kv_length: not a live cache");
  if (!n || seq < 0 || seq >= kv->cfg.max_seqs)
    return pbx_fail(kv->c, PBX_EINVAL, "pbx_kv_length: sequence %d outside [0, %d)", seq, kv->cfg.max_seqs);
  *n = kv->pages.seqs[seq].len;
  return PBX_OK;
}

extern "C" int pbx_kv_truncate(pbx_kv *kv, int seq, int n) try {
  if (!kv_ok(kv)) return pbx_fail(nullptr, PBX_EINVAL, "pbx_kv_truncate: not a live cache");
  std::string why;
  const int rc = kv->pages.truncate(seq, n, &why);
  if (rc) return pbx_fail(kv->c, rc, "pbx_kv_truncate: %s", why.c_str());
  for (pbx_kv_batch *b : kv->batches)
    if (kv_plan_reaches(b->plan, seq, n)) b->stale = true;
  return PBX_OK;
} catch (const std::bad_alloc &) {
  return pbx_fail(kv->c, PBX_ENOMEM, "pbx_kv_truncate: out of host memory");
}

extern "C" int pbx_kv_fork(pbx_kv *kv, int n, const int32_t *dsts, const int32_t *srcs, const int32_t *lens) {
  const char *who = "pbx_kv_fork";
  if (!kv_ok(kv)) return pbx_fail(nullptr, PBX_EINVAL, "%s: not a live cache", who);
  pbx_ctx *c = kv->c;
  if (n < 0 || (n && (!dsts || !srcs))) return pbx_fail(c, PBX_EINVAL, "%s: bad arguments", who);
  if (const int rc = pbx_not_capturing(c, who)) return rc;
  kv_pages &pages = kv->pages;
  const int known = (int)pages.seqs.size();
  // replays of a captured append write its rows' pages, whoever holds them by then
  for (const pbx_kv_batch *b : kv->batches) {
    if (!b->appends || b->stale) continue;
    for (int i = 0; i < n; ++i) {
      const int s = srcs[i];
      if (s < 0 || s >= known || s == dsts[i]) continue;
      const int len = lens ? lens[i] : pages.seqs[s].len;
      for (size_t k = 0; k < b->plan.seqs.size(); ++k)
        if (b->plan.seqs[k] == s && b->plan.counts[k] && b->plan.starts[k] / pages.page_tokens < pages.pages_of(len))
          return pbx_fail(c, PBX_EINVAL, "%s: a captured graph appends to pages of sequence %d", who, s);
    }
  }
  try {
    std::string why;
    const int rc = pages.fork(n, dsts, srcs, lens, &why);
    if (rc) return pbx_fail(c, rc, "%s: %s", who, why.c_str());
    for (pbx_kv_batch *b : kv->batches)
      if (kv_plan_moved(pages, b->plan)) b->stale = true;
  } catch (const std::bad_alloc &) {
    return pbx_fail(c, PBX_ENOMEM, "%s: out of host memory", who);
  }
  return PBX_OK;
}

struct KvPackHost {  // KvPack in pbx_kv.hip
  uint8_t *codes;
  float *scales;
  int64_t layer_codes, layer_scales;  // from one layer to the next
  const int32_t *items, *rows;
  int n_items, kv_heads, head_dim, page_shift;
};

extern "C" int pbx_kv_compact(pbx_kv *kv, int n, const int32_t *seqs, const int32_t *counts,
                              const int32_t *positions) {
  const char *who = "pbx_kv_compact";
  if (!kv_ok(kv)) return pbx_fail(nullptr, PBX_EINVAL, "%s: not a live cache", who);
  pbx_ctx *c = kv->c;
  if (n < 0 || (n && (!seqs || !counts))) return pbx_fail(c, PBX_EINVAL, "%s: bad arguments", who);
  for (int i = 0; i < n; ++i)
    if (counts[i] > 0 && !positions) return pbx_fail(c, PBX_EINVAL, "%s: positions is NULL", who);
  if (int rc = pbx_not_capturing(c, who)) return rc;
  if (hipSetDevice(c->device) != hipSuccess) return pbx_fail(c, PBX_EHIP, "%s: hipSetDevice failed", who);
  const pbx_kv_config &g = kv->cfg;
  try {
    std::string why;
    kv_pack_plan &p = kv->packing;
    int rc = kv_plan_pack(&kv->pages, n, seqs, counts, positions, &p, &why);
    if (rc) return pbx_fail(c, rc, "%s: %s", who, why.c_str());
    const size_t n_items = p.items.size() * sizeof(kv_pack_item) / 4;
    const size_t words = n_items + p.rows.size() * sizeof(kv_pack_row) / 4;
    bool lost = false;  // a launch that wrote pages given back before is under way
    if (words) {
      kv_lists &l = kv->lists;
      if (!(rc = lists_room(c, &l, words, who))) {
        memcpy(l.host, p.items.data(), n_items * 4);
        memcpy(l.host + n_items, p.rows.data(), p.rows.size() * sizeof(kv_pack_row));
        rc = lists_send(c, &l, words, who);
      }
      KvRopeHost r{kv->rope, g.rope_style, g.rope_dim};
      const int32_t *items = l.dev;
      const int most = kv_items_a_launch(g);
      for (size_t k = 0; k < p.launches.size() && !rc; ++k)
        for (int at = 0; at < p.launches[k] && !rc; at += most) {
          const int here = std::min(most, p.launches[k] - at);
          KvPackHost a{kv->codes, kv->scales, (int64_t)kv->layer_codes, (int64_t)kv->layer_scales, items,
                       l.dev + n_items, here, g.n_kv_heads, g.head_dim, kv->page_shift};
          void *args[] = {&a, &r};
          rc = kv_launch(c, kv->pack, "pbx_kv_pack", (int64_t)here * g.n_kv_heads * g.n_layers, pack_threads(kv->hdp),
                         args);
          lost = lost || (!rc && k);  // (the first ones write pages that were free)
          items += (size_t)here * sizeof(kv_pack_item) / 4;
        }
    }
    if (rc && !lost) {
      kv_pack_undo(&kv->pages, &p);
      return rc;
    }
    if (rc) kv_pack_cut(&kv->pages, p);
    for (pbx_kv_batch *b : kv->batches)
      if (kv_plan_moved(kv->pages, b->plan)) b->stale = true;
    return rc;
  } catch (const std::bad_alloc &) {
    return pbx_fail(c, PBX_ENOMEM, "%s: out of host memory", who);
  }
}

extern "C" int pbx_kv_batch_create(pbx_kv *kv, pbx_kv_batch **out) {
  if (!kv_ok(kv)) return pbx_fail(nullptr, PBX_EINVAL, "pbx_kv_batch_create: not a live cache");
  if (!out) return pbx_fail(kv->c, PBX_EINVAL, "pbx_kv_batch_create: NULL argument");
  *out = nullptr;
  if (const int rc = pbx_not_capturing(kv->c, "pbx_kv_batch_create")) return rc;
  try {
    kv->batches.reserve(kv->batches.size() + 1);
    pbx_kv_batch *b = new pbx_kv_batch();
    b->kv = kv;
    if (hipSetDevice(kv->c->device) != hipSuccess || b->lists.make()) {
      delete b;
      return pbx_fail(kv->c, PBX_EHIP, "pbx_kv_batch_create: event creation failed");
    }
    kv->batches.push_back(b);
    *out = b;
  } catch (const std::bad_alloc &) {
    return pbx_fail(kv->c, PBX_ENOMEM, "pbx_kv_batch_create: out of host memory");
  }
  return PBX_OK;
}

extern "C" int pbx_kv_batch_free(pbx_kv_batch *b) {
  if (!b) return PBX_OK;
  if (!batch_ok(b)) return pbx_fail(nullptr, PBX_EINVAL, "pbx_kv_batch_free: not a live batch");
  pbx_kv *kv = b->kv;
  if (const int rc = pbx_not_capturing(kv->c, "pbx_kv_batch_free")) return rc;
  hipSetDevice(kv->c->device);
  hipStreamSynchronize(kv->c->stream);
  kv->batches.erase(std::remove(kv->batches.begin(), kv->batches.end(), b), kv->batches.end());
  batch_release(b);
  return PBX_OK;
}

extern "C" int pbx_kv_batch_rows(const pbx_kv_batch *b, int *n_rows) {
  if (!batch_ok(b)) return pbx_fail(nullptr, PBX_EINVAL, "pbx_kv_batch_rows: not a live batch");
  if (!n_rows) return pbx_fail(b->kv->c, PBX_EINVAL, "pbx_kv_batch_rows: NULL argument");
  *n_rows = b->set ? b->plan.n_rows : 0;
  return PBX_OK;
}

// Copies the plan's lists to the device, one after the other.
static int batch_upload(pbx_kv_batch *b) {
  pbx_kv *kv = b->kv;
  pbx_ctx *c = kv->c;
  const kv_batch_plan &p = b->plan;
  const size_t n_blocks = p.blocks.size() * sizeof(kv_block_item) / 4;
  b->at_attn = n_blocks;
  b->at_pos = b->at_attn + p.attn.size() * sizeof(kv_attn_item) / 4;
  b->at_last = b->at_pos + p.row_pos.size();
  b->at_table = b->at_last + p.last_rows.size();
  b->at_copies = b->at_table + p.table.size();
  const size_t n = b->at_copies + p.copies.size() * sizeof(kv_page_copy) / 4;
  if (!n) return PBX_OK;
  int rc = lists_room(c, &b->lists, n, "pbx_kv_batch_set");
  if (rc) return rc;
  int32_t *host = b->lists.host;
  auto put = [&](size_t at, const void *from, size_t bytes) {
    if (bytes) memcpy(host + at, from, bytes);
  };
  put(0, p.blocks.data(), n_blocks * 4);
  put(b->at_attn, p.attn.data(), p.attn.size() * sizeof(kv_attn_item));
  put(b->at_pos, p.row_pos.data(), p.row_pos.size() * 4);
  put(b->at_last, p.last_rows.data(), p.last_rows.size() * 4);
  put(b->at_table, p.table.data(), p.table.size() * 4);
  put(b->at_copies, p.copies.data(), p.copies.size() * sizeof(kv_page_copy));
  // per slot and KV head: 16 rows of hdp sums, then their maxima and weights
  const size_t part = (size_t)p.n_slots * kv->cfg.n_kv_heads * 16 * (kv->hdp + 2) * 4;
  const size_t joins = (size_t)p.n_joins * kv->cfg.n_kv_heads * 128, joins_had = b->arrived_cap;
  if (part && ((rc = pbx_ensure_dev(c, (void **)&b->part, &b->part_cap, part)) ||
               (rc = pbx_ensure_dev(c, (void **)&b->arrived, &b->arrived_cap, joins))))
    return rc;
  if (b->arrived_cap != joins_had && hipMemsetAsync(b->arrived, 0, b->arrived_cap, c->stream) != hipSuccess) {
    hipFree(b->arrived);
    b->arrived = nullptr;
    b->arrived_cap = 0;
    return pbx_fail(c, PBX_EHIP, "pbx_kv_batch_set: clearing the counts failed");
  }
  return lists_send(c, &b->lists, n, "pbx_kv_batch_set");
}

// Whether batch o, of another plan than the last one, runs over pages that this one's
// sequences left for copies.
static bool knows_left(const pbx_kv *kv, const pbx_kv_batch *o) { return !o->stale && kv_plan_moved(kv->pages, o->plan); }

// Other batches that run over sequences which get copies of pages know the old pages: they
// have to be set again, and a graph that holds one cannot be, so then the batch is refused.
static int batch_may_own(const pbx_kv_batch *b, const kv_batch_plan &p) {
  for (const pbx_kv_batch *o : b->kv->batches)
    if (!p.copies.empty() && o != b && o->captured && knows_left(b->kv, o))
      return pbx_fail(b->kv->c, PBX_EINVAL, "pbx_kv_batch_set: a captured graph runs over pages that a sequence shares "
                      "and would leave");
  return PBX_OK;
}

// Pages that the batch's sequences shared, copied for them.
static int batch_own_pages(pbx_kv_batch *b) {
  pbx_kv *kv = b->kv;
  pbx_ctx *c = kv->c;
  const kv_batch_plan &p = b->plan;
  if (p.copies.empty()) return PBX_OK;
  const int32_t *copies = b->lists.dev + b->at_copies;
  const pbx_kv_config &g = kv->cfg;
  const int most = kv_items_a_launch(g), all = (int)p.copies.size();
  for (int at = 0; at < all; at += most) {
    KvPackHost a{kv->codes, kv->scales, (int64_t)kv->layer_codes, (int64_t)kv->layer_scales,
                 copies + (size_t)at * sizeof(kv_page_copy) / 4, nullptr, std::min(most, all - at), g.n_kv_heads,
                 2 * PBX_KV_BLOCK * kv->hdp, kv->page_shift};
    void *args[] = {&a};
    const int rc = kv_launch(c, c->fn[PBX_K_KV_COPY], "pbx_kv_copy", (int64_t)a.n_items * g.n_kv_heads * g.n_layers, 256,
                             args);
    if (rc) return rc;
  }
  for (pbx_kv_batch *o : kv->batches)
    if (o != b && knows_left(kv, o)) o->stale = true;
  return PBX_OK;
}

extern "C" int pbx_kv_batch_set(pbx_kv_batch *b, int n, const int32_t *seqs, const int32_t *starts,
                                const int32_t *counts) {
  if (!batch_ok(b)) return pbx_fail(nullptr, PBX_EINVAL, "pbx_kv_batch_set: not a live batch");
  pbx_kv *kv = b->kv;
  pbx_ctx *c = kv->c;
  if (n < 0 || (n && (!seqs || !counts)))
    return pbx_fail(c, PBX_EINVAL, "pbx_kv_batch_set: bad arguments");
  if (hipSetDevice(c->device) != hipSuccess)
    return pbx_fail(c, PBX_EHIP, "pbx_kv_batch_set: hipSetDevice failed");
  if (b->captured || pbx_capturing(c))
    return pbx_fail(c, PBX_EINVAL, "pbx_kv_batch_set: the batch's calls are captured in a graph, or its stream "
                    "is being captured");
  try {
    std::string why;
    kv_batch_plan plan;
    int rc = kv_plan_rows(&kv->pages, n, seqs, starts, counts, &plan, &why);
    if (rc) return pbx_fail(c, rc, "pbx_kv_batch_set: %s", why.c_str());
    if ((rc = batch_may_own(b, plan))) {
      kv_plan_undo(&kv->pages, plan);
      return rc;
    }
    b->set = false;
    try {
      std::swap(b->plan, plan);
      b->plan.take_lists(&plan);
      kv_plan_work(kv->pages, kv->cfg.n_heads / kv->cfg.n_kv_heads, kv->cfg.n_kv_heads, kv_max_tiles(kv->hdp),
                   2 * c->cu_count, &b->plan);
      rc = batch_upload(b);
      if (!rc) rc = batch_own_pages(b);
    } catch (const std::bad_alloc &) {
      rc = pbx_fail(c, PBX_ENOMEM, "pbx_kv_batch_set: out of host memory");
    }
    if (rc) {  // the sequences stay as they were
      kv_plan_undo(&kv->pages, b->plan);
      return rc;
    }
  } catch (const std::bad_alloc &) {
    return pbx_fail(c, PBX_ENOMEM, "pbx_kv_batch_set: out of host memory");
  }
  b->set = true;
  b->stale = false;
  b->alone = 0;
  return PBX_OK;
}

// A launch of a batch's call; one that goes into a graph holds the batch's rows from then on.
static int batch_launch(pbx_kv_batch *b, hipFunction_t f, const char *name, int64_t grid, int block, void **args) {
  pbx_ctx *c = b->kv->c;
  const int rc = kv_launch(c, f, name, grid, block, args);
  if (!rc && pbx_capturing(c)) {
    b->captured = true;
    b->appends = b->appends || f == b->kv->append;
  }
  return rc;
}

// What the three calls check alike; fills the kernels' view of the layer.
static int batch_begin(pbx_kv_batch *b, const char *who, int layer, KvArgsHost *a) {
  if (!batch_ok(b)) return pbx_fail(nullptr, PBX_EINVAL, "%s: not a live batch", who);
  pbx_kv *kv = b->kv;
  pbx_ctx *c = kv->c;
  const pbx_kv_config &g = kv->cfg;
  if (!b->set) return pbx_fail(c, PBX_EINVAL, "%s: the batch is not set", who);
  if (b->stale) return pbx_fail(c, PBX_EINVAL, "%s: positions of the batch were dropped or moved", who);
  if (layer < 0 || layer >= g.n_layers)
    return pbx_fail(c, PBX_EINVAL, "%s: layer %d outside [0, %d)", who, layer, g.n_layers);
  if (hipSetDevice(c->device) != hipSuccess) return pbx_fail(c, PBX_EHIP, "%s: hipSetDevice failed", who);
  *a = {kv->codes + layer * kv->layer_codes, kv->scales + layer * kv->layer_scales, g.n_kv_heads,
        g.n_heads / g.n_kv_heads, g.head_dim, kv->page_shift};
  return PBX_OK;
}

int pbx_kv_batch_look(const pbx_kv_batch *b, pbx_kv_batch_view *out) {
  if (!batch_ok(b)) return pbx_fail(nullptr, PBX_EINVAL, "not a live batch");
  if (!b->set) return pbx_fail(b->kv->c, PBX_EINVAL, "the batch is not set");
  *out = {b->kv->c, &b->kv->cfg, b->plan.n_rows, (int)b->plan.last_rows.size(), b->lists.dev + b->at_last};
  return PBX_OK;
}

static int rows_check(pbx_ctx *c, const char *who, const char *what, const void *p, int64_t *stride, int heads,
                      int head_dim) {
  const int64_t row = (int64_t)heads * head_dim;
  if (!*stride) *stride = row;
  if (!p) return pbx_fail(c, PBX_EINVAL, "%s: %s is NULL", who, what);
  if ((uintptr_t)p % 16 || *stride % 4 || *stride < row || *stride > (1ll << 40))
    return pbx_fail(c, PBX_EINVAL, "%s: %s needs a 16-byte aligned address and a stride of at least %lld floats, "
                    "a multiple of 4", who, what, (long long)row);
  return PBX_OK;
}

extern "C" int pbx_kv_append_dev(pbx_kv_batch *b, int layer, const float *dQ, int64_t q_stride, const float *dK,
                                 int64_t k_stride, const float *dV, int64_t v_stride, float *dQout,
                                 int64_t qout_stride) {
  const char *who = "pbx_kv_append_dev";
  KvArgsHost a;
  int rc = batch_begin(b, who, layer, &a);
  if (rc) return rc;
  pbx_kv *kv = b->kv;
  pbx_ctx *c = kv->c;
  const pbx_kv_config &g = kv->cfg;
  if (!b->plan.last)
    return pbx_fail(c, PBX_EINVAL, "%s: the batch's rows are not the last of their sequences", who);
  for (size_t i = 0; i < b->plan.seqs.size(); ++i)
    if (b->plan.counts[i] && kv->pages.seqs[b->plan.seqs[i]].len != b->plan.starts[i] + b->plan.counts[i])
      return pbx_fail(c, PBX_EINVAL, "%s: sequence %d grew past the batch's rows", who, b->plan.seqs[i]);
  if (!b->plan.n_rows) return PBX_OK;
  // a batch that lengthened its sequences got pages of their own for its rows; since then, or
  // where it runs over rows that were there, others may share them
  const kv_pages &pages = kv->pages;
  if (b->alone != pages.forks + 1) {
    for (size_t i = 0; i < b->plan.seqs.size(); ++i) {
      const int s = b->plan.seqs[i], end = b->plan.starts[i] + b->plan.counts[i];
      for (int j = b->plan.starts[i] / pages.page_tokens; b->plan.counts[i] && j < pages.pages_of(end); ++j)
        if (pages.refs[pages.seqs[s].pages[j]] > 1)
          return pbx_fail(c, PBX_EINVAL, "%s: sequence %d shares pages of the batch's rows: truncate it to %d and set "
                          "the batch again", who, s, b->plan.starts[i]);
    }
    b->alone = pages.forks + 1;
  }
  if ((rc = rows_check(c, who, "dK", dK, &k_stride, g.n_kv_heads, g.head_dim)) ||
      (rc = rows_check(c, who, "dV", dV, &v_stride, g.n_kv_heads, g.head_dim)))
    return rc;
  if (dQ || dQout) {
    if ((rc = rows_check(c, who, "dQ", dQ, &q_stride, g.n_heads, g.head_dim)) ||
        (rc = rows_check(c, who, "dQout", dQout, &qout_stride, g.n_heads, g.head_dim)))
      return rc;
    if (dQ == dQout && q_stride != qout_stride)
      return pbx_fail(c, PBX_EINVAL, "%s: queries rotated in place need one stride", who);
  }
  KvRopeHost r{kv->rope, g.rope_style, g.rope_dim};
  const int32_t *items = b->lists.dev, *pos = b->lists.dev + b->at_pos;
  const int n_blocks = (int)b->plan.blocks.size();
  void *args[] = {&a, &r, &items, (void *)&n_blocks, &pos, &dK, &k_stride, &dV, &v_stride, &dQ, &q_stride,
                  &dQout, &qout_stride};
  return batch_launch(b, kv->append, "pbx_kv_append", (int64_t)n_blocks * g.n_kv_heads + (dQ ? b->plan.n_rows : 0),
                      kv_threads(kv->hdp), args);
}

extern "C" int pbx_kv_attention_dev(pbx_kv_batch *b, int layer, const float *dQ, int64_t q_stride, float scale,
                                    float *dOut, int64_t out_stride) {
  const char *who = "pbx_kv_attention_dev";
  KvArgsHost a;
  int rc = batch_begin(b, who, layer, &a);
  if (rc) return rc;
  pbx_kv *kv = b->kv;
  pbx_ctx *c = kv->c;
  const pbx_kv_config &g = kv->cfg;
  if (!b->plan.n_rows) return PBX_OK;
  if (!isfinite(scale)) return pbx_fail(c, PBX_EINVAL, "%s: scale is not finite", who);
  if ((rc = rows_check(c, who, "dQ", dQ, &q_stride, g.n_heads, g.head_dim)) ||
      (rc = rows_check(c, who, "dOut", dOut, &out_stride, g.n_heads, g.head_dim)))
    return rc;
  if (dQ == dOut && q_stride != out_stride)
    return pbx_fail(c, PBX_EINVAL, "%s: attention in place needs one stride", who);
  if (scale == 0.f) scale = (float)(1.0 / sqrt((double)g.head_dim));
  const int32_t *items = b->lists.dev + b->at_attn, *table = b->lists.dev + b->at_table;
  for (int k = 0; k < 3; ++k) {
    const int n = b->plan.n_attn[k];
    if (!n) continue;
    void *args[] = {&a, &items, &table, &dQ, &q_stride, &scale, &dOut, &out_stride, &b->part, &b->arrived};
    if ((rc = batch_launch(b, kv->attn[k], "pbx_kv_attn", (int64_t)n * g.n_kv_heads, 256, args))) return rc;
    items += n * (sizeof(kv_attn_item) / 4);
  }
  return PBX_OK;
}

extern "C" int pbx_kv_read_dev(pbx_kv_batch *b, int layer, float *dK, int64_t k_stride, float *dV,
                               int64_t v_stride) {
  const char *who = "pbx_kv_read_dev";
  KvArgsHost a;
  int rc = batch_begin(b, who, layer, &a);
  if (rc) return rc;
  pbx_kv *kv = b->kv;
  pbx_ctx *c = kv->c;
  const pbx_kv_config &g = kv->cfg;
  if (!b->plan.n_rows || (!dK && !dV)) return PBX_OK;
  if ((dK && (rc = rows_check(c, who, "dK", dK, &k_stride, g.n_kv_heads, g.head_dim))) ||
      (dV && (rc = rows_check(c, who, "dV", dV, &v_stride, g.n_kv_heads, g.head_dim))))
    return rc;
  const int32_t *items = b->lists.dev;
  void *args[] = {&a, &items, &dK, &k_stride, &dV, &v_stride};
  return batch_launch(b, kv->read, "pbx_kv_read", (int64_t)b->plan.blocks.size() * g.n_kv_heads,
                      kv_threads(kv->hdp), args);
}
