// pbx_logprobs.cpp -- the log probability entry points of include/pbx.h.

#include "pbx_internal.h"

#include <algorithm>

// LP_T * LP_SHARE * 4 of pbx_logprobs.hip: elements of one workgroup at most,
// in the kernels of 512 and of 256 threads
#define LP_ELEMENTS (512 * 64 * 4)
#define LP_ELEMENTS_256 (256 * 8 * 4)
#define LP_MERGED_ROWS 512  // of pbx_logprobs.hip, too

struct LogprobsOutHost {  // Out in pbx_logprobs.hip
  const int32_t *targets;
  float *logp, *entropy;
  int32_t *top_ids;
  float *top_logp;
};

static int lp_check(pbx_ctx *c, const char *who, int64_t rows, int64_t vocab, int top) {
  if (rows < 0 || vocab <= 0 || top < 0 || top > vocab)
    return pbx_fail(c, PBX_EINVAL, "%s: rows %lld, vocab %lld, top %d", who, (long long)rows, (long long)vocab, top);
  if (top > PBX_LOGPROBS_TOP_MAX || vocab > (1 << 28) || rows > (1 << 24))
    return pbx_fail(c, PBX_ENOTSUP, "%s: at most %d top tokens, 2^28 logits a row and 2^24 rows", who,
                    PBX_LOGPROBS_TOP_MAX);
  return PBX_OK;
}

// Workgroups a row: as many as fill the GPU twice over, of at least 4096
// logits, and no more logits than a workgroup can take.  Up to LP_WHOLE logits
// one workgroup is done before several and their join are (one row of 20,000:
// 8.6 against 10.4 us, 60 of 32,003: 10.8 against 12.2; its time grows by 0.09 us
// per 1,000).
#define LP_WHOLE 36000

static int64_t lp_parts(const pbx_ctx *c, int64_t rows, int64_t vocab) {
  if (vocab <= LP_WHOLE) return 1;
  const int64_t least = (vocab + 3 + 8 + LP_ELEMENTS - 1) / LP_ELEMENTS;
  const int64_t fill = 2 * c->cu_count / std::max<int64_t>(rows, 1);
  return std::max(least, std::min<int64_t>({fill, (vocab + 4095) / 4096, 64}));
}

static size_t lp_bytes(int64_t rows, int64_t parts, int top) {
  return parts == 1 ? 0 : ((size_t)rows * parts * (8 * (size_t)top + 12) + 15) / 16 * 16;
}

extern "C" int pbx_logprobs_workspace(pbx_ctx *c, int64_t rows, int64_t vocab, int top, size_t *bytes) {
  if (!c) return pbx_fail(nullptr, PBX_EINVAL, "pbx_logprobs_workspace: ctx is NULL");
  if (!bytes) return pbx_fail(c, PBX_EINVAL, "pbx_logprobs_workspace: NULL argument");
  const int rc = lp_check(c, "pbx_logprobs_workspace", rows, vocab, top);
  if (!rc) *bytes = lp_bytes(rows, lp_parts(c, rows, vocab), top);
  return rc;
}

extern "C" int pbx_logprobs_dev(pbx_ctx *c, const float *dLogits, int64_t stride, int64_t rows, int64_t vocab,
                                const int32_t *dTargets, int top, float *dLogp, float *dEntropy,
                                int32_t *dTopIds, float *dTopLogp, void *work, size_t work_bytes) {
  const char *who = "pbx_logprobs_dev";
  if (!c) return pbx_fail(nullptr, PBX_EINVAL, "%s: ctx is NULL", who);
  int rc = lp_check(c, who, rows, vocab, top);
  if (rc) return rc;
  if (!stride) stride = vocab;
  if (stride < vocab) return pbx_fail(c, PBX_EINVAL, "%s: stride %lld < vocab", who, (long long)stride);
  if (!rows) return PBX_OK;
  if (!dLogits || (uintptr_t)dLogits % 4 || (!dTargets != !dLogp))
    return pbx_fail(c, PBX_EINVAL, "%s: dLogits, and dTargets and dLogp together, are needed", who);
  if (!dTopIds && !dTopLogp) top = 0;
  if (!top) dTopIds = nullptr, dTopLogp = nullptr;
  int64_t parts64 = lp_parts(c, rows, vocab);
  const size_t need = lp_bytes(rows, parts64, top);
  if (need && (!work || work_bytes < need || (uintptr_t)work % 16))
    return pbx_fail(c, PBX_EINVAL, "%s: needs %zu bytes of 16-byte aligned workspace, got %zu", who, need, work_bytes);
  if (rows * parts64 > 0x7fffffff) return pbx_fail(c, PBX_ENOTSUP, "%s: too many rows", who);
  if (hipSetDevice(c->device) != hipSuccess) return pbx_fail(c, PBX_EHIP, "%s: hipSetDevice failed", who);
  // (a part has at most a group more than its even share)
  const bool small = (vocab + 3) / parts64 + 8 <= LP_ELEMENTS_256;
  LogprobsOutHost out{dTargets, dLogp, dEntropy, dTopIds, dTopLogp};
  int v = (int)vocab, parts = (int)parts64;
  void *keys = work;
  float *sums = need ? (float *)((char *)work + 8 * (size_t)rows * parts * top) : nullptr;
  // The last workgroup of a row joins its parts in the same launch, except where
  // the launch may run beside another of this context (a captured one replayed on
  // another stream): the counts are the context's.
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  int merged = parts > 1 && rows <= LP_MERGED_ROWS &&
               hipStreamIsCapturing(c->stream, &st) == hipSuccess && st == hipStreamCaptureStatusNone;
  void *args[] = {(void *)&dLogits, &stride, &v, &parts, &top, &out, &sums, &keys, &merged};
  rc = pbx_launch(c, small ? PBX_K_LOGPROBS_PART_256 : PBX_K_LOGPROBS_PART_512, dim3((unsigned)(rows * parts)),
                  dim3(small ? 256 : 512), args);
  if (rc || parts == 1 || merged) return rc;
  return pbx_launch(c, PBX_K_LOGPROBS_JOIN, dim3((unsigned)rows), dim3(256), args);
}
