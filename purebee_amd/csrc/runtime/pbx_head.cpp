// pbx_head.cpp -- log probabilities of rows straight from a head's weights and their
// gradient (include/pbx.h): pieces of the vocabulary, workspace and launches.

#include "pbx_internal.h"

#include <algorithm>
#include <new>
#include <string>

namespace {

struct BackArgsHost {  // BackArgs in pbx_head.hip
  const void *qs, *dsc, *msc, *hi, *lo, *G32, *peaks, *f_peaks;
  int n_f_peaks;
  float *part;
  int M, Mpad, K, B, blocks, rows, KS, add;
};

struct SixArgsHost {  // SixArgs in pbx_head.hip
  const void *qs, *dsc;
  const float *X;
  int N, SB;
  const int32_t *targets;
  void *parts;
  int n_parts;
  float *hit, *Z;
  int64_t stride;
};

struct ReduceArgsHost {  // ReduceArgs in pbx_head.hip
  const float *part;
  int KS, M, K, folds;
  const int32_t *targets;
  int vocab;
  const float *grad;
  float *dX;
  const float *hit, *others;
  int n_others, type;
  const void *qs, *dsc, *msc;
};

#define HEAD_SHARE 8192          // of pbx_head.hip, too
#define HEAD_PIECE (64u << 20)   // bytes of a piece's logits, or factors, at most
#define HEAD_PAIRS (128u << 20)  // bytes of a piece's weights as pairs at most
#define PAIRS_GROUPS 1024        // workgroups that make them at most

// The head's rows from v0 on (a multiple of 128), n of them.
pbx_weight rows_of(const pbx_weight &w, int64_t v0, int64_t n) {
  pbx_weight v = w;
  const size_t scales = w.type == PBX_TYPE_Q6_K ? w.K / 256 : w.B;
  const size_t row = w.type == PBX_TYPE_F32    ? w.K * 4
                     : w.type == PBX_TYPE_F16  ? w.K * 2
                     : w.type == PBX_TYPE_Q6_K ? scales * 208
                     : w.type == PBX_TYPE_Q8_0 ? scales * 32
                                               : scales * 16;
  v.qs = (char *)w.qs + v0 * row;
  if (w.d) v.d = (char *)w.d + v0 * scales * 2;
  if (w.m) v.m = (char *)w.m + v0 * scales * 2;
  v.Npad = w.Npad - v0;
  v.N = std::min(v.Npad, (n + 3) / 4 * 4);  // rows of logits begin 16-byte aligned; padding rows are zero
  return v;
}

// One to three rows of a Q6_K head have a kernel of their own: lanes of a row (eight a
// superblock, 64 at most) and workgroups, up to three a CU.
bool six(const pbx_weight *w, int64_t M) { return w->type == PBX_TYPE_Q6_K && M <= 3; }
int six_lanes(const pbx_weight *w) {
  int lanes = 8;
  while (lanes < 64 && lanes < w->K / 32) lanes *= 2;
  return lanes;
}
int six_groups(const pbx_ctx *c, const pbx_weight *w) {
  const int64_t steps = ((w->N + 3) / 4 * six_lanes(w) + 63) / 64;  // of a wave
  return (int)std::min<int64_t>(3 * c->cu_count, (steps + 3) / 4);
}

// F32 and Q6_K heads are turned into pairs of halves, a piece at a time, where that and
// the fp16 products (of 2 K columns) take less than kernels of their own: the fp32 matrix
// rate is a sixteenth of fp16's, and Q6_K's products are made for few rows.  Turning costs a
// pass over the head and 4 bytes written for each of its values (20000 x 2048 60 us from
// F32, 40 from Q6_K), so heads of under 10 million values are left as they are, but for
// gradients of many rows (us, as pairs / else):
// * gradient, Q6_K: 20000 x 512 40 rows 83 / 90, 500 rows 198 / 431; 20000 x 2048 40 rows 156 /
//   178, 500 rows 469 / 1091; 9000 x 2048 40 rows 110 / 109; 3000 x 1024 100 rows 80 / 59, 200 83 / 87.
// * gradient, F32: 20000 x 2048 2 rows 180 / 205, 4 rows 180 / 170, 16 rows 181 / 229, 500 rows 497 /
//   1194; 60000 x 512 4 rows 108 / 133; 3000 x 1024 100 rows 78 / 58, 200 rows 82 / 90.
// * sums, Q6_K: 20000 x 512 64 rows 48 / 36, 100 rows 53 / 58; 60000 x 512 500 rows 220 / 539;
//   20000 x 2048 200 rows 167 / 138, 500 rows 241 / 293.
// * sums, F32: 60000 x 512 2 rows 68 / 128, 100 rows 88 / 93; 20000 x 2048 8 rows 146 / 141, 32 rows 146 /
//   187, 100 rows 166 / 151, 200 rows 199 / 275.
bool pairs(const pbx_weight *w, int64_t M, bool grad) {
  const int64_t values = w->N * w->K, ten = 10000000;
  const bool shorter = w->K <= 1024;
  if (w->type == PBX_TYPE_Q6_K) {
    if (grad) return M > 32 && values * M >= 40 * ten;
    return shorter ? M >= 96 && values >= ten : M >= 320 && values >= 2 * ten;
  }
  if (w->type != PBX_TYPE_F32) return false;
  if (grad && M > 32 && values * M >= 60 * ten) return true;
  if (values < ten || M < 2) return false;
  if (grad) return shorter || M < 4 || M >= 8;
  return shorter || M >= 128 || (M >= 16 && M <= 32);
}
// A piece of such a head: an F16 weight of 2 K columns.
pbx_weight pairs_of(const pbx_weight &w, int64_t n, void *halves) {
  pbx_weight v;
  v.magic = w.magic;
  v.type = PBX_TYPE_F16;
  v.N = v.Npad = n;
  v.K = 2 * w.K;
  v.B = 2 * w.B;
  v.qs = halves;
  return v;
}

struct Plan {
  bool pairs;      // the head's pieces become pairs of halves
  bool fused;      // logits leave the GEMM as sums or as the gradient's factor, not as such
  int64_t piece;   // vocabulary entries of a piece, but for the last
  int n_pieces, n_parts;
  int Mpad, TT, KS, n_others;
  // workspace: byte offsets
  size_t gemm, z, parts, hit, others, g, peaks, part, halves, f, f_peaks, bytes;
};

size_t padded(size_t n) { return (n + 255) / 256 * 256; }

Plan make_plan(pbx_ctx *c, const pbx_weight *w, int64_t M, bool grad) {
  Plan p{};
  const int64_t V = w->N;
  p.TT = M > 32 ? 2 : 1;
  p.Mpad = M <= 32 ? 32 : (int)((M + 63) / 64 * 64);
  p.pairs = pairs(w, M, grad);
  p.fused = p.pairs || pbx_gemm_has_head(c, w, M);
  const int64_t K = p.pairs ? 2 * w->K : w->K;  // columns of the products
  const int64_t row = 4 * (grad ? p.Mpad : M);
  p.piece = std::min<int64_t>((V + 127) / 128 * 128, std::max<int64_t>(128, HEAD_PIECE / std::max<int64_t>(row, 256) / 128 * 128));
  if (p.fused && !grad) p.piece = (V + 127) / 128 * 128;
  // (the gradient's kernels address a piece's weights by 31 bits)
  if (grad) p.piece = std::min<int64_t>(p.piece, std::max<int64_t>(128, (int64_t)(1u << 31) / (2 * K) / 128 * 128 - 128));
  if (p.pairs) p.piece = std::min<int64_t>(p.piece, std::max<int64_t>(128, HEAD_PAIRS / (2 * K) / 128 * 128));
  p.n_pieces = (int)((V + p.piece - 1) / p.piece);
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t from = at;
    at += padded(n);
    return from;
  };
  const int64_t last = V - (p.n_pieces - 1) * p.piece;
  size_t gemm = 0;
  if (p.pairs) {
    const pbx_weight part = pairs_of(*w, p.piece, nullptr);
    gemm = pbx_gemm_head_space(&part, (int)M);
  } else if (p.fused)
    gemm = pbx_gemm_head_space(w, (int)M);
  else
    for (int64_t n : {std::min(p.piece, V), last}) {
      const pbx_weight part = rows_of(*w, 0, n);
      gemm = std::max(gemm, pbx_linear_space(c, &part, (int)M));
    }
  auto shares = [](int64_t n) { return (int)((n + HEAD_SHARE - 1) / HEAD_SHARE); };
  const bool alone = six(w, M) && !p.pairs;
  if (alone) gemm = 0;
  p.n_parts = alone ? six_groups(c, w) : p.fused ? (int)((V + 127) / 128) : (p.n_pieces - 1) * shares(p.piece) + shares(last);
  p.gemm = take(gemm);
  p.z = take(p.fused ? 0 : (size_t)M * p.piece * 4);
  p.hit = take((size_t)M * 4);
  if (!grad) {
    p.parts = take((size_t)M * p.n_parts * 16);
  } else {
    // of a piece, which the ones after it add to: by the GEMM's tiles, or pbx_head_g's blocks
    const int64_t first = std::min(p.piece, V);
    p.n_others = (int)(p.fused ? (first + 127) / 128 : (first + 31) / 32);
    p.others = take((size_t)M * p.n_others * 4);
    const int64_t tiles = (K + 127) / 128 * ((M + 32 * p.TT - 1) / (32 * p.TT));
    // about two waves a SIMD (an F32 head's workgroups are one wave, the others' four)
    const int waves = w->type == PBX_TYPE_F32 && !p.pairs ? 1 : 4;
    p.KS = (int)std::max<int64_t>(1, std::min<int64_t>(8 / waves * c->cu_count / tiles, p.piece / (32 * waves)));
    p.g = take((size_t)p.Mpad * p.piece * 4);
    p.peaks = take(PBX_HEAD_PEAKS * 4);
    p.part = take((size_t)p.KS * M * K * 4);
  }
  if (p.pairs) {
    p.halves = take((size_t)p.piece * K * 2);
    p.f = take((size_t)p.piece * 4);
    p.f_peaks = take(PAIRS_GROUPS * 4);
  }
  p.bytes = at;
  return p;
}

int check(pbx_ctx *c, const char *who, const pbx_weight *w, int64_t rows) {
  if (!pbx_weight_ok(w)) return pbx_fail(c, PBX_EINVAL, "%s: not a live weight handle", who);
  if (rows < 0) return pbx_fail(c, PBX_EINVAL, "%s: %lld rows", who, (long long)rows);
  if (w->type == PBX_TYPE_Q8_REF) return pbx_fail(c, PBX_ENOTSUP, "%s: a Q8_REF weight", who);
  if (rows > 65535 || w->N > (1 << 28)) return pbx_fail(c, PBX_ENOTSUP, "%s: at most 65,535 rows and 2^28 tokens", who);
  if (w->type == PBX_TYPE_Q6_K && w->B > 512)
    return pbx_fail(c, PBX_ENOTSUP, "%s: K=%lld exceeds the Q6_K limit of 16384", who, (long long)w->K);
  return PBX_OK;
}

int check_work(pbx_ctx *c, const char *who, const Plan &p, const void *work, size_t bytes) {
  if (!work || bytes < p.bytes || (uintptr_t)work % 256)
    return pbx_fail(c, PBX_EINVAL, "%s: needs %zu bytes of 256-byte aligned workspace, got %zu", who, p.bytes, bytes);
  if (hipSetDevice(c->device) != hipSuccess) return pbx_fail(c, PBX_EHIP, "%s: hipSetDevice failed", who);
  return PBX_OK;
}

int launch_six(pbx_ctx *c, const pbx_weight *w, int M, SixArgsHost a) {
  const std::string name = "pbx_head_q6k_" + std::to_string(M) + "_" + (w->K > 2048 ? "long" : std::to_string(six_lanes(w)));
  hipFunction_t f = pbx_kernel_by_name(c, name);
  if (!f) return pbx_fail(c, PBX_ELOAD, "pbx_linear_logprobs: kernel %s missing", name.c_str());
  void *args[] = {&a};
  return pbx_launch_fn(c, f, name.c_str(), dim3(six_groups(c, w)), dim3(256), args, c->stream);
}

// Logits of the piece from v0 on, n entries.
int piece_logits(pbx_ctx *c, const pbx_weight *w, const Plan &p, char *ws, const float *dX, int64_t M, int64_t v0,
                 int64_t n, pbx_weight *rows) {
  *rows = rows_of(*w, v0, n);
  if (six(w, M) && !p.pairs)
    return launch_six(c, rows, (int)M, {rows->qs, rows->d, dX, (int)rows->N, (int)(rows->K / 256), nullptr, nullptr, 0,
                                        nullptr, (float *)(ws + p.z), rows->N});
  const pbx_workspace space{ws + p.gemm, p.z - p.gemm};
  return pbx_linear_enqueue(c, rows, dX, M, nullptr, (float *)(ws + p.z), c->stream, &space);
}

// The rows of X, prepared for pairs; and the piece from v0 on, n entries (and zeros up to
// a multiple of 32), as pairs.
int pairs_rows(pbx_ctx *c, const pbx_weight *w, const Plan &p, char *ws, const float *dX, int64_t M) {
  const pbx_weight v = pairs_of(*w, p.piece, ws + p.halves);
  const pbx_head_rows x = pbx_gemm_head_rows(&v, (int)M, ws + p.gemm);
  const int rc = pbx_gemm_head_prep(c, dX, (int)M, (int)w->K, x.x16, x.x16lo, x.inv);
  if (rc) return rc;
  void *hi = x.x16, *lo = x.x16lo;
  int64_t n16 = (M + 127) / 128 * 128 * w->K / 8;
  void *args[] = {&hi, &lo, &n16};
  return pbx_launch(c, PBX_K_HEAD_TWICE, dim3((unsigned)((n16 + 255) / 256)), dim3(256), args);
}
int pairs_piece(pbx_ctx *c, const pbx_weight *w, const Plan &p, char *ws, int64_t v0, int64_t n, pbx_weight *v,
                pbx_head_epilogue *e) {
  const pbx_weight rows = rows_of(*w, v0, n);
  *v = pairs_of(*w, n, ws + p.halves);
  e->f = (const int32_t *)(ws + p.f);
  e->f_peaks = (const int32_t *)(ws + p.f_peaks);
  int k = (int)w->K, m = (int)n, padded_rows = (int)((n + 31) / 32 * 32);
  e->n_f_peaks = std::min(PAIRS_GROUPS, padded_rows / 4);
  void *args[] = {(void *)&rows.qs, (void *)&rows.d, &k, &m, &padded_rows, &v->qs, &e->f, &e->f_peaks};
  return pbx_launch(c, w->type == PBX_TYPE_F32 ? PBX_K_HEAD_PAIRS_F32 : PBX_K_HEAD_PAIRS_Q6K,
                    dim3((unsigned)e->n_f_peaks), dim3(256), args);
}

}  // namespace

extern "C" int pbx_linear_logprobs_workspace(pbx_ctx *c, const pbx_weight *w, int64_t rows, int grad, size_t *bytes) try {
  const char *who = "pbx_linear_logprobs_workspace";
  if (!c) return pbx_fail(nullptr, PBX_EINVAL, "%s: ctx is NULL", who);
  if (!bytes) return pbx_fail(c, PBX_EINVAL, "%s: NULL argument", who);
  const int rc = check(c, who, w, rows);
  if (!rc) *bytes = rows ? make_plan(c, w, rows, grad != 0).bytes : 0;
  return rc;
} catch (const std::bad_alloc &) {
  return pbx_fail(c, PBX_ENOMEM, "pbx_linear_logprobs_workspace: out of host memory");
}

extern "C" int pbx_linear_logprobs_dev(pbx_ctx *c, const pbx_weight *w, const float *dX, int64_t M,
                                       const int32_t *dTargets, float *dLogp, float *dEntropy, float *dLse, void *work,
                                       size_t work_bytes) try {
  const char *who = "pbx_linear_logprobs_dev";
  if (!c) return pbx_fail(nullptr, PBX_EINVAL, "%s: ctx is NULL", who);
  int rc = check(c, who, w, M);
  if (rc || !M) return rc;
  if (!dX || (uintptr_t)dX % 16) return pbx_fail(c, PBX_EINVAL, "%s: dX needs a 16-byte aligned address", who);
  if (!dTargets != !dLogp) return pbx_fail(c, PBX_EINVAL, "%s: dTargets and dLogp go together", who);
  const Plan p = make_plan(c, w, M, false);
  if ((rc = check_work(c, who, p, work, work_bytes))) return rc;
  char *ws = (char *)work;
  float *z = (float *)(ws + p.z), *hit = (float *)(ws + p.hit);
  void *parts = ws + p.parts;
  int n_parts = p.n_parts, part0 = 0;
  pbx_head_epilogue e;
  e.targets = dTargets;
  e.parts = parts;
  e.n_parts = n_parts;
  e.hit = dLogp ? hit : nullptr;
  e.vocab = (int)w->N;
  if (p.pairs) {
    if ((rc = pairs_rows(c, w, p, ws, dX, M))) return rc;
    for (int64_t v0 = 0; v0 < w->N; v0 += p.piece) {
      pbx_weight v;
      e.v0 = (int)v0;
      e.part0 = (int)(v0 / 128);
      if ((rc = pairs_piece(c, w, p, ws, v0, std::min(p.piece, w->N - v0), &v, &e)) ||
          (rc = pbx_gemm_head(c, &v, (int)M, ws + p.gemm, e)))
        return rc;
    }
  } else if (p.fused) {
    const pbx_head_rows x = pbx_gemm_head_rows(w, (int)M, ws + p.gemm);
    if ((rc = pbx_gemm_head_prep(c, dX, (int)M, (int)w->K, x.x16, x.x16lo, x.inv)) ||
        (rc = pbx_gemm_head(c, w, (int)M, ws + p.gemm, e)))
      return rc;
  }
  const bool alone = six(w, M) && !p.pairs;
  if (alone &&
      (rc = launch_six(c, w, (int)M, {w->qs, w->d, dX, (int)w->N, (int)(w->K / 256), dTargets, parts, n_parts,
                                      dLogp ? hit : nullptr, nullptr, 0})))
    return rc;
  for (int64_t v0 = 0; v0 < w->N && !p.fused && !alone; v0 += p.piece) {
    pbx_weight rows;
    int n = (int)std::min(p.piece, w->N - v0), at = (int)v0;
    if ((rc = piece_logits(c, w, p, ws, dX, M, v0, n, &rows))) return rc;
    const int here = (n + HEAD_SHARE - 1) / HEAD_SHARE;
    int64_t stride = rows.N;
    float *h = dLogp ? hit : nullptr;
    void *args[] = {&z, &stride, &n, &at, (void *)&dTargets, &parts, &n_parts, &part0, &h};
    if ((rc = pbx_launch(c, PBX_K_HEAD_STATS, dim3(here, (unsigned)M), dim3(256), args))) return rc;
    part0 += here;
  }
  int vocab = (int)w->N;
  void *args[] = {&parts, &n_parts, (void *)&dTargets, &vocab, &hit, &dLogp, &dEntropy, &dLse};
  return pbx_launch(c, PBX_K_HEAD_JOIN, dim3((unsigned)M), dim3(256), args);
} catch (const std::bad_alloc &) {
  return pbx_fail(c, PBX_ENOMEM, "pbx_linear_logprobs_dev: out of host memory");
}

extern "C" int pbx_linear_logprobs_grad_dev(pbx_ctx *c, const pbx_weight *w, const float *dX, int64_t M,
                                            const int32_t *dTargets, const float *dLse, const float *dGradLogp,
                                            float *dGradX, void *work, size_t work_bytes) try {
  const char *who = "pbx_linear_logprobs_grad_dev";
  if (!c) return pbx_fail(nullptr, PBX_EINVAL, "%s: ctx is NULL", who);
  int rc = check(c, who, w, M);
  if (rc || !M) return rc;
  if (!dX || !dGradX || (uintptr_t)dX % 16 || (uintptr_t)dGradX % 16)
    return pbx_fail(c, PBX_EINVAL, "%s: dX and dGradX need 16-byte aligned addresses", who);
  if (dGradX == dX) return pbx_fail(c, PBX_EINVAL, "%s: dGradX is dX itself", who);
  if (!dTargets || !dLse || !dGradLogp) return pbx_fail(c, PBX_EINVAL, "%s: NULL argument", who);
  const Plan p = make_plan(c, w, M, true);
  if ((rc = check_work(c, who, p, work, work_bytes))) return rc;
  const bool f32 = w->type == PBX_TYPE_F32 && !p.pairs;
  const char *tag = f32                                  ? "f32"
                    : w->type == PBX_TYPE_F16 || p.pairs ? "f16"
                    : w->type == PBX_TYPE_Q8_0           ? "q8"
                    : w->type == PBX_TYPE_Q4_0           ? "q4"
                    : w->type == PBX_TYPE_Q4_1           ? "q41"
                                                         : "q6k";
  const std::string name = std::string("pbx_head_back_") + tag + "_" + std::to_string(p.TT);
  hipFunction_t back = pbx_kernel_by_name(c, name);
  if (!back) return pbx_fail(c, PBX_ELOAD, "%s: kernel %s missing", who, name.c_str());
  char *ws = (char *)work;
  float *z = (float *)(ws + p.z), *part = (float *)(ws + p.part);
  float *hit = (float *)(ws + p.hit), *others = (float *)(ws + p.others);
  void *peaks = ws + p.peaks;
  pbx_head_scales scales{};
  if (w->d && !p.pairs)
    scales = {w->d, w->Npad * (w->type == PBX_TYPE_Q6_K ? w->K / 256 : w->B) / 8 * (w->m ? 2 : 1), peaks};
  int m = (int)M, k = (int)w->K, vocab = (int)w->N, Mpad = p.Mpad, KS = p.KS, folds = p.pairs ? 2 : 1;
  int n_others = p.n_others;
  const int columns = k * folds;
  if (p.pairs) {
    rc = pairs_rows(c, w, p, ws, dX, M);
  } else if (p.fused) {
    const pbx_head_rows x = pbx_gemm_head_rows(w, m, ws + p.gemm);
    rc = pbx_gemm_head_prep(c, dX, m, k, x.x16, x.x16lo, x.inv, scales);
  }
  if (rc) return rc;
  for (int64_t v0 = 0; v0 < w->N; v0 += p.piece) {
    pbx_weight rows;
    int n = (int)std::min(p.piece, w->N - v0), at = (int)v0;
    if (!p.fused && (rc = piece_logits(c, w, p, ws, dX, M, v0, n, &rows))) return rc;
    const int blocks = (n + 31) / 32;
    int add = v0 > 0;
    int64_t stride = rows.N;
    void *hi = ws + p.g, *lo = ws + p.g + (size_t)blocks * 32 * Mpad * 2;
    pbx_head_epilogue e;
    if (p.fused) {
      e.targets = dTargets;
      e.lse = dLse;
      e.hi = hi;
      e.lo = lo;
      e.Mpad = Mpad;
      e.v0 = at;
      e.vocab = vocab;
      e.hit = hit;
      e.others = others;
      e.n_others = n_others;
      e.add = add;
      if (p.pairs) {
        if ((rc = pairs_piece(c, w, p, ws, v0, n, &rows, &e))) return rc;
      } else {
        rows = rows_of(*w, v0, n);
        rows.N = n;
      }
      rc = pbx_gemm_head(c, &rows, m, ws + p.gemm, e);
    } else if (f32) {
      void *args[] = {&z, &stride, &n, &at, (void *)&dLse, (void *)&dTargets, &vocab, &m, &Mpad, &hi,
                      &hit, &others, &n_others, &add};
      rc = pbx_launch(c, PBX_K_HEAD_G32, dim3(blocks, (Mpad + 63) / 64), dim3(256), args);
    } else {
      int here = blocks;
      void *args[] = {&z, &stride, &n, &at, (void *)&dLse, (void *)&dTargets, &vocab, &m, &Mpad, &hi, &lo,
                      &here, &scales.scales, &scales.n8, &peaks, &hit, &others, &n_others, &add};
      rc = pbx_launch(c, PBX_K_HEAD_G, dim3(blocks + (w->d && !v0 ? PBX_HEAD_PEAKS : 0), (Mpad + 63) / 64), dim3(256), args);
    }
    if (rc) return rc;
    BackArgsHost b{rows.qs, rows.d, rows.m, hi, lo, hi, peaks, e.f_peaks, e.n_f_peaks, part, m, Mpad, columns, (int)rows.B, blocks,
                   (int)rows.Npad, KS, add};
    void *args[] = {&b};
    if ((rc = pbx_launch_fn(c, back, name.c_str(), dim3((columns + 127) / 128, (m + 32 * p.TT - 1) / (32 * p.TT), KS),
                            dim3(f32 ? 64 : 256), args, c->stream)))
      return rc;
  }
  ReduceArgsHost r{part, KS, m, k, folds, dTargets, vocab, dGradLogp, dGradX, hit, others, n_others,
                   pbx_kernel_type(w->type), w->qs, w->d, w->m};
  void *args[] = {&r};
  return pbx_launch(c, PBX_K_HEAD_REDUCE, dim3((k / 4 + 15) / 16, (unsigned)M), dim3(256), args);
} catch (const std::bad_alloc &) {
  return pbx_fail(c, PBX_ENOMEM, "pbx_linear_logprobs_grad_dev: out of host memory");
}
