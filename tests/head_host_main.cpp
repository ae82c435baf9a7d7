// The head's calls (purebee_amd/csrc/runtime/pbx_head.cpp, with pbx_gemm.cpp's plans) without a
// GPU, in a process whose memory runs out: no exception leaves an entry point.
#include "pbx_internal.h"

#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>

#include <new>

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

extern "C" hipError_t hipSetDevice(int) { return hipSuccess; }
int pbx_fail(pbx_ctx *, int code, const char *fmt, ...) {
  if (code != PBX_ENOMEM) printf("%s\n", fmt);
  return code;
}
bool pbx_weight_ok(const pbx_weight *w) { return w; }
size_t pbx_type_row_bytes(int, int64_t K) { return (size_t)K * 4; }
hipFunction_t pbx_kernel_by_name(pbx_ctx *, const std::string &) { return (hipFunction_t)1; }
int pbx_launch(pbx_ctx *, int, dim3, dim3, void **, hipStream_t) { return PBX_OK; }
int pbx_launch_fn(pbx_ctx *, hipFunction_t, const char *, dim3, dim3, void **, hipStream_t) { return PBX_OK; }
int pbx_ensure_dev(pbx_ctx *, void **, size_t *, size_t) { return PBX_OK; }
int pbx_linear_enqueue(pbx_ctx *c, const pbx_weight *w, const float *dX, int64_t M, const float *dBias, float *dY,
                       hipStream_t stream, const pbx_workspace *ws) {
  if (M < PBX_GEMM_MIN_M || w->type == PBX_TYPE_Q6_K) return PBX_OK;
  return pbx_gemm_enqueue(c, w, dX, M, dBias, dY, stream, ws);
}

int main() {
  pbx_ctx c;
  alignas(256) static char some[256];
  float *f = (float *)some;
  int refused = 0, planned = 0;
  for (int type : {PBX_TYPE_Q4_0, PBX_TYPE_Q4_1, PBX_TYPE_Q8_0, PBX_TYPE_Q6_K, PBX_TYPE_F16, PBX_TYPE_F32})
    for (int64_t N : {100, 1000, 20000, 128256})
      for (int64_t M : {1, 3, 8, 40, 300}) {
        pbx_weight w;
        w.type = type, w.N = N, w.K = 2048, w.B = 64, w.Npad = (N + 63) / 64 * 64;
        for (int grad = 0; grad < 2; ++grad)
          for (left = 0; left < 12; ++left) {  // (counted down by the call, and set again)
            const int had = left;
            size_t bytes = 0;
            int rc = pbx_linear_logprobs_workspace(&c, &w, M, grad, &bytes);
            if (rc == PBX_OK) {
              ++planned;
              left = had;
              rc = grad ? pbx_linear_logprobs_grad_dev(&c, &w, f, M, (int32_t *)f, f, f, f + 32, some, bytes)
                        : pbx_linear_logprobs_dev(&c, &w, f, M, (int32_t *)f, f, f, f, some, bytes);
            }
            refused += rc == PBX_ENOMEM;
            if (rc != PBX_OK && rc != PBX_ENOMEM) return printf("rc %d\n", rc), 1;
            left = had;
          }
        left = -1;
      }
  printf("refused %d planned %d\n", refused, planned);
  return 0;
}
