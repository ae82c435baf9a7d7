// pbx_head_peaks.h -- what the head's kernels (pbx_head.hip) and the GEMM's epilogues for it
// (pbx_gemm.hip) share: the largest scale of a quantised head, which its gradient's
// products are scaled by, and the target's place in the gradient's first factor.
#ifndef PBX_HEAD_PEAKS_H
#define PBX_HEAD_PEAKS_H

#include "pbx_gemv_impl.h"

#define HEAD_PEAKS 256  // shares of the plane (pbx_head.cpp, too)

// Share `part` of a plane of halves (n8 groups of 8): its largest magnitude's bits.
// A workgroup of 256 threads.
__device__ __forceinline__ void head_peaks(const uint16_t *plane, int64_t n8, unsigned *peaks, int part) {
  __shared__ unsigned red[4];
  unsigned m = 0;
  for (int64_t i = (int64_t)part * 256 + threadIdx.x; i < n8; i += HEAD_PEAKS * 256) {
    const uint4 v = reinterpret_cast<const uint4 *>(plane)[i];
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) m = max(m, max(w[e] & 0x7fffu, (w[e] >> 16) & 0x7fffu));
  }
#pragma unroll
  for (int off = 32; off >= 1; off /= 2) m = max(m, (unsigned)__shfl_xor((int)m, off, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) peaks[part] = max(max(red[0], red[1]), max(red[2], red[3]));
}

// The largest of n exponents; by every wave for itself.
__device__ __forceinline__ int head_f_peak(const int *peaks, int n) {
  int m = -200;
  for (int i = threadIdx.x & 63; i < n; i += 64) m = max(m, peaks[i]);
#pragma unroll
  for (int off = 32; off >= 1; off /= 2) m = max(m, __shfl_xor(m, off, 64));
  return m;
}

// The target's G from d = l - lse, 1 - e^d.  Where it is likelier than not, lse (rounded to
// 2^-24 of itself, so to 10^-6 of e^lse) leaves little or nothing of 1 - e^d, while the sum of
// the other entries' e^(l - lse), which it stands for, is off by no more than they are:
// there G is 0 here, and pbx_head_reduce adds that sum times the target's weights.
__device__ __forceinline__ bool head_likely(float d) { return d > -0.6931472f; }
__device__ __forceinline__ float head_target_g(float d) { return head_likely(d) ? 0.f : -expm1f(d); }

#endif
