// pbx_head.hip -- log probabilities of rows straight from a head's weights, a piece of
// the vocabulary at a time, and the rows' gradient.
//
// With logits l_v = x . W_v, m = max l, S = sum e^(l - m), T = sum e^(l - m) (l - m):
//   lse = m + log S,  log p_t = l_t - lse,  entropy = log S - T / S,
// where (m, S, T) of parts of the vocabulary join as
//   S = S1 e^(m1 - m) + S2 e^(m2 - m),  T = sum (Ti + (mi - m) Si) e^(mi - m);
// and d log p_t / dx = W_t - sum_v p_v W_v = sum_v G_v W_v with G = (v == t) - e^(l - lse),
// G_t being the sum of the others' e^(l - lse), too.

#include "pbx_head_peaks.h"

using namespace pbx;

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2t __attribute__((ext_vector_type(2)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

// The maximum before any element: finite, so differences need no special case
// (an element of -inf adds nothing; a row of nothing else keeps S == 0).
constexpr float LOWEST = -3.402823466e38f;

struct Sums {
  float m, s, t;
};
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504f); }
// e^d is 0 from -104 on; the bound keeps products with 0 finite
__device__ __forceinline__ float bounded(float d) { return fmaxf(d, -200.f); }
__device__ __forceinline__ Sums moved(Sums a, float m) {  // to the larger maximum m
  const float d = bounded(a.m - m), f = exp_of(d);
  return {m, a.s * f, fmaf(d, a.s, a.t) * f};
}

// The sums of all 256 threads: one maximum first, then each moves once.
__device__ __forceinline__ Sums join_threads(Sums a, float (*buf)[4]) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  float m = wave_max(a.m);
  if (lane == 0) buf[wave][0] = m;
  __syncthreads();
  m = fmaxf(fmaxf(buf[0][0], buf[1][0]), fmaxf(buf[2][0], buf[3][0]));
  a = moved(a, m);
  const float s = wave_sum(a.s), t = wave_sum(a.t);
  if (lane == 0) {
    buf[wave][1] = s;
    buf[wave][2] = t;
  }
  __syncthreads();
  return {m, buf[0][1] + buf[1][1] + buf[2][1] + buf[3][1], buf[0][2] + buf[1][2] + buf[2][2] + buf[3][2]};
}

}  // namespace

#define HEAD_SHARE 8192  // logits of a workgroup of pbx_head_stats

// Sums of a piece's logits Z [M][stride] (n of a row count; it starts at vocabulary
// entry v0): workgroup (part of 8192, row) -> parts[row][part0 + part], and the targets'
// logits.  One pass, a running maximum a thread; heads whose products the GEMM's epilogue
// does not take (there the logits are never written).
extern "C" __global__ void __launch_bounds__(256)
pbx_head_stats(const float *Z, int64_t stride, int n, int v0, const int *targets, float4 *parts, int n_parts,
               int part0, float *hit) {
  __shared__ float buf[4][4];
  const int64_t row = blockIdx.y;
  const float *z = Z + row * stride;
  const int at = blockIdx.x * HEAD_SHARE;
  float4 x[HEAD_SHARE / 1024];
  Sums a{LOWEST, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < HEAD_SHARE / 1024; ++i) {
    const int v = at + 4 * (int)threadIdx.x + 1024 * i;
    x[i] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    if (v < n) {
      x[i] = *reinterpret_cast<const float4 *>(z + v);
      if (v + 1 >= n) x[i].y = -INFINITY;
      if (v + 2 >= n) x[i].z = -INFINITY;
      if (v + 3 >= n) x[i].w = -INFINITY;
    }
    a.m = fmaxf(fmaxf(fmaxf(a.m, x[i].x), fmaxf(x[i].y, x[i].z)), x[i].w);
  }
#pragma unroll
  for (int i = 0; i < HEAD_SHARE / 1024; ++i) {
    const float v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float d = bounded(v[e] - a.m), f = exp_of(d);
      // (the bound hides a NaN: a NaN logit has to reach the sum)
      a.s += v[e] != v[e] ? v[e] : f;
      a.t = fmaf(d, f, a.t);
    }
  }
  a = join_threads(a, buf);
  if (threadIdx.x == 0) {
    parts[row * n_parts + part0 + blockIdx.x] = make_float4(a.m, a.s, a.t, 0.f);
    if (blockIdx.x == 0 && hit) {
      const int64_t t = (int64_t)targets[row] - v0;
      if (t >= 0 && t < n) hit[row] = z[t];
    }
  }
}

// A row's parts joined: workgroup = row.  1,000 rows of 1,002 parts 6.5 us.
extern "C" __global__ void __launch_bounds__(256)
pbx_head_join(const float4 *parts, int n_parts, const int *targets, int vocab, const float *hit, float *logp,
              float *entropy, float *lse) {
  __shared__ float buf[4][4];
  const int64_t row = blockIdx.x;
  Sums a{LOWEST, 0.f, 0.f};
  for (int i = threadIdx.x; i < n_parts; i += 256) {
    const float4 p = parts[row * n_parts + i];
    const float m = fmaxf(a.m, p.x);
    const Sums u = moved(a, m), w = moved({p.x, p.y, p.z}, m);
    a = {m, u.s + w.s, u.t + w.t};
  }
  a = join_threads(a, buf);
  if (threadIdx.x) return;
  const float none = __uint_as_float(0x7fc00000u);
  const bool ok = a.s > 0.f && a.s < INFINITY && a.m < INFINITY;
  const float log_s = logf(a.s), all = a.m + log_s;
  if (lse) lse[row] = ok ? all : none;
  if (entropy) entropy[row] = ok ? log_s - a.t / a.s : none;
  if (logp) {
    const int t = targets[row];
    // x_t - m first: it is exact where the target is the likeliest
    logp[row] = ok && t >= 0 && t < vocab ? hit[row] - a.m - log_s : none;
  }
}

// ---- one to three rows of a Q6_K head ------------------------------------------------

namespace {

// The value of the lane that differs in bit OFF, by moves that need no trip through LDS.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), CTRL, 0xf, 0xf, false));
}
template <int OFF>
__device__ __forceinline__ float partner(float v, int lane) {
  if constexpr (OFF == 1) return dpp<0xB1>(v);              // quad_perm 1 0 3 2
  else if constexpr (OFF == 2) return dpp<0x4E>(v);         // quad_perm 2 3 0 1
  else if constexpr (OFF == 4) return dpp<0x1B>(dpp<0x141>(v));  // row_half_mirror, quad_perm 3 2 1 0
  else if constexpr (OFF == 8) return dpp<0x128>(v);        // row_ror 8
  else {
    const unsigned u = __float_as_uint(v);
    const auto r = OFF == 16 ? __builtin_amdgcn_permlane16_swap(u, u, false, false)
                             : __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(lane & OFF ? r[0] : r[1]);
  }
}

struct SixArgs {
  const uint8_t *qs;
  const uint16_t *dsc;
  const float *X;  // [M][K]
  int N, SB;
  // the answer's sums [M][n_parts] (a part is a workgroup) and the targets' logits, or (Z)
  // the logits [M][stride]
  const int *targets;
  float4 *parts;
  int n_parts;
  float *hit, *Z;
  int64_t stride;
};

// Logits of M rows.  A lane takes 16 bytes of low nibbles:
// the 16 codes of one 32-code group of half a superblock and the 16 of the group two
// further on, whose high bits lie in 16 bytes that it shares with one other lane; eight lanes a
// superblock, so a row of 2,048 is one wave's (of the plain GEMV a lane takes a 32-code
// block, 64 bytes for 24 of its own: 128,256 x 2,048 70 us).  A step is four rows
// (whose superblock scales are one load) for each group of LANES lanes, the next step's
// in flight; the lanes' sums of four rows are added in 7 steps instead of 24, halving what
// each lane holds.
// Up to 2,048 columns (one pass of the lanes) the lane keeps its activations as integers
// of up to 8,355,711 in three signed bytes (0.5 / 2^22 of the largest of its 32 is what they
// may be off), so that v_dot4 sums four products with codes exactly; 32 times the bytes'
// sums, for codes less 32, is taken off as an integer (128,256 x 2,048: 49 us, 4.4 TB/s; 56 us with
// f32 products, 207 vector instructions a row, 43 us of them).  Longer rows: f32, 128,256 x 4,096
// 122 us with the join, where the head's bytes take 84 at a copy's rate; integers would be made anew
// for each pass of the lanes.
template <int M, int LANES, bool WHOLE>
__device__ __forceinline__ void six_body(const SixArgs &a) {
  constexpr int SLOTS = 64 / LANES;
  __shared__ float buf[4][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int slot = lane / LANES, sb0 = lane % LANES / 8, c = lane & 3, half = lane >> 2 & 1;
  const int step = (int)gridDim.x * 4 * SLOTS, groups = (a.N + 3) / 4;
  const int its = WHOLE ? 1 : (a.SB + LANES / 8 - 1) / (LANES / 8);
  struct Raw {
    uint4 l[4], h[4];
    uint2 sc[4], d;
  };
  // (a slot or superblock past the end reads the last one, and adds nothing)
  auto load = [&](int g, int it, Raw &q) {
    const int n = 4 * min(g, groups - 1), sb = min(sb0 + it * (LANES / 8), a.SB - 1);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint8_t *blk = a.qs + ((int64_t)(n + r) * a.SB + sb) * PBX_Q6K_BYTES;
      q.l[r] = ld_stream(blk + 64 * half + 16 * c);
      q.h[r] = ld_stream(blk + 128 + 32 * half + 16 * (c & 1));
      q.sc[r] = *reinterpret_cast<const uint2 *>(blk + 192 + 8 * half);
    }
    q.d = *reinterpret_cast<const uint2 *>(a.dsc + dsc_index(n, sb, a.SB));
  };
  float x[M][WHOLE ? 1 : 32];
  // [byte 0 .. 2 of an activation][group][4 activations each dword], and 32 times their sums
  int limb[M][3][8], offset[M][2][3];
  float unit[M];
  auto split_x = [&]() {
#pragma unroll
    for (int m = 0; m < M; ++m) {
      float v[32], most = 0.f;
      bool odd = false;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float4 t = sb0 < a.SB ? *reinterpret_cast<const float4 *>(a.X + ((int64_t)m * a.SB + sb0) * 256 + 128 * half +
                                                                        16 * c + 64 * (j >> 2) + 4 * (j & 3))
                                    : make_float4(0.f, 0.f, 0.f, 0.f);
        v[4 * j] = t.x, v[4 * j + 1] = t.y, v[4 * j + 2] = t.z, v[4 * j + 3] = t.w;
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        most = fmaxf(most, fabsf(v[j]));
        odd = odd || !(fabsf(v[j]) < INFINITY);
      }
      int e = 0;
      if (most > 0.f && most < INFINITY) frexpf(most, &e);
      e = max(e, -100);
      float up = ldexpf(1.f, 23 - e);
      if (most * up > 8355711.f) up *= 0.5f;
      // a row with a NaN or an infinity has no logits
      unit[m] = __ballot(odd) ? __uint_as_float(0x7fc00000u) : 1.f / up;
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int l = 0; l < 3; ++l) offset[m][g][l] = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        unsigned w[3] = {0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int q = (int)rintf(fminf(fmaxf(v[4 * j + i] * up, -8355711.f), 8355711.f));
          const int q0 = (int)(int8_t)q, q1 = (int)(int8_t)((q - q0) >> 8), q2 = (q - q0 - 256 * q1) >> 16;
          w[0] |= (unsigned)(q0 & 255) << (8 * i);
          w[1] |= (unsigned)(q1 & 255) << (8 * i);
          w[2] |= (unsigned)(q2 & 255) << (8 * i);
          offset[m][j >> 2][0] += 32 * q0;
          offset[m][j >> 2][1] += 32 * q1;
          offset[m][j >> 2][2] += 32 * q2;
        }
#pragma unroll
        for (int l = 0; l < 3; ++l) limb[m][l][j] = (int)w[l];
      }
    }
  };
  auto load_x = [&](int it) {
    const int sb = sb0 + it * (LANES / 8);
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float4 v = sb < a.SB ? *reinterpret_cast<const float4 *>(a.X + ((int64_t)m * a.SB + sb) * 256 + 128 * half +
                                                                       16 * c + 64 * (j >> 2) + 4 * (j & 3))
                                   : make_float4(0.f, 0.f, 0.f, 0.f);
        if constexpr (!WHOLE) x[m][4 * j] = v.x, x[m][4 * j + 1] = v.y, x[m][4 * j + 2] = v.z, x[m][4 * j + 3] = v.w;
      }
  };
  float z[M][4];
  auto add = [&](const Raw &q) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float d = f16_bits_to_f32((r & 2 ? q.d.y : q.d.x) >> (16 * (r & 1)));
      const float d0 = d * (float)(int8_t)(q.sc[r].x >> (8 * c)), d1 = d * (float)(int8_t)(q.sc[r].y >> (8 * c));
      const unsigned l[4] = {q.l[r].x, q.l[r].y, q.l[r].z, q.l[r].w}, h[4] = {q.h[r].x, q.h[r].y, q.h[r].z, q.h[r].w};
      if constexpr (WHOLE) {
        int t[M][2][3];
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int k = 0; k < 3; ++k) t[m][g][k] = -offset[m][g][k];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const unsigned hi = h[j] >> (c & 2);  // groups 0, 2 or 1, 3
          const int q0 = (int)((l[j] & 0x0F0F0F0Fu) | (hi << 4 & 0x30303030u));
          const int q1 = (int)((l[j] >> 4 & 0x0F0F0F0Fu) | (hi & 0x30303030u));
#pragma unroll
          for (int m = 0; m < M; ++m)
#pragma unroll
            for (int k = 0; k < 3; ++k) {
              t[m][0][k] = __builtin_amdgcn_sdot4(limb[m][k][j], q0, t[m][0][k], false);
              t[m][1][k] = __builtin_amdgcn_sdot4(limb[m][k][4 + j], q1, t[m][1][k], false);
            }
        }
#pragma unroll
        for (int m = 0; m < M; ++m) {
          const float s0 = fmaf((float)t[m][0][2], 65536.f, fmaf((float)t[m][0][1], 256.f, (float)t[m][0][0]));
          const float s1 = fmaf((float)t[m][1][2], 65536.f, fmaf((float)t[m][1][1], 256.f, (float)t[m][1][0]));
          z[m][r] = unit[m] * fmaf(d0, s0, d1 * s1);
        }
        continue;
      }
      float s0[M], s1[M];
#pragma unroll
      for (int m = 0; m < M; ++m) s0[m] = s1[m] = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned hi = h[j] >> (c & 2);  // groups 0, 2 or 1, 3
        const unsigned q0 = (l[j] & 0x0F0F0F0Fu) | (hi << 4 & 0x30303030u);
        const unsigned q1 = (l[j] >> 4 & 0x0F0F0F0Fu) | (hi & 0x30303030u);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float c0 = (float)(q0 >> (8 * e) & 255u) - 32.f, c1 = (float)(q1 >> (8 * e) & 255u) - 32.f;
#pragma unroll
          for (int m = 0; m < M; ++m) {
            s0[m] = fmaf(x[m][WHOLE ? 0 : 4 * j + e], c0, s0[m]);
            s1[m] = fmaf(x[m][WHOLE ? 0 : 16 + 4 * j + e], c1, s1[m]);
          }
        }
      }
#pragma unroll
      for (int m = 0; m < M; ++m) z[m][r] = fmaf(d0, s0[m], fmaf(d1, s1[m], z[m][r]));
    }
  };
  Sums sum[M];
#pragma unroll
  for (int m = 0; m < M; ++m) sum[m] = {LOWEST, 0.f, 0.f};
  const int first = ((int)blockIdx.x * 4 + wave) * SLOTS + slot;
  // every lane of a wave runs as many steps as its first slot
  const int g0 = ((int)blockIdx.x * 4 + wave) * SLOTS;
  Raw q, next;
  load(first, 0, q);
  if constexpr (WHOLE) split_x();
  for (int g = first, w = g0; w < groups; g += step, w += step) {
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) z[m][r] = 0.f;
    for (int it = 0; it < its; ++it) {
      if constexpr (!WHOLE) load_x(it);
      const bool more = it + 1 < its;
      load(more ? g : g + step, more ? it + 1 : 0, next);
      add(q);
      q = next;
    }
    // row r of the four is left in the lanes whose bits 0 and 1 are r
    const int r = lane & 3, n = 4 * g + r;
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const bool b0 = lane & 1, b1 = lane & 2;
      float u = (b0 ? z[m][1] : z[m][0]) + partner<1>(b0 ? z[m][0] : z[m][1], lane);
      const float v = (b0 ? z[m][3] : z[m][2]) + partner<1>(b0 ? z[m][2] : z[m][3], lane);
      u = (b1 ? v : u) + partner<2>(b1 ? u : v, lane);
      u += partner<4>(u, lane);
      if constexpr (LANES > 8) u += partner<8>(u, lane);
      if constexpr (LANES > 16) u += partner<16>(u, lane);
      if constexpr (LANES > 32) u += partner<32>(u, lane);
      if (n < a.N && g < groups) {
        if (a.Z) {
          if (lane % LANES < 4) a.Z[m * a.stride + n] = u;
        } else {
          const float top = fmaxf(sum[m].m, u);
          sum[m] = moved(sum[m], top);
          const float d = bounded(u - top), f = exp_of(d);
          sum[m].s += u != u ? u : f;
          sum[m].t = fmaf(d, f, sum[m].t);
          if (a.hit && lane % LANES < 4 && a.targets[m] == n) a.hit[m] = u;
        }
      }
    }
  }
  if (a.Z) return;
#pragma unroll
  for (int m = 0; m < M; ++m) {
    if (lane % LANES >= 4) sum[m] = {LOWEST, 0.f, 0.f};  // the same rows again
    const Sums all = join_threads(sum[m], buf);
    if (threadIdx.x == 0) a.parts[(int64_t)m * a.n_parts + blockIdx.x] = make_float4(all.m, all.s, all.t, 0.f);
    __syncthreads();
  }
}

}  // namespace

#define HEAD_SIX_KERNEL(M, TAG, LANES, WHOLE)                                                                        \
  extern "C" __global__ void __launch_bounds__(256) pbx_head_q6k_##M##_##TAG(SixArgs a) { six_body<M, LANES, WHOLE>(a); }
#define HEAD_SIX(M)                  \
  HEAD_SIX_KERNEL(M, 8, 8, true)     \
  HEAD_SIX_KERNEL(M, 16, 16, true)   \
  HEAD_SIX_KERNEL(M, 32, 32, true)   \
  HEAD_SIX_KERNEL(M, 64, 64, true)   \
  HEAD_SIX_KERNEL(M, long, 64, false)
HEAD_SIX(1)
HEAD_SIX(2)
HEAD_SIX(3)

// ---- F32 and Q6_K heads as pairs of halves --------------------------------------------

namespace {

// Row n of a piece as halves [hi of K | lo of K], scaled by 2^-f[n] so that its largest
// magnitude (Q6_K: what its scales allow) is below 2^15.  A wave's row; returns its f.
// Rows past the piece's last one are zeros.
template <int TYPE>
__device__ __forceinline__ int pairs_row(const uint8_t *qs, const uint16_t *dsc, int K, int n, _Float16 *out, int *f,
                                         int row) {
  typedef _Float16 half4t __attribute__((ext_vector_type(4)));
  const int lane = threadIdx.x & 63;
  _Float16 *hi = out + (int64_t)row * 2 * K, *lo = hi + K;
  if (row >= n) {
    for (int k = 8 * lane; k < K; k += 512) {
      *reinterpret_cast<half8 *>(hi + k) = half8{};
      *reinterpret_cast<half8 *>(lo + k) = half8{};
    }
    if (lane == 0) f[row] = -200;
    return -200;
  }
  const float4 *w4 = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(qs) + (int64_t)row * K);
  const int SB = K >> 8;
  const uint8_t *six = qs + (int64_t)row * SB * PBX_Q6K_BYTES;
  float most = 0.f;
  if constexpr (TYPE == PBX_F32) {
    for (int k = lane; k < K / 4; k += 64) {
      const float4 v = w4[k];
      most = fmaxf(most, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
    }
  } else {
    for (int i = lane; i < SB * 16; i += 64) {
      const float d = f16_bits_to_f32(dsc[dsc_index(row, i >> 4, SB)]);
      most = fmaxf(most, fabsf(d * (float)(int8_t)six[(int64_t)(i >> 4) * PBX_Q6K_BYTES + 192 + (i & 15)]) * 32.f);
    }
  }
  most = wave_max(most);
  int e = -185;
  if (most > 0.f && most < INFINITY) frexpf(most, &e);
  e = max(e, -110);  // (2^(15 - e) stays a normal number)
  const float up = __uint_as_float((unsigned)(15 - e + 127) << 23);
  if (lane == 0) f[row] = e - 15;
  auto split = [&](float v, _Float16 &h, _Float16 &l) {
    h = (_Float16)v;
    l = (_Float16)(v - (float)h);
  };
  if constexpr (TYPE == PBX_F32) {
    for (int k = lane; k < K / 4; k += 64) {
      const float4 v = w4[k];
      half4t h, l;
      _Float16 a, b;
      split(v.x * up, a, b), h[0] = a, l[0] = b;
      split(v.y * up, a, b), h[1] = a, l[1] = b;
      split(v.z * up, a, b), h[2] = a, l[2] = b;
      split(v.w * up, a, b), h[3] = a, l[3] = b;
      reinterpret_cast<half4t *>(hi)[k] = h;
      reinterpret_cast<half4t *>(lo)[k] = l;
    }
  } else {
    // eight lanes a superblock, as in six_body
    for (int i = lane; i < SB * 8; i += 64) {
      const int sb = i >> 3, half = i >> 2 & 1, c = i & 3;
      const uint8_t *blk = six + (int64_t)sb * PBX_Q6K_BYTES;
      const uint4 l4 = ld_stream(blk + 64 * half + 16 * c), h4 = ld_stream(blk + 128 + 32 * half + 16 * (c & 1));
      const float d = f16_bits_to_f32(dsc[dsc_index(row, sb, SB)]) * up;
      const float d0 = d * (float)(int8_t)blk[192 + 8 * half + c], d1 = d * (float)(int8_t)blk[196 + 8 * half + c];
      const unsigned ql[4] = {l4.x, l4.y, l4.z, l4.w}, qh[4] = {h4.x, h4.y, h4.z, h4.w};
      const int64_t at = 256 * sb + 128 * half + 16 * c;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          half8 h, l;
#pragma unroll
          for (int t = 0; t < 8; ++t) {
            const unsigned x = ql[j + (t >> 2)] >> (4 * g), y = qh[j + (t >> 2)] >> ((c & 2) + 4 * g);
            const int code = (int)((x >> (8 * (t & 3)) & 15u) | (y >> (8 * (t & 3)) & 3u) << 4) - 32;
            _Float16 a, b;
            split((g ? d1 : d0) * (float)code, a, b);
            h[t] = a;
            l[t] = b;
          }
          *reinterpret_cast<half8 *>(hi + at + 64 * g + 4 * j) = h;
          *reinterpret_cast<half8 *>(lo + at + 64 * g + 4 * j) = l;
        }
      }
    }
  }
  return e - 15;
}

// All rows, `rows` with those past the last one, a wave each in turn; peaks[workgroup]:
// the largest f of its rows.  Bound by bytes, 4 written for every value: 20,000 x 2,048
// F32 60 us, Q6_K 40.
template <int TYPE>
__device__ __forceinline__ void pairs_body(const uint8_t *qs, const uint16_t *dsc, int K, int n, int rows, _Float16 *out,
                                           int *f, int *peaks) {
  __shared__ int most[4];
  const int wave = threadIdx.x >> 6;
  int top = -200;
  for (int row = blockIdx.x * 4 + wave; row < rows; row += gridDim.x * 4)
    top = max(top, pairs_row<TYPE>(qs, dsc, K, n, out, f, row));
  if ((threadIdx.x & 63) == 0) most[wave] = top;
  __syncthreads();
  if (threadIdx.x == 0) peaks[blockIdx.x] = max(max(most[0], most[1]), max(most[2], most[3]));
}

}  // namespace

extern "C" __global__ void __launch_bounds__(256)
pbx_head_pairs_f32(const uint8_t *qs, const uint16_t *dsc, int K, int n, int rows, _Float16 *out, int *f, int *peaks) {
  pairs_body<PBX_F32>(qs, dsc, K, n, rows, out, f, peaks);
}
extern "C" __global__ void __launch_bounds__(256)
pbx_head_pairs_q6k(const uint8_t *qs, const uint16_t *dsc, int K, int n, int rows, _Float16 *out, int *f, int *peaks) {
  pairs_body<PBX_Q6K>(qs, dsc, K, n, rows, out, f, peaks);
}

// The other factor: the prepared rows' hi plane again and zeros beside it (n16 times 16
// bytes of each), for the products with the low halves.
extern "C" __global__ void __launch_bounds__(256)
pbx_head_twice(uint4 *hi, uint4 *lo, int64_t n16) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n16) return;
  hi[n16 + i] = hi[i];
  lo[n16 + i] = make_uint4(0, 0, 0, 0);
}

// ---- the gradient --------------------------------------------------------------------


namespace {

// The power of two that weights enter the products with: the largest scale (or Q4_1
// minimum) comes to just below 2^TARGET, or less: 2^21 times it, as 2^(21 + 9) is two
// halves' product (back_body).
__device__ __forceinline__ int head_shift(const unsigned *peaks, int target) {
  unsigned m = 0;
  for (int i = threadIdx.x & 63; i < HEAD_PEAKS; i += 64) m = max(m, peaks[i]);
#pragma unroll
  for (int off = 32; off >= 1; off /= 2) m = max(m, (unsigned)__shfl_xor((int)m, off, 64));
  int e = 0;
  if (m) frexpf(f16_bits_to_f32(m), &e);  // 2^(e - 1) <= it < 2^e
  if (m >= 0x7c00u) e = 16;
  return __builtin_amdgcn_readfirstlane(min(target - e, 21));
}
template <int TYPE> struct HeadTarget { static constexpr int value = TYPE == PBX_Q8 ? -5 : TYPE == PBX_Q6K ? -10 : TYPE == PBX_Q41 ? -2 : -1; };

}  // namespace

// G of a piece as fp16 pairs times 2^15, [n / 32][Mpad][32]: workgroup (block of 32
// vocabulary entries, 64 rows); zeros past the vocabulary, the rows, and in rows
// without a target; and each row's others [M][n_others], by block of a piece (add: to those
// of the pieces before), and hit, the target's logit less lse.  Workgroups past the blocks
// (HEAD_PEAKS of them where there are any) look for the head's largest scales.  Few rows, where
// the GEMM's epilogue does not take the head: a pass over the piece's logits, bound by bytes.
extern "C" __global__ void __launch_bounds__(256)
pbx_head_g(const float *Z, int64_t stride, int n, int v0, const float *lse, const int *targets, int vocab, int M,
           int Mpad, _Float16 *hi, _Float16 *lo, int blocks, const uint16_t *scales, int64_t n8, unsigned *peaks,
           float *hit, float *others, int n_others, int add) {
  if ((int)blockIdx.x >= blocks) {
    if (blockIdx.y == 0) head_peaks(scales, n8, peaks, blockIdx.x - blocks);
    return;
  }
  const int row = blockIdx.y * 64 + threadIdx.x / 4, v = blockIdx.x * 32 + 8 * (threadIdx.x % 4);
  if (row >= Mpad) return;
  half8 H = {}, L = {};
  const int t = row < M ? targets[row] : -1;
  float sum = 0.f;
  if (t >= 0 && t < vocab) {
    const float *z = Z + (int64_t)row * stride;
    const float s = lse[row];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (v + e >= n) continue;
      const float d = z[v + e] - s;
      float g = -expf(d);
      if (v0 + v + e == t) {
        g = head_target_g(d);
        hit[row] = d;
      } else {
        sum -= g;
      }
      g *= 32768.f;
      H[e] = (_Float16)g;
      L[e] = (_Float16)(g - (float)H[e]);
    }
  }
  const int64_t at = ((int64_t)blockIdx.x * Mpad + row) * 32 + 8 * (threadIdx.x % 4);
  *reinterpret_cast<half8 *>(hi + at) = H;
  *reinterpret_cast<half8 *>(lo + at) = L;
  sum += __shfl_xor(sum, 1);
  sum += __shfl_xor(sum, 2);
  if (threadIdx.x % 4 == 0 && row < M) {
    float *p = others + (int64_t)row * n_others + blockIdx.x;
    *p = add ? *p + sum : sum;
  }
}

// The same in f32 for an F32 head: [n][Mpad].
extern "C" __global__ void __launch_bounds__(256)
pbx_head_g32(const float *Z, int64_t stride, int n, int v0, const float *lse, const int *targets, int vocab, int M,
             int Mpad, float *G, float *hit, float *others, int n_others, int add) {
  __shared__ float sums[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = blockIdx.y * 64 + lane, v = blockIdx.x * 32 + 8 * wave;
  const int t = row < M ? targets[row] : -1;
  const bool on = t >= 0 && t < vocab;
  const float s = on ? lse[row] : 0.f;
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float g = 0.f;
    if (on && v + e < n) {
      const float d = Z[(int64_t)row * stride + v + e] - s;
      g = -expf(d);
      if (v0 + v + e == t) {
        g = head_target_g(d);
        hit[row] = d;
      } else {
        sum -= g;
      }
    }
    if (row < Mpad) G[(int64_t)(v + e) * Mpad + row] = g;
  }
  sums[wave][lane] = sum;
  __syncthreads();
  if (wave || row >= M) return;
  sum = sums[0][lane] + sums[1][lane] + sums[2][lane] + sums[3][lane];
  float *p = others + (int64_t)row * n_others + blockIdx.x;
  *p = add ? *p + sum : sum;
}

struct BackArgs {
  const uint8_t *qs;   // planes from the piece's first row on
  const uint16_t *dsc, *msc;
  const _Float16 *hi, *lo;  // G
  const float *G32;
  const unsigned *peaks;
  const int *f_peaks;  // F16 as pairs: the largest f of parts of the piece (the products are 2^(-15 - f) of theirs)
  int n_f_peaks;
  float *part;         // [KS][M][K]
  int M, Mpad, K, B;   // B: 32-wide blocks of a row
  int blocks, rows;    // blocks of 32 entries of the piece, and weight rows that may be read
  int KS, add;         // add: to the partial sums of the pieces before
};

namespace {

// 2^e, -126 <= e <= 127.
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }
__device__ __forceinline__ half2t as_half2(unsigned x) { return __builtin_bit_cast(half2t, x); }
// Byte i of x and of y, as two halves u * 2^-24 (the bits of a half of exponent 0).
__device__ __forceinline__ unsigned byte_pair(unsigned x, unsigned y, int i) {
  return __builtin_amdgcn_perm(y, x, 0x0c000c00u | (unsigned)i | (unsigned)(4 + i) << 16);
}

// Column of the wave's 128 that lane lr's tile i holds.
template <int TYPE>
__device__ __forceinline__ int column_of(int lr, int i) {
  if constexpr (TYPE == PBX_Q4 || TYPE == PBX_Q41) return 32 * (lr >> 3) + 16 * (i >> 1) + 2 * (lr & 7) + (i & 1);
  if constexpr (TYPE == PBX_Q6K) return 32 * i + lr;
  return 4 * lr + i;
}

// What 16 entries' part of a wave's operands is made of, as loaded.
template <int TYPE, int TT>
struct BackRaw {
  static constexpr int NW = TYPE == PBX_F16 ? 16 : TYPE == PBX_Q6K ? 24 : 8;
  unsigned w[NW];
  uint2 d[TYPE == PBX_Q6K ? 8 : 2], mn[TYPE == PBX_Q41 ? 2 : 1];
  unsigned ds[TYPE == PBX_Q6K ? 8 : 1];
  half8 Ah[TT], Al[TT];
};

// Steps whose loads are under way: four where the registers allow it (few rows, which
// wait for memory: 5 rows of 49,152 x 576 Q4_0 17 us), else two.
#define BACK_DEPTH(TYPE, TT) ((TYPE) == PBX_Q6K || (TT) == 2 ? 2 : 4)

// Workgroup = 32 TT rows of G, 128 columns of the head and a share of its entries, whose
// blocks four waves take in turn; their sums meet in LDS.  A step is 16 entries: a lane
// loads 4 columns (as they lie in a row's bytes) of 8 rows, so that the operands, 8
// entries of a column, are put together in registers, byte by byte with no trip through
// LDS, while the next step's loads are under way.  Codes times scales are pairs of fp16
// (three products with G's pair; F16 weights two).  Many rows are bound by the matrix
// instructions: 512 rows of 32,768 x 2,048 Q8_0 205 us (1,000 TFLOP/s of products), 37
// rows of 32,003 x 2,048 F16 37 us.  Splitting over the entries, and joining, instead of
// more rows a workgroup: a head has few columns, and G is small beside it.
template <int TYPE, int TT>
__device__ __forceinline__ void back_body(const BackArgs &a) {
  __shared__ float red[2][TT * 4 * 16 * 64];
  const int lane = threadIdx.x & 63, lr = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int k0 = blockIdx.x * 128, m0 = blockIdx.y * (32 * TT);
  // (fewer than 2^14 blocks and 2^12 shares)
  const int b0 = (int)((unsigned)a.blocks * blockIdx.z / (unsigned)a.KS);
  const int b1 = (int)((unsigned)a.blocks * (blockIdx.z + 1) / (unsigned)a.KS);
  constexpr bool NIB = TYPE == PBX_Q4 || TYPE == PBX_Q41;
  const floatx16 zero = {};
  floatx16 acc[TT][4];
#pragma unroll
  for (int t = 0; t < TT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[t][i] = zero;
  // past the row's end columns repeat the last ones (and are not stored)
  const int kc = min(k0 + 4 * lr, a.K - 4), kb = min((k0 >> 5) + (lr >> 3), a.B - 1);
  const int SB = a.B >> 3, sb = min(k0 >> 8, SB - 1), hf = (k0 >> 7) & 1;
  // a row's bytes, and the lane's first byte in the rows 8 h on
  const unsigned row = TYPE == PBX_F16   ? a.K * 2
                       : TYPE == PBX_Q8  ? a.K
                       : TYPE == PBX_Q6K ? SB * PBX_Q6K_BYTES
                                         : a.B * 16;
  const unsigned woff = 8 * h * row + (TYPE == PBX_F16   ? 2 * kc
                                       : TYPE == PBX_Q8  ? kc
                                       : TYPE == PBX_Q6K ? sb * PBX_Q6K_BYTES + 64 * hf
                                                         : kb * 16 + 2 * (lr & 7));
  const unsigned srow = 8 * (TYPE == PBX_Q6K ? SB : a.B);  // bytes of the scales of four rows
  const unsigned doff = 2 * h * srow + (TYPE == PBX_Q6K ? sb : kb) * 8;
  const unsigned aoff = (m0 + lr) * 64 + 16 * h, astep = a.Mpad * 64;
  // Buffers from the share's first block on: a load's address is a buffer's, a scalar
  // and a lane's offset, with no vector arithmetic; the host sees to it that a share is
  // under 2 GB.  The rows of a piece reach past its last block (they are padded to 64),
  // so no step reads beyond them.
  const int64_t shared_rows = (int64_t)(b1 - b0) * 32;
  auto buffer = [](const void *p, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, (int)bytes, 0x00020000);
  };
  const auto wbuf = buffer(a.qs + (int64_t)b0 * 32 * row, shared_rows * row);
  const auto dbuf = buffer(TYPE == PBX_F16 ? (const uint8_t *)a.hi : reinterpret_cast<const uint8_t *>(a.dsc) + (int64_t)b0 * 8 * srow,
                           TYPE == PBX_F16 ? 0 : shared_rows / 4 * srow);
  const auto mbuf = buffer(TYPE == PBX_Q41 ? reinterpret_cast<const uint8_t *>(a.msc) + (int64_t)b0 * 8 * srow : (const uint8_t *)a.hi,
                           TYPE == PBX_Q41 ? shared_rows / 4 * srow : 0);
  const auto hbuf = buffer(reinterpret_cast<const uint8_t *>(a.hi) + (int64_t)b0 * astep, (int64_t)(b1 - b0) * astep);
  const auto lbuf = buffer(reinterpret_cast<const uint8_t *>(a.lo) + (int64_t)b0 * astep, (int64_t)(b1 - b0) * astep);
  auto load = [&](int step, BackRaw<TYPE, TT> &q) {  // (step: from the share's first block on)
    const unsigned w = step * 16 * row, d = step * 4 * srow;
    if constexpr (TYPE == PBX_Q6K) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const unsigned s = w + e * row;
        q.w[3 * e] = __builtin_amdgcn_raw_buffer_load_b8(wbuf, woff + lr, s, 0);
        q.w[3 * e + 1] = __builtin_amdgcn_raw_buffer_load_b8(wbuf, woff + lr + 32, s, 0);
        q.w[3 * e + 2] = __builtin_amdgcn_raw_buffer_load_b8(wbuf, woff + lr + 128 - 32 * hf, s, 0);
        q.d[e] = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(wbuf, woff + 192 - 56 * hf, s, 0));
        q.ds[e] = __builtin_amdgcn_raw_buffer_load_b16(dbuf, doff + 2 * (e & 3), d + (e >> 2) * srow, 0);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const unsigned s = w + e * row;
        if constexpr (TYPE == PBX_F16) {
          const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(wbuf, woff, s, 0));
          q.w[2 * e] = x.x;
          q.w[2 * e + 1] = x.y;
        } else if constexpr (NIB) {
          q.w[e] = __builtin_amdgcn_raw_buffer_load_b16(wbuf, woff, s, 0);
        } else {
          q.w[e] = __builtin_amdgcn_raw_buffer_load_b32(wbuf, woff, s, 0);
        }
      }
      if constexpr (TYPE != PBX_F16) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          q.d[g] = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(dbuf, doff, d + g * srow, 0));
          if constexpr (TYPE == PBX_Q41)
            q.mn[g] = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(mbuf, doff, d + g * srow, 0));
        }
      }
    }
    const unsigned at = (step >> 1) * astep + 32 * (step & 1);
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      q.Ah[t] = __builtin_bit_cast(half8, __builtin_amdgcn_raw_buffer_load_b128(hbuf, aoff + 2048 * t, at, 0));
      q.Al[t] = __builtin_bit_cast(half8, __builtin_amdgcn_raw_buffer_load_b128(lbuf, aoff + 2048 * t, at, 0));
    }
  };
  auto multiply = [&](const BackRaw<TYPE, TT> &q, _Float16 f1, _Float16 f2, float fs) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      half8 H, L = {};
      if constexpr (TYPE == PBX_F16) {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const half2t z = as_half2(__builtin_amdgcn_perm(q.w[4 * p + 2 + (i >> 1)], q.w[4 * p + (i >> 1)],
                                                          i & 1 ? 0x07060302u : 0x05040100u));
          H[2 * p] = z[0];
          H[2 * p + 1] = z[1];
        }
      } else if constexpr (TYPE == PBX_Q6K || TYPE == PBX_Q41) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float v;
          if constexpr (TYPE == PBX_Q6K) {
            // tile i is the i-th 32-code group of half a superblock
            const unsigned s8 = ((i < 2 ? q.d[e].x : q.d[e].y) >> (16 * (i & 1) + 8 * (lr >> 4))) & 255u;
            const int code = (int)((q.w[3 * e + (i & 1)] >> (4 * (i >> 1)) & 15u) | ((q.w[3 * e + 2] >> (2 * i) & 3u) << 4)) - 32;
            v = f16_bits_to_f32(q.ds[e]) * fs * (float)(int8_t)s8 * (float)code;
          } else {
            const unsigned dw = e & 2 ? q.d[e >> 2].y : q.d[e >> 2].x, mw = e & 2 ? q.mn[e >> 2].y : q.mn[e >> 2].x;
            v = fmaf((float)(q.w[e] >> (8 * (i & 1) + 4 * (i >> 1)) & 15u), f16_bits_to_f32(dw >> (16 * (e & 1))) * fs,
                     f16_bits_to_f32(mw >> (16 * (e & 1))) * fs);
          }
          H[e] = (_Float16)v;
          L[e] = (_Float16)(v - (float)H[e]);
        }
      } else {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const half2t d = as_half2(p & 1 ? q.d[p >> 1].y : q.d[p >> 1].x) * f1 * f2;
          half2t y;
          if constexpr (TYPE == PBX_Q4) {
            const unsigned x = byte_pair(q.w[2 * p], q.w[2 * p + 1], i & 1);
            const half2t off = {(_Float16)-0.015625f, (_Float16)-0.015625f};  // -8 2^-9
            const _Float16 up = i < 2 ? (_Float16)32768.f : (_Float16)2048.f;
            y = __builtin_elementwise_fma(as_half2(x & (i < 2 ? 0x000F000Fu : 0x00F000F0u)), half2t{up, up}, off);
          } else {
            const half2t off = {(_Float16)-0.25f, (_Float16)-0.25f};  // -128 2^-9
            const half2t up = {(_Float16)32768.f, (_Float16)32768.f};
            y = __builtin_elementwise_fma(as_half2(byte_pair(q.w[2 * p] ^ 0x80808080u, q.w[2 * p + 1] ^ 0x80808080u, i)), up, off);
          }
          const half2t hi = y * d, lo = __builtin_elementwise_fma(y, d, -hi);
          H[2 * p] = hi[0];
          H[2 * p + 1] = hi[1];
          L[2 * p] = lo[0];
          L[2 * p + 1] = lo[1];
        }
      }
#pragma unroll
      for (int t = 0; t < TT; ++t) acc[t][i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(q.Ah[t], H, acc[t][i], 0, 0, 0);
#pragma unroll
      for (int t = 0; t < TT; ++t) acc[t][i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(q.Al[t], H, acc[t][i], 0, 0, 0);
      if constexpr (TYPE != PBX_F16) {
#pragma unroll
        for (int t = 0; t < TT; ++t) acc[t][i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(q.Ah[t], L, acc[t][i], 0, 0, 0);
      }
    }
  };
  // step j of the wave: half of its block j / 2; D - 1 steps are under way beside the one
  // that is multiplied
  constexpr int D = BACK_DEPTH(TYPE, TT);
  const int steps = b0 + wave < b1 ? 2 * ((b1 - b0 - wave + 3) / 4) : 0;
  auto step_of = [&](int j) {  // (past the end: the last one again)
    const int i = min(j, steps - 1);
    return 2 * (wave + 4 * (i >> 1)) + (i & 1);
  };
  BackRaw<TYPE, TT> q[D];
  if (steps) {
#pragma unroll
    for (int j = 0; j < D - 1; ++j) load(step_of(j), q[j]);
  }
  const int shift = TYPE == PBX_F16 ? 0 : head_shift(a.peaks, HeadTarget<TYPE>::value);
  // codes enter as u 2^-9, so their scales take 2^9 more; by two factors, either of
  // which a half holds
  const int both = shift + 9, s1 = min(15, max(-14, both));
  const _Float16 f1 = (_Float16)power_of_two(s1), f2 = (_Float16)power_of_two(both - s1);
  const float fs = power_of_two(shift);
  int j = 0;
  for (; j + D <= steps; j += D) {
#pragma unroll
    for (int s = 0; s < D; ++s) {
      load(step_of(j + s + D - 1), q[(s + D - 1) % D]);
      __builtin_amdgcn_sched_barrier(0);  // (the loads stay ahead of the products)
      multiply(q[s], f1, f2, fs);
    }
  }
#pragma unroll
  for (int s = 0; s < D - 1; ++s)
    if (j + s < steps) multiply(q[s], f1, f2, fs);
  // the waves' sums, in a fixed order: (0 + 2) + (1 + 3)
  float *mine = red[wave & 1];
#pragma unroll
  for (int way = 0; way < 2; ++way) {
    const int from = way ? 1 : 2;  // waves from .. 2 from - 1 hand theirs to those `from` below
    if (wave >= from && wave < 2 * from) {
#pragma unroll
      for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) mine[((t * 4 + i) * 16 + r) * 64 + lane] = acc[t][i][r];
    }
    __syncthreads();
    if (wave < from) {
      const float *theirs = red[way ? 1 : wave];
#pragma unroll
      for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[t][i][r] += theirs[((t * 4 + i) * 16 + r) * 64 + lane];
    }
    __syncthreads();
  }
  if (wave) return;
  // (of pairs down to 2^-140, so no factor)
  const int undo = TYPE == PBX_F16 && a.n_f_peaks ? head_f_peak(a.f_peaks, a.n_f_peaks) - 15 : -15 - shift;
  float *part = a.part + (int64_t)blockIdx.z * a.M * a.K;
#pragma unroll
  for (int t = 0; t < TT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int m = m0 + 32 * t + 8 * (r >> 2) + 4 * h + (r & 3);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = k0 + column_of<TYPE>(lr, i);
        if (m >= a.M || k >= a.K) continue;
        float *p = part + (int64_t)m * a.K + k;
        const float x = ldexpf(acc[t][i][r], undo);
        *p = a.add ? *p + x : x;
      }
    }
}

// An F32 head: v_mfma_f32_32x32x2_f32, one entry for each half of the wave.
template <int TT>
__device__ __forceinline__ void back_f32(const BackArgs &a) {
  const int lane = threadIdx.x, lr = lane & 31, h = lane >> 5;
  const int k0 = blockIdx.x * 128, m0 = blockIdx.y * (32 * TT);
  // (fewer than 2^14 blocks and 2^12 shares)
  const int b0 = (int)((unsigned)a.blocks * blockIdx.z / (unsigned)a.KS);
  const int b1 = (int)((unsigned)a.blocks * (blockIdx.z + 1) / (unsigned)a.KS);
  const floatx16 zero = {};
  floatx16 acc[TT][4];
#pragma unroll
  for (int t = 0; t < TT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[t][i] = zero;
  const int kc = min(k0 + 4 * lr, a.K - 4);
  const float *W = reinterpret_cast<const float *>(a.qs);
  for (int b = b0; b < b1; ++b) {
#pragma unroll 4
    for (int j = 0; j < 32; j += 2) {
      const int64_t v = 32 * b + j + h;
      const float4 w = *reinterpret_cast<const float4 *>(W + min(v, (int64_t)a.rows - 1) * a.K + kc);
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const float g = a.G32[v * a.Mpad + m0 + 32 * t + lr];
        acc[t][0] = __builtin_amdgcn_mfma_f32_32x32x2f32(g, w.x, acc[t][0], 0, 0, 0);
        acc[t][1] = __builtin_amdgcn_mfma_f32_32x32x2f32(g, w.y, acc[t][1], 0, 0, 0);
        acc[t][2] = __builtin_amdgcn_mfma_f32_32x32x2f32(g, w.z, acc[t][2], 0, 0, 0);
        acc[t][3] = __builtin_amdgcn_mfma_f32_32x32x2f32(g, w.w, acc[t][3], 0, 0, 0);
      }
    }
  }
  float *part = a.part + (int64_t)blockIdx.z * a.M * a.K;
#pragma unroll
  for (int t = 0; t < TT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int m = m0 + 32 * t + 8 * (r >> 2) + 4 * h + (r & 3), k = k0 + 4 * lr;
      if (m >= a.M || k >= a.K) continue;
      float4 *p = reinterpret_cast<float4 *>(part + (int64_t)m * a.K + k);
      float4 x = make_float4(acc[t][0][r], acc[t][1][r], acc[t][2][r], acc[t][3][r]);
      if (a.add) x.x += p->x, x.y += p->y, x.z += p->z, x.w += p->w;
      *p = x;
    }
}

}  // namespace

#define HEAD_BACK(TAG, TYPE)                                                                                     \
  extern "C" __global__ void __launch_bounds__(256, 2) pbx_head_back_##TAG##_1(BackArgs a) { back_body<TYPE, 1>(a); } \
  extern "C" __global__ void __launch_bounds__(256, 2) pbx_head_back_##TAG##_2(BackArgs a) { back_body<TYPE, 2>(a); }
HEAD_BACK(q4, PBX_Q4)
HEAD_BACK(q41, PBX_Q41)
HEAD_BACK(q8, PBX_Q8)
HEAD_BACK(q6k, PBX_Q6K)
HEAD_BACK(f16, PBX_F16)
extern "C" __global__ void __launch_bounds__(64) pbx_head_back_f32_1(BackArgs a) { back_f32<1>(a); }
extern "C" __global__ void __launch_bounds__(64) pbx_head_back_f32_2(BackArgs a) { back_f32<2>(a); }

struct ReduceArgs {
  const float *part;
  int KS, M, K, folds;
  const int *targets;
  int vocab;
  const float *grad;
  float *dX;
  const float *hit, *others;  // of pbx_head_g
  int n_others;
  // the head
  int type;
  const uint8_t *qs;
  const uint16_t *dsc, *msc;
};

// dX = grad * (the partial sums together), rows without a target 0: workgroup (16
// float4s of a row), the partials over 16 threads each.  folds 2: the partial sums have
// 2 K columns, of the head's high halves and of its low ones.  Rows whose target is likelier
// than not: and the others' sum times the target's weights.  Few rows are a launch's own time and
// two chains of loads (5 rows of 576 columns, 102 partials, 384 sums of others: 5.2 us, 4.8 with no
// likely target); 512 rows of 2,048, 4 partials: 15 us.
extern "C" __global__ void __launch_bounds__(256)
pbx_head_reduce(ReduceArgs a) {
  __shared__ float4 sum[16][17];
  __shared__ __attribute__((aligned(16))) float weight[64];
  __shared__ float other[4];
  const int64_t row = blockIdx.y, MK4 = (int64_t)a.M * a.K / 4 * a.folds;
  const int c = threadIdx.x % 16, j = threadIdx.x / 16, k4 = blockIdx.x * 16 + c;
  const int t = a.targets[row];
  const float d = a.hit[row], grad = a.grad[row];  // (d: anything in a row without a target)
  const bool on = t >= 0 && t < a.vocab, likely = on && head_likely(d);
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (k4 < a.K / 4)
    for (int i = j; i < a.KS * a.folds; i += 16) {
      const int64_t at = i / a.folds * MK4 + row * a.folds * (a.K / 4) + i % a.folds * (a.K / 4) + k4;
      const float4 p = reinterpret_cast<const float4 *>(a.part)[at];
      s.x += p.x, s.y += p.y, s.z += p.z, s.w += p.w;
    }
  sum[j][c] = s;
  if (likely) {
    const int col = blockIdx.x * 64 + threadIdx.x;
    if (threadIdx.x < 64 && col < a.K) weight[threadIdx.x] = row_value(a.qs, a.dsc, a.msc, a.type, t, col, a.K);
    float g = 0.f;
    for (int i = threadIdx.x; i < a.n_others; i += 256) g += a.others[row * a.n_others + i];
    g = wave_sum(g);
    if ((threadIdx.x & 63) == 0) other[threadIdx.x >> 6] = g;
  }
  __syncthreads();
  if (j || k4 >= a.K / 4) return;
  for (int i = 1; i < 16; ++i) s.x += sum[i][c].x, s.y += sum[i][c].y, s.z += sum[i][c].z, s.w += sum[i][c].w;
  if (likely) {
    const float g = other[0] + other[1] + other[2] + other[3];
    const float4 w = *reinterpret_cast<const float4 *>(weight + 4 * c);
    s.x = fmaf(g, w.x, s.x), s.y = fmaf(g, w.y, s.y), s.z = fmaf(g, w.z, s.z), s.w = fmaf(g, w.w, s.w);
  }
  float4 *out = reinterpret_cast<float4 *>(a.dX) + row * (a.K / 4) + k4;
  *out = on ? make_float4(grad * s.x, grad * s.y, grad * s.z, grad * s.w) : make_float4(0.f, 0.f, 0.f, 0.f);
}
