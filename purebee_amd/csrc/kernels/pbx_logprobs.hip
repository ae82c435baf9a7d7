// pbx_logprobs.hip -- log probabilities of given tokens, entropy and the most
// likely tokens of rows of logits.
//
// With m = max x, S = sum e^(x - m) and T = sum e^(x - m) (x - m) of a row:
//   log p_t = x_t - m - log S,  entropy = log S - T / S
// in one pass over the row: (m, S, T) join with those of other elements as
//   S = S1 e^(m1 - m) + S2 e^(m2 - m),  T = sum (Ti + (mi - m) Si) e^(mi - m).

#include "pbx_gemv_impl.h"

using namespace pbx;

namespace {

// The maximum before any element: finite, so differences need no special case
// (an element of -inf adds nothing; a row of nothing else keeps S == 0).
constexpr float LOWEST = -3.402823466e38f;
constexpr int LP_TOP = 32;

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
__device__ __forceinline__ Sums joined(Sums a, Sums b) {
  const float m = fmaxf(a.m, b.m);
  a = moved(a, m);
  b = moved(b, m);
  return {m, a.s + b.s, a.t + b.t};
}

// Larger logits have larger keys, equal ones the lower index.
__device__ __forceinline__ uint64_t key_of(float x, unsigned i) {
  const unsigned u = __float_as_uint(x + 0.f);  // -0 as 0
  return (uint64_t)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (0xFFFFFFFFu - i);
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const unsigned u = (unsigned)(k >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

// The value of the lane that differs in bit OFF, without a trip through LDS:
// DPP moves inside a row of 16 lanes (lane ^ 4 as (lane ^ 7) ^ 3), lane swaps
// across rows and halves.
template <int CTRL>
__device__ __forceinline__ unsigned dpp(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
}
template <int OFF>
__device__ __forceinline__ unsigned partner(unsigned v, bool upper) {
  if constexpr (OFF == 1) return dpp<0xB1>(v);         // quad_perm 1 0 3 2
  else if constexpr (OFF == 2) return dpp<0x4E>(v);    // quad_perm 2 3 0 1
  else if constexpr (OFF == 4) return dpp<0x1B>(dpp<0x141>(v));  // row_half_mirror, quad_perm 3 2 1 0
  else if constexpr (OFF == 8) return dpp<0x128>(v);   // row_ror 8
  else if constexpr (OFF == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return upper ? r[0] : r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return upper ? r[0] : r[1];
  }
}
// One step of a bitonic network over bit OFF: the lanes with `first` keep the
// larger key.
template <int OFF>
__device__ __forceinline__ uint64_t exchange(uint64_t v, int lane, bool first) {
  const bool upper = lane & OFF;
  const uint64_t o = (uint64_t)partner<OFF>((unsigned)(v >> 32), upper) << 32 | partner<OFF>((unsigned)v, upper);
  return first == (o > v) ? o : v;
}
// From a bitonic sequence over 2 OFF lanes to a sorted one.
template <int OFF>
__device__ __forceinline__ uint64_t settle(uint64_t v, int lane, bool down) {
  v = exchange<OFF>(v, lane, ((lane & OFF) == 0) == down);
  if constexpr (OFF > 1) v = settle<OFF / 2>(v, lane, down);
  return v;
}
// A wave's 64 keys in descending (down) or ascending order.
__device__ __forceinline__ uint64_t sort_wave(uint64_t v, int lane, bool down) {
  v = settle<1>(v, lane, (lane & 2) == 0);
  v = settle<2>(v, lane, (lane & 4) == 0);
  v = settle<4>(v, lane, (lane & 8) == 0);
  v = settle<8>(v, lane, (lane & 16) == 0);
  v = settle<16>(v, lane, (lane & 32) == 0);
  return settle<32>(v, lane, down);
}
// The 64 largest of a descending list and an ascending one, in descending order.
__device__ __forceinline__ uint64_t merge_wave(uint64_t down, uint64_t up, int lane) {
  return settle<32>(up > down ? up : down, lane, true);
}

// The 64 largest keys of W waves' descending lists, in wave 0.
template <int W>
__device__ __forceinline__ uint64_t merge_waves(uint64_t v, uint64_t (*buf)[64], int wave, int lane) {
#pragma unroll
  for (int h = W / 2; h >= 1; h /= 2) {
    if (wave >= h && wave < 2 * h) buf[wave][lane] = v;
    __syncthreads();
    if (wave < h) v = merge_wave(v, buf[wave + h][63 - lane], lane);
    __syncthreads();
  }
  return v;
}

// The sums of all threads of W waves: one maximum first, then each moves once.
template <int W>
__device__ __forceinline__ Sums join_waves(Sums a, float (*buf)[4], int wave, int lane) {
  float m = wave_max(a.m);
  if (lane == 0) buf[wave][0] = m;
  __syncthreads();
  m = buf[0][0];
#pragma unroll
  for (int w = 1; w < W; ++w) m = fmaxf(m, buf[w][0]);
  a = moved(a, m);
  const float s = wave_sum(a.s), t = wave_sum(a.t);
  if (lane == 0) {
    buf[wave][1] = s;
    buf[wave][2] = t;
  }
  __syncthreads();
  a = {m, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < W; ++w) {
    a.s += buf[w][1];
    a.t += buf[w][2];
  }
  return a;
}

struct Out {
  const int *targets;
  float *logp, *entropy;
  int *top_ids;
  float *top_logp;
};

// The target's logit in row `row` at x, NaN where there is none.  It is asked for
// early, in two steps: one load waits for the other.
__device__ __forceinline__ int target_of(const Out &o, int64_t row) { return o.logp ? o.targets[row] : -1; }
__device__ __forceinline__ float logit_of(const float *x, int target, int vocab) {
  return target >= 0 && target < vocab ? x[target] : __uint_as_float(0x7fc00000u);
}
// The answers for row `row` from its target's logit xt, its sums and (lane i) i-th largest key.
__device__ __forceinline__ void answer(const Out &o, int64_t row, float xt, int top, Sums a, uint64_t key, int lane) {
  const bool none = !(a.s > 0.f && a.s < INFINITY);  // no distribution
  const float ls = logf(a.s), nan = __uint_as_float(0x7fc00000u);
  if (lane == 0) {
    if (o.logp) o.logp[row] = none ? nan : xt - a.m - ls;
    if (o.entropy) o.entropy[row] = none ? nan : ls - a.t / a.s;
  }
  if (lane < top) {
    if (o.top_ids) o.top_ids[row * top + lane] = none ? -1 : (int)(0xFFFFFFFFu - (unsigned)key);
    if (o.top_logp) o.top_logp[row * top + lane] = none ? nan : key_value(key) - a.m - ls;
  }
}

// Four elements join a thread's sums, and the group its first largest one.  The
// maximum follows only when passed by SLACK (e^8 of a probability): among 64
// lanes some would meet a new maximum in nearly every group.
constexpr float SLACK = 8.f;
struct Share {
  Sums a;
  float best;
  int at;
};
__device__ __forceinline__ void take(Share &t, float4 v, int g) {
  const float top4 = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
  if (top4 > t.best || t.at < 0 || (top4 == t.best && g < t.at)) {
    t.best = top4;
    t.at = g;
  }
  if (top4 > t.a.m + SLACK) t.a = moved(t.a, top4);
  const float d[4] = {v.x - t.a.m, v.y - t.a.m, v.z - t.a.m, v.w - t.a.m};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float p = exp_of(d[e]);
    t.a.s += p;
    t.a.t = fmaf(p, bounded(d[e]), t.a.t);
  }
}

// The elements i .. i + 3 of a row at its ends: absent ones as -inf.
__device__ __forceinline__ float4 end_group(const float *x, int i, int vocab) {
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = i + e >= 0 && i + e < vocab ? x[i + e] : -INFINITY;
  return make_float4(v[0], v[1], v[2], v[3]);
}
// Parts' results cross workgroups, of one launch as well: stores and loads at the
// device's coherence point.
template <typename T>
__device__ __forceinline__ void put(T *p, T v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ T get(const T *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Row `row`'s parts put together by W waves.
template <int W>
__device__ __forceinline__ void join_parts(int parts, int top, const Out &out, const float *sums,
                                           const uint64_t *keys, int64_t row, float xt, float (*sbuf)[4],
                                           uint64_t (*kbuf)[64]) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  Sums a = {LOWEST, 0.f, 0.f};
  for (int i = tid; i < parts; i += 64 * W) {
    const float *s = sums + 3 * (row * parts + i);
    a = joined(a, {get(s), get(s + 1), get(s + 2)});
  }
  uint64_t key = 0;
  const int n = parts * top;
  for (int i = tid - lane; i < n; i += 64 * W)
    key = merge_wave(key, sort_wave(i + lane < n ? get(keys + row * n + i + lane) : 0, lane, false), lane);
  a = join_waves<W>(a, sbuf, wave, lane);
  if (top) key = merge_waves<W>(key, kbuf, wave, lane);
  if (!wave) answer(out, row, xt, top, a, key, lane);
}

// Parts done so far of a row, each count in a cache line of its own; zero between
// launches.  Every context loads its own; its eager launches follow one another.
constexpr int LP_MERGED_ROWS = 512;
__device__ unsigned lp_arrived[32 * LP_MERGED_ROWS];

// Workgroup (part, row): the row's 16-byte groups in `parts` pieces of at most
// LP_SHARE groups a thread.  A thread keeps its sums and its first largest
// group; the `top` threads with the largest ones hold the piece's `top` largest
// elements among them (those threads' maxima alone are `top` elements as large),
// so only their groups, read again, are looked through.  Many rows are bound by
// bytes (512 x 128256, 20 tokens: 56 us, 4.7 TB/s); few by one chain of loads,
// sorts and merges, and the same again where parts are joined (1 x 128256, 8
// tokens: 10.2 us; 37 x 32003, 5 tokens, not split: 9.8).  The last workgroup of a
// row joins its parts: 6 % less than in a launch of its own.
template <int LP_T, int LP_SHARE>
__device__ __forceinline__ void part_body(const float *logits, int64_t stride, int vocab, int parts, int top, Out out,
                                          float *sums, uint64_t *keys, int merged) {
  constexpr int W = LP_T / 64;
  __shared__ float sbuf[W][4];
  __shared__ uint64_t kbuf[W][64];
  __shared__ int chosen[LP_TOP];
  __shared__ int count, n_chosen, last;
  __shared__ uint64_t limit;
  __shared__ uint64_t list[LP_TOP * LP_SHARE * 4 + 8];  // (and the cut groups)
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x / parts;
  const int part = (int)(blockIdx.x % parts);
  const float *x = logits + row * stride;
  const int skew = (int)((uintptr_t)x / 4 & 3);  // elements of the first group before the row
  const int groups = (int)(((int64_t)vocab + skew + 3) / 4);
  const int g0 = (int)((int64_t)groups * part / parts), g1 = (int)((int64_t)groups * (part + 1) / parts);
  // whole groups, four of a thread under way at once, then a row's cut ones
  const int full = (vocab + skew) / 4;
  const int f0 = max(g0, skew ? 1 : 0), f1 = min(g1, full);
  const int target = target_of(out, row);
  Share t = {{LOWEST, 0.f, 0.f}, -INFINITY, -1};
  const float4 *x4 = reinterpret_cast<const float4 *>(x - skew);
  int g = f0 + tid;
  for (; g + 3 * LP_T < f1; g += 4 * LP_T) {
    float4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = x4[g + k * LP_T];
#pragma unroll
    for (int k = 0; k < 4; ++k) take(t, v[k], g + k * LP_T);
  }
  for (; g < f1; g += LP_T) take(t, x4[g], g);
  // (a row that lies within one group is its first)
  const bool head = skew && g0 == 0, tail = full < groups && g1 == groups && !(skew && full == 0);
  if (head && tid == 0) take(t, end_group(x, -skew, vocab), 0);
  if (tail && tid == 64) take(t, end_group(x, 4 * full - skew, vocab), full);
  const float xt = logit_of(x, target, vocab);
  Sums a = t.a;
  const int at = t.at;
  a = join_waves<W>(a, sbuf, wave, lane);
  uint64_t key = 0;
  if (top) {
    const uint64_t mine = at < 0 ? 0 : key_of(t.best, (unsigned)at);
    key = merge_waves<W>(sort_wave(mine, lane, true), kbuf, wave, lane);
    if (tid == top - 1) limit = key;
    if (tid == 0) count = n_chosen = 0;
    __syncthreads();
    if (mine && mine >= limit) chosen[atomicAdd(&n_chosen, 1)] = tid;
    __syncthreads();
    // a group's key is at most those of its largest elements, which have its value
    const float floor_value = limit ? key_value(limit) : -INFINITY;
    auto look = [&](float4 v, int i0) {
      const float u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i0 + e >= 0 && i0 + e < vocab && u[e] >= floor_value)
          list[atomicAdd(&count, 1)] = key_of(u[e], (unsigned)(i0 + e));
    };
    const int share = (max(f1 - f0, 0) + LP_T - 1) / LP_T, n = n_chosen * share;
    for (int i = tid; i < n; i += LP_T) {
      const int g = f0 + chosen[i / share] + i % share * LP_T;
      if (g < f1) look(x4[g], 4 * g - skew);
    }
    if (head && tid == 0) look(end_group(x, -skew, vocab), -skew);
    if (tail && tid == 64) look(end_group(x, 4 * full - skew, vocab), 4 * full - skew);
    __syncthreads();
    key = 0;
    if (count <= 64) {  // nearly always
      if (!wave) key = sort_wave(lane < count ? list[lane] : 0, lane, true);
    } else {
      for (int i = 64 * wave; i < count; i += LP_T)
        key = merge_wave(key, sort_wave(i + lane < count ? list[i + lane] : 0, lane, false), lane);
      key = merge_waves<W>(key, kbuf, wave, lane);
    }
  }
  if (parts == 1) {
    if (!wave) answer(out, row, xt, top, a, key, lane);
    return;
  }
  if (!wave) {
    float *s = sums + 3 * (int64_t)blockIdx.x;
    if (lane < 3) put(s + lane, lane == 0 ? a.m : lane == 1 ? a.s : a.t);
    if (lane < top) put(keys + blockIdx.x * (int64_t)top + lane, key);
  }
  if (!merged) return;
  // the part lies at the coherence point before it is counted; the workgroup
  // that completes the row's count reads the others' from there
  if (tid == 0) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    last = __hip_atomic_fetch_add(&lp_arrived[32 * row], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
           (unsigned)parts - 1;
    if (last) __hip_atomic_store(&lp_arrived[32 * row], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (last) join_parts<W>(parts, top, out, sums, keys, row, xt, sbuf, kbuf);
}

}  // namespace

// Parts of up to 8 groups a thread (short ones, whose time is their latency) run
// on four waves, with a merge less; longer ones on eight.
extern "C" __global__ void __launch_bounds__(256)
pbx_logprobs_part_256(const float *logits, int64_t stride, int vocab, int parts, int top, Out out, float *sums,
                      uint64_t *keys, int merged) {
  part_body<256, 8>(logits, stride, vocab, parts, top, out, sums, keys, merged);
}
extern "C" __global__ void __launch_bounds__(512)
pbx_logprobs_part_512(const float *logits, int64_t stride, int vocab, int parts, int top, Out out, float *sums,
                      uint64_t *keys, int merged) {
  part_body<512, 64>(logits, stride, vocab, parts, top, out, sums, keys, merged);
}

// A row's parts put together in a launch of their own: one workgroup of four waves a row.
extern "C" __global__ void __launch_bounds__(256)
pbx_logprobs_join(const float *logits, int64_t stride, int vocab, int parts, int top, Out out, const float *sums,
                  const uint64_t *keys) {
  __shared__ float sbuf[4][4];
  __shared__ uint64_t kbuf[4][64];
  const int64_t row = blockIdx.x;
  const float xt = logit_of(logits + row * stride, target_of(out, row), vocab);
  join_parts<4>(parts, top, out, sums, keys, row, xt, sbuf, kbuf);
}
