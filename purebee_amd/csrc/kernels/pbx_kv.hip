// pbx_kv.hip -- the paged 8-bit KV cache: append with the position rotation,
// attention over the cache, and reading it back.
//
// A block is PBX_KV_BLOCK = 32 positions of one sequence and KV head: 32 HDP
// bytes of keys, then as many of values (HDP: head_dim padded to the kernel's
// width), each byte a code + 128, and two f32 scales.  Both halves lie as the
// operands of v_mfma_f32_16x16x32_f16 take them, 16 bytes a lane (lane l = 16 g
// + c), a wave's load 1 KB in one piece:
//   keys    [HDP / 64][32 keys][64 dims]: lane (c, g) reads dims 16 g .. + 15 of
//           key c of a 16-key tile, 8 for each of two products; the last 32 dims
//           of an odd HDP / 32 as [32 keys][32 dims], 8 bytes a lane
//   values  [HDP / 32][16 dims][4][2][8 keys]: lane (c, g) reads dims c and
//           c + 16 of a 32-dim group at the keys 4 g .. + 3 and 16 + 4 g .. + 3,
//           which are those whose scores the lane holds (the D layout's rows)

#include "pbx_gemv_impl.h"

using namespace pbx;

namespace {

constexpr int BLK = 32;

struct KvArgs {
  uint8_t *codes;  // of the layer: [page][kv head][block][keys | values]
  float *scales;   // [page][kv head][block][key, value]
  int kv_heads, groups, head_dim, page_shift;
};
struct KvRope {
  const double *table;  // [position][dim / 2][cos, sin]
  int style, dim;       // PBX_ROPE_*
};
// kv_block_item, kv_attn_item and kv_join_item of pbx_kv_plan.h
struct BlockItem {
  int page, sub, pos0, start, count, row0, pad[2];
};
struct AttnItem {
  int start, count, row0, tile, blk0, blk1, tab, slot;
};
struct JoinItem {
  int count, row0, tile, slot, n, pad[3];
};

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2t __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
typedef unsigned uintx2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ int64_t block_index(const KvArgs &a, int page, int head, int sub) {
  return (((int64_t)page * a.kv_heads + head) << a.page_shift) + sub;
}

template <int HDP>
__device__ __forceinline__ int key_byte(int key, int dim) {
  return dim < HDP / 64 * 64 ? (dim >> 6) * (BLK * 64) + key * 64 + (dim & 63)
                             : HDP / 64 * (BLK * 64) + key * 32 + (dim & 31);
}
__device__ __forceinline__ int value_byte(int key, int dim) {
  const int slot = 8 * ((key >> 2) & 3) + 4 * (key >> 4) + (key & 3);
  return (dim >> 5) * 1024 + (dim & 15) * 64 + (slot >> 3) * 16 + ((dim >> 4) & 1) * 8 + (slot & 7);
}

// x / s rounded half to even, as the true quotient: x * (1 / s) is a few ulp off
// it, so only quotients next to a border need the division.
__device__ __forceinline__ int code_of(double x, double s, double inv) {
  if (!(s > 0.0 && s < INFINITY)) return 0;
  const double q = x * inv;
  double r = rint(q);
  if (fabs(fabs(q - r) - 0.5) < 1e-9) r = rint(x / s);
  return (int)r;
}

// The scale that a largest magnitude asks for (in bits: a NaN is the largest).
__device__ __forceinline__ float scale_of(uint64_t peak) {
  const float s = (float)(__longlong_as_double((long long)peak) / 127.0);
  return s < 0x1p-120f ? 0.f : s;
}
__device__ __forceinline__ float larger(float a, float b) {  // of scales: a NaN is the largest
  return __float_as_uint(a) > __float_as_uint(b) ? a : b;
}
__device__ __forceinline__ uint64_t magnitude(double x) {
  return (uint64_t)__double_as_longlong(x) & 0x7fffffffffffffffull;
}

// Where unit u (4 dims: two pairs that turn, or 4 that do not) of a head lies:
// dims a, a + 1 and b, b + 1.
__device__ __forceinline__ void unit_dims(const KvRope &r, int u, int &a, int &b) {
  if (r.style == 2 && 4 * u < r.dim) {
    a = 2 * u;
    b = 2 * u + r.dim / 2;
  } else {
    a = 4 * u;
    b = 4 * u + 2;
  }
}
// Turns unit u by position pos: x[0..1] at dims a, a + 1, x[2..3] at b, b + 1.
__device__ __forceinline__ void turn(const KvRope &r, int u, int pos, double x[4]) {
  if (4 * u >= r.dim) return;
  const double2 *cs = reinterpret_cast<const double2 *>(r.table) + (size_t)pos * (r.dim / 2) + 2 * u;
  const double2 p = cs[0], q = cs[1];
  const double x0 = x[0], x1 = x[1], x2 = x[2], x3 = x[3];
  if (r.style == 2) {
    x[0] = x0 * p.x - x2 * p.y;
    x[2] = x0 * p.y + x2 * p.x;
    x[1] = x1 * q.x - x3 * q.y;
    x[3] = x1 * q.y + x3 * q.x;
  } else {
    x[0] = x0 * p.x - x1 * p.y;
    x[1] = x0 * p.y + x1 * p.x;
    x[2] = x2 * q.x - x3 * q.y;
    x[3] = x2 * q.y + x3 * q.x;
  }
}

__device__ __forceinline__ uint64_t block_max_u64(uint64_t v, uint64_t *red) {
  v = wave_max_u64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < 4; ++w) v = red[w] > v ? red[w] : v;
  return v;
}

// Append: workgroup (block, KV head), then workgroups of 256 query units.  The
// block's new rows are read once, turned and held in registers; the block's
// codes are put together in LDS (with the earlier rows' codes, if there are any)
// and stored whole.
template <int HDP>
__device__ __forceinline__ void append_body(const KvArgs &a, const KvRope &r, const BlockItem *items,
                                            int n_blocks, const int *row_pos, int n_rows, const float *K,
                                            int64_t ks, const float *V, int64_t vs, const float *Q, int64_t qs,
                                            float *Qout, int64_t qos) {
  constexpr int UNITS = BLK * HDP / 4 / 256;  // a thread's units of a block
  __shared__ __attribute__((aligned(16))) uint8_t img[2 * BLK * HDP];
  __shared__ uint64_t red[4];
  const int units = a.head_dim / 4, tid = threadIdx.x;
  const int64_t wg = blockIdx.x;
  if (wg >= (int64_t)n_blocks * a.kv_heads) {
    const int64_t i = (wg - (int64_t)n_blocks * a.kv_heads) * 256 + tid;
    const int heads = a.kv_heads * a.groups;
    const int64_t row = i / (heads * units);
    if (row >= n_rows) return;
    const int h = (int)(i % (heads * units)) / units, u = (int)(i % units);
    int da, db;
    unit_dims(r, u, da, db);
    const float *q = Q + row * qs + (int64_t)h * a.head_dim;
    const float2 lo = *reinterpret_cast<const float2 *>(q + da), hi = *reinterpret_cast<const float2 *>(q + db);
    double x[4] = {lo.x, lo.y, hi.x, hi.y};
    turn(r, u, row_pos[row], x);
    float *o = Qout + row * qos + (int64_t)h * a.head_dim;
    *reinterpret_cast<float2 *>(o + da) = make_float2((float)x[0], (float)x[1]);
    *reinterpret_cast<float2 *>(o + db) = make_float2((float)x[2], (float)x[3]);
    return;
  }
  const BlockItem it = items[wg / a.kv_heads];
  const int head = (int)(wg % a.kv_heads);
  const int64_t bi = block_index(a, it.page, head, it.sub);
  uint8_t *codes = a.codes + bi * (2 * BLK * HDP);
  // rows lo .. hi - 1 of the block are new, those before lo were there
  const int lo = it.start > it.pos0 ? it.start - it.pos0 : 0;
  const int hi = min(BLK, it.start + it.count - it.pos0);
  const int nu = (hi - lo) * units;  // units of the new rows
  double xk[UNITS][4];
  float xv[UNITS][4];
  uint64_t pk = 0, pv = 0;
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    const int j = tid + 256 * i;
    if (j < nu) {
      const int key = lo + j / units, u = j % units;
      const int64_t row = (int64_t)it.row0 + it.pos0 + key - it.start;
      int da, db;
      unit_dims(r, u, da, db);
      const float *k = K + row * ks + (int64_t)head * a.head_dim;
      const float2 k0 = *reinterpret_cast<const float2 *>(k + da), k1 = *reinterpret_cast<const float2 *>(k + db);
      const float4 v = *reinterpret_cast<const float4 *>(V + row * vs + (int64_t)head * a.head_dim + 4 * u);
      xk[i][0] = k0.x; xk[i][1] = k0.y; xk[i][2] = k1.x; xk[i][3] = k1.y;
      xv[i][0] = v.x; xv[i][1] = v.y; xv[i][2] = v.z; xv[i][3] = v.w;
      turn(r, u, it.pos0 + key, xk[i]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t mk = magnitude(xk[i][e]), mv = magnitude(xv[i][e]);
        pk = mk > pk ? mk : pk;
        pv = mv > pv ? mv : pv;
      }
    }
  }
  float ok = 0.f, ov = 0.f;
  if (lo > 0) {
    ok = a.scales[2 * bi];
    ov = a.scales[2 * bi + 1];
    for (int i = tid; i < 2 * BLK * HDP / 16; i += 256)
      reinterpret_cast<uintx4 *>(img)[i] = reinterpret_cast<const uintx4 *>(codes)[i];
  } else {
    for (int i = tid; i < 2 * BLK * HDP / 4; i += 256) reinterpret_cast<unsigned *>(img)[i] = 0x80808080u;
  }
  const float nk = larger(ok, scale_of(block_max_u64(pk, red))), nv = larger(ov, scale_of(block_max_u64(pv, red)));
  const double ik = 1.0 / (double)nk, iv = 1.0 / (double)nv;
  // (the reductions' barriers order the image's fill before this)
  if (lo > 0) {
    const bool gk = __float_as_uint(nk) != __float_as_uint(ok), gv = __float_as_uint(nv) != __float_as_uint(ov);
    if (gk || gv) {
      for (int i = tid; i < lo * HDP; i += 256) {
        const int key = i / HDP, dim = i % HDP;
        uint8_t *pkb = img + key_byte<HDP>(key, dim), *pvb = img + BLK * HDP + value_byte(key, dim);
        if (gk) *pkb = (uint8_t)(code_of((double)((int)*pkb - 128) * (double)ok, nk, ik) + 128);
        if (gv) *pvb = (uint8_t)(code_of((double)((int)*pvb - 128) * (double)ov, nv, iv) + 128);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    const int j = tid + 256 * i;
    if (j < nu) {
      const int key = lo + j / units, u = j % units;
      int da, db;
      unit_dims(r, u, da, db);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int dk = (e < 2 ? da : db) + (e & 1);
        img[key_byte<HDP>(key, dk)] = (uint8_t)(code_of(xk[i][e], nk, ik) + 128);
        img[BLK * HDP + value_byte(key, 4 * u + e)] = (uint8_t)(code_of(xv[i][e], nv, iv) + 128);
      }
    }
  }
  __syncthreads();
  for (int i = tid; i < 2 * BLK * HDP / 16; i += 256)
    reinterpret_cast<uintx4 *>(codes)[i] = reinterpret_cast<const uintx4 *>(img)[i];
  if (tid == 0) *reinterpret_cast<float2 *>(a.scales + 2 * bi) = make_float2(nk, nv);
}

// Reading back: workgroup (block, KV head).
template <int HDP>
__device__ __forceinline__ void read_body(const KvArgs &a, const BlockItem *items, float *K, int64_t ks, float *V,
                                          int64_t vs) {
  const BlockItem it = items[blockIdx.x / a.kv_heads];
  const int head = (int)(blockIdx.x % a.kv_heads);
  const int64_t bi = block_index(a, it.page, head, it.sub);
  const uint8_t *codes = a.codes + bi * (2 * BLK * HDP);
  const float sk = a.scales[2 * bi], sv = a.scales[2 * bi + 1];
  const int lo = it.start > it.pos0 ? it.start - it.pos0 : 0;
  const int hi = min(BLK, it.start + it.count - it.pos0);
  const int units = a.head_dim / 4;
  for (int j = threadIdx.x; j < (hi - lo) * units; j += 256) {
    const int key = lo + j / units, d = 4 * (j % units);
    const int64_t row = (int64_t)it.row0 + it.pos0 + key - it.start;
    if (K) {
      const uint8_t *p = codes + key_byte<HDP>(key, d);
      *reinterpret_cast<float4 *>(K + row * ks + (int64_t)head * a.head_dim + d) =
          make_float4((p[0] - 128) * sk, (p[1] - 128) * sk, (p[2] - 128) * sk, (p[3] - 128) * sk);
    }
    if (V) {
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (codes[BLK * HDP + value_byte(key, d + e)] - 128) * sv;
      *reinterpret_cast<float4 *>(V + row * vs + (int64_t)head * a.head_dim + d) =
          make_float4(v[0], v[1], v[2], v[3]);
    }
  }
}

// 8 codes + 128 as halves: byte b under the exponent byte 0x64 is the half
// 1024 + b.
__device__ __forceinline__ half8 halves(unsigned w0, unsigned w1) {
  union {
    unsigned u[4];
    half2t h[4];
    half8 v;
  } x;
  x.u[0] = __builtin_amdgcn_perm(0x64646464u, w0, 0x04010400u);
  x.u[1] = __builtin_amdgcn_perm(0x64646464u, w0, 0x04030402u);
  x.u[2] = __builtin_amdgcn_perm(0x64646464u, w1, 0x04010400u);
  x.u[3] = __builtin_amdgcn_perm(0x64646464u, w1, 0x04030402u);
  const half2t off = {(_Float16)1152.f, (_Float16)1152.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) x.h[i] -= off;
  return x.v;
}

// Score of a masked key and the running maximum before any visible one: finite,
// so that differences of maxima need no special case.
constexpr float NONE = -1e38f;
// Probabilities are held times 2^12 (their sum too): an fp16 pair then keeps
// 22 bits of them down to 2^-15 of the row's largest, and some down to 2^-36.
constexpr float LIFT = 12.f;

// One row's state while it travels between waves or workgroups: maximum (in
// powers of two), sum and weighted values.
//
// Attention: workgroup (item, KV head), four waves that take the item's blocks
// in turn.  A wave holds 16 query rows (token, head of the group) as the columns
// of its products: scores S = K Q^T of 32 keys (two 16-key tiles), a softmax
// step whose maxima and sums stay within a column (lanes c, c + 16, c + 32,
// c + 48), and O^T += V^T P^T with P taken from the score registers as they lie.
// Codes are exact in fp16; queries (divided by a power of two near the row's
// largest) and probabilities enter as fp16 pairs, two products each, summed in
// f32.  The block's key scale joins the row's factor, its value scale weighs the
// block's products as they are added up.
template <int HDP>
__device__ __forceinline__ void attn_body(const KvArgs &a, const AttnItem *items, const int *table, const float *Q,
                                          int64_t qs, float scale, float *O, int64_t os, float *part) {
  constexpr int HC = HDP / 32, PAIRS = HDP / 64, DT = HDP / 16;
  __shared__ __attribute__((aligned(16))) float mrg[2][DT * 64 * 4];
  __shared__ float mrg_ml[4][2][16];
  const AttnItem it = items[blockIdx.x / a.kv_heads];
  const int head = (int)(blockIdx.x % a.kv_heads);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
  const int r = it.tile * 16 + c, tok = r / a.groups;
  const bool live = tok < it.count;
  const int pos = live ? it.start + tok : -1;
  const int64_t row = (int64_t)it.row0 + tok;
  const int qhead = head * a.groups + r % a.groups;
  half8 qh[HC], ql[HC];
  float factor;  // of the products: the row's power of two, scale, log2(e)
  {
    float x[HC][8];
    const float *q = Q + row * qs + (int64_t)qhead * a.head_dim;
    unsigned peak = 0;
#pragma unroll
    for (int i = 0; i < HC; ++i)
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const int d = i < 2 * PAIRS ? 64 * (i >> 1) + 16 * g + 8 * (i & 1) + e : 32 * i + 8 * g + e;
        const float4 v = live && d < a.head_dim ? *reinterpret_cast<const float4 *>(q + d)
                                                : make_float4(0.f, 0.f, 0.f, 0.f);
        x[i][e] = v.x; x[i][e + 1] = v.y; x[i][e + 2] = v.z; x[i][e + 3] = v.w;
#pragma unroll
        for (int k = 0; k < 4; ++k) peak = max(peak, __float_as_uint(x[i][e + k]) & 0x7fffffffu);
      }
    peak = max(peak, (unsigned)__shfl_xor((int)peak, 16, 64));
    peak = max(peak, (unsigned)__shfl_xor((int)peak, 32, 64));
    const unsigned ex = min(max(peak >> 23, 1u), 253u);
    const float down = __uint_as_float((254u - ex) << 23);  // 2^(127 - ex)
    factor = __uint_as_float(ex << 23) * scale * 1.44269504f;
#pragma unroll
    for (int i = 0; i < HC; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = x[i][e] * down;
        const _Float16 h = (_Float16)y;
        qh[i][e] = h;
        ql[i][e] = (_Float16)(y - (float)h);
      }
  }
  const floatx4 zero = {0.f, 0.f, 0.f, 0.f};
  floatx4 acc[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) acc[i] = zero;
  float m = NONE, l = 0.f;
  for (int b = it.blk0 + wave; b < it.blk1; b += 4) {
    const int page = table[it.tab + (b >> a.page_shift)];
    const int64_t bi = block_index(a, page, head, b & ((1 << a.page_shift) - 1));
    const uint8_t *kb = a.codes + bi * (2 * BLK * HDP), *vb = kb + BLK * HDP;
    const float2 sc = *reinterpret_cast<const float2 *>(a.scales + 2 * bi);
    floatx4 s[2] = {zero, zero};
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int p = 0; p < PAIRS; ++p) {
        const uintx4 w = *reinterpret_cast<const uintx4 *>(kb + p * (BLK * 64) + (16 * t + c) * 64 + 16 * g);
        const half8 k0 = halves(w[0], w[1]), k1 = halves(w[2], w[3]);
        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qh[2 * p], s[t], 0, 0, 0);
        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, ql[2 * p], s[t], 0, 0, 0);
        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qh[2 * p + 1], s[t], 0, 0, 0);
        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, ql[2 * p + 1], s[t], 0, 0, 0);
      }
      if constexpr (HC % 2) {
        const uintx2 w = *reinterpret_cast<const uintx2 *>(kb + PAIRS * (BLK * 64) + (16 * t + c) * 32 + 8 * g);
        const half8 k0 = halves(w[0], w[1]);
        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qh[HC - 1], s[t], 0, 0, 0);
        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, ql[HC - 1], s[t], 0, 0, 0);
      }
    }
    const float f = factor * sc.x;
    float x[8], mx = NONE;
    const int p0 = b * BLK + 4 * g;
    const bool whole = b * BLK + BLK - 1 <= it.start;  // every live row sees the block
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int p = p0 + 16 * (e >> 2) + (e & 3);
      x[e] = s[e >> 2][e & 3] * f;
      if (!whole && p > pos) x[e] = NONE;
      mx = fmaxf(mx, x[e]);
    }
    mx = pair_max<32>(pair_max<16>(mx));
    const float mn = fmaxf(m, mx);
    const float al = __builtin_amdgcn_exp2f(m - mn);
    const float base = mn == NONE ? 0.f : mn - LIFT;
    float sum = 0.f;
    half8 ph, pl;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float p = __builtin_amdgcn_exp2f(x[e] - base);
      sum += p;
      const _Float16 h = (_Float16)p;
      ph[e] = h;
      pl[e] = (_Float16)(p - (float)h);
    }
    l = fmaf(l, al, sum);  // of this lane's keys: the column's sum is taken at the end
    m = mn;
#pragma unroll
    for (int i = 0; i < HC; ++i) {
      const uintx4 w = *reinterpret_cast<const uintx4 *>(vb + i * 1024 + c * 64 + 16 * g);
      const half8 v0 = halves(w[0], w[1]), v1 = halves(w[2], w[3]);
      floatx4 d0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph, zero, 0, 0, 0);
      floatx4 d1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, ph, zero, 0, 0, 0);
      d0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pl, d0, 0, 0, 0);
      d1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pl, d1, 0, 0, 0);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        acc[2 * i][e] = fmaf(d0[e], sc.y, acc[2 * i][e] * al);
        acc[2 * i + 1][e] = fmaf(d1[e], sc.y, acc[2 * i + 1][e] * al);
      }
    }
  }
  l = pair_sum<32>(pair_sum<16>(l));
  // the waves' states: one maximum, then the sums, waves 2 and 3 into 0 and 1,
  // 1 into 0
  if (g == 0) mrg_ml[wave][0][c] = m;
  __syncthreads();
  float M = mrg_ml[0][0][c];
#pragma unroll
  for (int w = 1; w < 4; ++w) M = fmaxf(M, mrg_ml[w][0][c]);
  const float al = __builtin_amdgcn_exp2f(m - M);
  l *= al;
  if (g == 0) mrg_ml[wave][1][c] = l;
#pragma unroll
  for (int i = 0; i < DT; ++i) acc[i] *= al;
#pragma unroll
  for (int half = 2; half >= 1; half /= 2) {
    if (wave >= half && wave < 2 * half)
#pragma unroll
      for (int i = 0; i < DT; ++i)
        *reinterpret_cast<floatx4 *>(&mrg[wave - half][(i * 64 + lane) * 4]) = acc[i];
    __syncthreads();
    if (wave < half)
#pragma unroll
      for (int i = 0; i < DT; ++i) acc[i] += *reinterpret_cast<const floatx4 *>(&mrg[wave][(i * 64 + lane) * 4]);
    __syncthreads();
  }
  if (wave) return;
  l = mrg_ml[0][1][c] + mrg_ml[1][1][c] + mrg_ml[2][1][c] + mrg_ml[3][1][c];
  if (it.slot < 0) {
    if (!live) return;
    const float inv = 1.f / l;
    float *o = O + row * os + (int64_t)qhead * a.head_dim;
#pragma unroll
    for (int i = 0; i < DT; ++i)
      if (16 * i + 4 * g < a.head_dim)
        *reinterpret_cast<float4 *>(o + 16 * i + 4 * g) =
            make_float4(acc[i][0] * inv, acc[i][1] * inv, acc[i][2] * inv, acc[i][3] * inv);
    return;
  }
  float *p = part + ((int64_t)it.slot * a.kv_heads + head) * (16 * (HDP + 2));
#pragma unroll
  for (int i = 0; i < DT; ++i)
    *reinterpret_cast<floatx4 *>(p + c * HDP + 16 * i + 4 * g) = acc[i];
  if (g == 0) {
    p[16 * HDP + c] = M;
    p[16 * HDP + 16 + c] = l;
  }
}

// Split rows: workgroup (tile, KV head) adds up the tile's partial states in
// the order of their keys.
template <int HDP>
__device__ __forceinline__ void join_body(const KvArgs &a, const JoinItem *items, const float *part, float *O,
                                          int64_t os) {
  const JoinItem it = items[blockIdx.x / a.kv_heads];
  const int head = (int)(blockIdx.x % a.kv_heads);
  const int64_t step = (int64_t)a.kv_heads * (16 * (HDP + 2));
  const float *p = part + ((int64_t)it.slot * a.kv_heads + head) * (16 * (HDP + 2));
  for (int i = threadIdx.x; i < 16 * HDP / 4; i += 256) {
    const int c = i / (HDP / 4), d = 4 * (i % (HDP / 4));
    const int r = it.tile * 16 + c, tok = r / a.groups;
    if (tok >= it.count || d >= a.head_dim) continue;
    float M = NONE, l = 0.f;
    for (int k = 0; k < it.n; ++k) M = fmaxf(M, p[k * step + 16 * HDP + c]);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < it.n; ++k) {
      const float f = __builtin_amdgcn_exp2f(p[k * step + 16 * HDP + c] - M);
      const float4 v = *reinterpret_cast<const float4 *>(p + k * step + c * HDP + d);
      l = fmaf(p[k * step + 16 * HDP + 16 + c], f, l);
      o.x = fmaf(v.x, f, o.x); o.y = fmaf(v.y, f, o.y);
      o.z = fmaf(v.z, f, o.z); o.w = fmaf(v.w, f, o.w);
    }
    const float inv = 1.f / l;
    *reinterpret_cast<float4 *>(O + ((int64_t)it.row0 + tok) * os +
                                (int64_t)(head * a.groups + r % a.groups) * a.head_dim + d) =
        make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  }
}

}  // namespace

// cos and sin of every position's angles, [position][pair].
extern "C" __global__ void __launch_bounds__(256)
pbx_kv_rope_table(const double *freq, double *table, int half, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  double s, c;
  sincos((double)(i / half) * freq[i % half], &s, &c);
  table[2 * i] = c;
  table[2 * i + 1] = s;
}

#define PBX_KV_KERNELS(HDP)                                                                                        \
  extern "C" __global__ void __launch_bounds__(256)                                                                \
      pbx_kv_append_##HDP(KvArgs a, KvRope r, const BlockItem *items, int n_blocks, const int *row_pos,            \
                          int n_rows, const float *K, int64_t ks, const float *V, int64_t vs, const float *Q,      \
                          int64_t qs, float *Qout, int64_t qos) {                                                  \
    append_body<HDP>(a, r, items, n_blocks, row_pos, n_rows, K, ks, V, vs, Q, qs, Qout, qos);                      \
  }                                                                                                                \
  extern "C" __global__ void __launch_bounds__(256)                                                                \
      pbx_kv_read_##HDP(KvArgs a, const BlockItem *items, float *K, int64_t ks, float *V, int64_t vs) {            \
    read_body<HDP>(a, items, K, ks, V, vs);                                                                        \
  }                                                                                                                \
  extern "C" __global__ void __launch_bounds__(256)                                                                \
      pbx_kv_attn_##HDP(KvArgs a, const AttnItem *items, const int *table, const float *Q, int64_t qs,             \
                        float scale, float *O, int64_t os, float *part) {                                          \
    attn_body<HDP>(a, items, table, Q, qs, scale, O, os, part);                                                    \
  }                                                                                                                \
  extern "C" __global__ void __launch_bounds__(256)                                                                \
      pbx_kv_join_##HDP(KvArgs a, const JoinItem *items, const float *part, float *O, int64_t os) {                \
    join_body<HDP>(a, items, part, O, os);                                                                         \
  }
PBX_KV_KERNELS(32)
PBX_KV_KERNELS(64)
PBX_KV_KERNELS(96)
PBX_KV_KERNELS(128)
PBX_KV_KERNELS(192)
PBX_KV_KERNELS(256)
