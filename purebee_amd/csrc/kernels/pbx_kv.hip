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
// kv_block_item and kv_attn_item of pbx_kv_plan.h
struct BlockItem {
  int page, sub, pos0, start, count, row0, pad[2];
};
struct AttnItem {
  int start, count, row0, tile, blk0, blk1, tab, part, parts, slot, join, pad, pages[4];
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

// x / s rounded half to even, as the true quotient.  In f32, x * (1 / s) of at
// most 128 is off it by less than 2^-15, so only quotients nearer than 10^-4 to
// a border (one in 5,000) need the division.  A turned pair may be past f32's
// range though both its keys are in it: q is then infinite, its distance from r a
// NaN, and the comparison, which holds for no NaN, leaves the division to it too.
__device__ __forceinline__ int code_of(double x, double s, float inv) {
  if (!(s > 0.0 && s < INFINITY)) return 0;
  const float q = (float)x * inv;
  float r = rintf(q);
  if (!(fabsf(fabsf(q - r) - 0.5f) >= 1e-4f)) r = (float)rint(x / s);
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
// cos and sin of unit u's two pairs at position pos.
struct Angles {
  double2 p, q;
};
__device__ __forceinline__ Angles angles_of(const KvRope &r, int u, int pos) {
  if (4 * u >= r.dim) return {make_double2(1.0, 0.0), make_double2(1.0, 0.0)};
  const double2 *cs = reinterpret_cast<const double2 *>(r.table) + (size_t)pos * (r.dim / 2) + 2 * u;
  return {cs[0], cs[1]};
}
// Turns unit u: x[0..1] at dims a, a + 1, x[2..3] at b, b + 1.
__device__ __forceinline__ void turn(const KvRope &r, int u, const Angles &cs, double x[4]) {
  if (4 * u >= r.dim) return;
  const double x0 = x[0], x1 = x[1], x2 = x[2], x3 = x[3];
  if (r.style == 2) {
    x[0] = x0 * cs.p.x - x2 * cs.p.y;
    x[2] = x0 * cs.p.y + x2 * cs.p.x;
    x[1] = x1 * cs.q.x - x3 * cs.q.y;
    x[3] = x1 * cs.q.y + x3 * cs.q.x;
  } else {
    x[0] = x0 * cs.p.x - x1 * cs.p.y;
    x[1] = x0 * cs.p.y + x1 * cs.p.x;
    x[2] = x2 * cs.q.x - x3 * cs.q.y;
    x[3] = x2 * cs.q.y + x3 * cs.q.x;
  }
}

// Append: workgroup (block, KV head), then a workgroup for each row's queries.
// The block's new rows are read once, keys turned, and held in registers (keys
// by 4 dims, values by 4 positions, as their codes lie side by side); the
// block's codes are put together in LDS (with the earlier rows' codes, if there
// are any) and stored whole.  Bound by bytes where there are many rows (6,124 of
// six prompts, 32 / 8 heads of 128: 60 us, 4.4 TB/s of queries in and out, keys,
// values and codes), else by one chain of loads, maximum, LDS and store: 32 / 8
// heads of 64, one row 4.7 us and 64 of 64 sequences 5.6 where no scale rises (the
// same rows again), 5.4 and 7.4 at new positions, of which most blocks round some
// earlier codes again, 6.5 and 7.9 where every row raises its block's scale.
// Threads of a workgroup: two units each (a wide head's block on 256 threads took
// three times as long where there are few).
constexpr int append_threads(int hdp) { return hdp <= 64 ? 256 : 4 * hdp; }

template <int HDP>
__device__ __forceinline__ void append_body(const KvArgs &a, const KvRope &r, const BlockItem *items,
                                            int n_blocks, const int *row_pos, const float *K,
                                            int64_t ks, const float *V, int64_t vs, const float *Q, int64_t qs,
                                            float *Qout, int64_t qos) {
  constexpr int T = append_threads(HDP), UNITS = BLK * HDP / 4 / T;  // a thread's units of a block
  __shared__ __attribute__((aligned(16))) uint8_t img[2 * BLK * HDP];
  __shared__ uint64_t red_k[T / 64];
  __shared__ unsigned red_v[T / 64];
  const int units = a.head_dim / 4, tid = threadIdx.x;
  const int64_t wg = blockIdx.x;
  if (wg >= (int64_t)n_blocks * a.kv_heads) {
    const int64_t row = wg - (int64_t)n_blocks * a.kv_heads;
    const int n = a.kv_heads * a.groups * units, pos = row_pos[row];
    const float *q = Q + row * qs;
    float *o = Qout + row * qos;
    // four units at a time, all read before any is written (in place, too: a unit
    // is read and written by one thread); with a power of two of units a head a
    // thread meets the same angles in every head
    const bool same = T % units == 0;
    Angles cs = angles_of(r, tid % units, pos);
    for (int i0 = tid; i0 < n; i0 += 4 * T) {
      float2 x[4][2];
      int at[4][2];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = min(i0 + T * k, n - 1), u = i % units, h = 4 * (i - u);  // h: the head's first dim
        unit_dims(r, u, at[k][0], at[k][1]);
        at[k][0] += h;
        at[k][1] += h;
        x[k][0] = *reinterpret_cast<const float2 *>(q + at[k][0]);
        x[k][1] = *reinterpret_cast<const float2 *>(q + at[k][1]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = i0 + T * k, u = i % units;
        if (i >= n) break;
        if (!same) cs = angles_of(r, u, pos);
        double y[4] = {x[k][0].x, x[k][0].y, x[k][1].x, x[k][1].y};
        turn(r, u, cs, y);
        *reinterpret_cast<float2 *>(o + at[k][0]) = make_float2((float)y[0], (float)y[1]);
        *reinterpret_cast<float2 *>(o + at[k][1]) = make_float2((float)y[2], (float)y[3]);
      }
    }
    return;
  }
  const BlockItem it = items[wg / a.kv_heads];
  const int head = (int)(wg % a.kv_heads);
  const int64_t bi = block_index(a, it.page, head, it.sub);
  uint8_t *codes = a.codes + bi * (2 * BLK * HDP);
  // rows lo .. hi - 1 of the block are new, those before lo were there
  const int lo = it.start > it.pos0 ? it.start - it.pos0 : 0;
  const int hi = min(BLK, it.start + it.count - it.pos0);
  const int64_t row0 = (int64_t)it.row0 + it.pos0 - it.start;  // of the block's first position
  K += row0 * ks + (int64_t)head * a.head_dim;
  V += row0 * vs + (int64_t)head * a.head_dim;
  const int nk_units = (hi - lo) * units;
  const int v0 = lo / 4, nv_units = ((hi + 3) / 4 - v0) * a.head_dim;
  double xk[UNITS][4];
  float xv[UNITS][4];
  uint64_t pk = 0;
  unsigned pv = 0;
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    const int j = tid + T * i;
    if (j < nv_units) {
      const int key = 4 * (v0 + j / a.head_dim), d = j % a.head_dim;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // (a quad's positions that are not new load one that is)
        const float x = V[min(max(key + e, lo), hi - 1) * vs + d];
        xv[i][e] = x;
        pv = max(pv, __float_as_uint(x) & 0x7fffffffu);
      }
    }
    if (j < nk_units) {
      const int key = lo + j / units, u = j % units;
      int da, db;
      unit_dims(r, u, da, db);
      const float2 k0 = *reinterpret_cast<const float2 *>(K + key * ks + da);
      const float2 k1 = *reinterpret_cast<const float2 *>(K + key * ks + db);
      xk[i][0] = k0.x; xk[i][1] = k0.y; xk[i][2] = k1.x; xk[i][3] = k1.y;
      turn(r, u, angles_of(r, u, it.pos0 + key), xk[i]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t mk = magnitude(xk[i][e]);
        pk = mk > pk ? mk : pk;
      }
    }
  }
  float ok = 0.f, ov = 0.f;
  if (lo > 0) {
    ok = a.scales[2 * bi];
    ov = a.scales[2 * bi + 1];
    for (int i = tid; i < 2 * BLK * HDP / 16; i += T)
      reinterpret_cast<uintx4 *>(img)[i] = reinterpret_cast<const uintx4 *>(codes)[i];
  } else if (hi < BLK || a.head_dim < HDP) {
    for (int i = tid; i < 2 * BLK * HDP / 4; i += T) reinterpret_cast<unsigned *>(img)[i] = 0x80808080u;
  }
  pk = wave_max_u64(pk);
#pragma unroll
  for (int off = 32; off >= 1; off /= 2) pv = max(pv, (unsigned)__shfl_xor((int)pv, off, 64));
  if ((tid & 63) == 0) {
    red_k[tid >> 6] = pk;
    red_v[tid >> 6] = pv;
  }
  __syncthreads();  // (and the image is filled)
#pragma unroll
  for (int w = 0; w < T / 64; ++w) {
    pk = red_k[w] > pk ? red_k[w] : pk;
    pv = max(pv, red_v[w]);
  }
  const float nk = larger(ok, scale_of(pk)), nv = larger(ov, scale_of(magnitude((double)__uint_as_float(pv))));
  const float ik = 1.f / nk, iv = 1.f / nv;
  if (lo > 0) {
    const bool gk = __float_as_uint(nk) != __float_as_uint(ok), gv = __float_as_uint(nv) != __float_as_uint(ov);
    if (gk || gv) {
      for (int i = tid; i < lo * HDP; i += T) {
        const int key = i / HDP, dim = i % HDP;
        uint8_t *pkb = img + key_byte<HDP>(key, dim), *pvb = img + BLK * HDP + value_byte(key, dim);
        if (gk) *pkb = (uint8_t)(code_of((double)((int)*pkb - 128) * (double)ok, nk, ik) + 128);
        if (gv) *pvb = (uint8_t)(code_of((double)((int)*pvb - 128) * (double)ov, nv, iv) + 128);
      }
      __syncthreads();  // a quad of values below may hold earlier positions' codes
    }
  }
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    const int j = tid + T * i;
    if (j < nk_units) {
      const int key = lo + j / units, u = j % units;
      int da, db;
      unit_dims(r, u, da, db);
      unsigned w = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) w |= (unsigned)(code_of(xk[i][e], nk, ik) + 128) << (8 * e);
      *reinterpret_cast<uint16_t *>(img + key_byte<HDP>(key, da)) = (uint16_t)w;
      *reinterpret_cast<uint16_t *>(img + key_byte<HDP>(key, db)) = (uint16_t)(w >> 16);
    }
    if (j < nv_units) {
      const int key = 4 * (v0 + j / a.head_dim), d = j % a.head_dim;
      uint8_t *at = img + BLK * HDP + value_byte(key, d);
      unsigned w = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) w |= (unsigned)(code_of(xv[i][e], nv, iv) + 128) << (8 * e);
      if (key >= lo && key + 4 <= hi) {
        *reinterpret_cast<unsigned *>(at) = w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (key + e >= lo && key + e < hi) at[e] = (uint8_t)(w >> (8 * e));
      }
    }
  }
  __syncthreads();
  for (int i = tid; i < 2 * BLK * HDP / 16; i += T)
    reinterpret_cast<uintx4 *>(codes)[i] = reinterpret_cast<const uintx4 *>(img)[i];
  if (tid == 0) *reinterpret_cast<float2 *>(a.scales + 2 * bi) = make_float2(nk, nv);
}

// Reading back: workgroup (block, KV head); the codes by way of LDS, where single
// bytes are cheap.  Bound by bytes (the rows above: 14 us, 4.4 TB/s).
template <int HDP>
__device__ __forceinline__ void read_body(const KvArgs &a, const BlockItem *items, float *K, int64_t ks, float *V,
                                          int64_t vs) {
  constexpr int T = append_threads(HDP);
  __shared__ __attribute__((aligned(16))) uint8_t img[2 * BLK * HDP];
  const BlockItem it = items[blockIdx.x / a.kv_heads];
  const int head = (int)(blockIdx.x % a.kv_heads);
  const int64_t bi = block_index(a, it.page, head, it.sub);
  const uint8_t *codes = a.codes + bi * (2 * BLK * HDP);
  const float sk = a.scales[2 * bi], sv = a.scales[2 * bi + 1];
  for (int i = threadIdx.x; i < 2 * BLK * HDP / 16; i += T)
    reinterpret_cast<uintx4 *>(img)[i] = reinterpret_cast<const uintx4 *>(codes)[i];
  __syncthreads();
  const int lo = it.start > it.pos0 ? it.start - it.pos0 : 0;
  const int hi = min(BLK, it.start + it.count - it.pos0);
  const int units = a.head_dim / 4;
  for (int j = threadIdx.x; j < (hi - lo) * units; j += T) {
    const int key = lo + j / units, d = 4 * (j % units);
    const int64_t row = (int64_t)it.row0 + it.pos0 + key - it.start;
    if (K) {
      const unsigned w = *reinterpret_cast<const unsigned *>(img + key_byte<HDP>(key, d));
      *reinterpret_cast<float4 *>(K + row * ks + (int64_t)head * a.head_dim + d) =
          make_float4(((int)(w & 255) - 128) * sk, ((int)(w >> 8 & 255) - 128) * sk,
                      ((int)(w >> 16 & 255) - 128) * sk, ((int)(w >> 24) - 128) * sk);
    }
    if (V) {
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (img[BLK * HDP + value_byte(key, d + e)] - 128) * sv;
      *reinterpret_cast<float4 *>(V + row * vs + (int64_t)head * a.head_dim + d) =
          make_float4(v[0], v[1], v[2], v[3]);
    }
  }
}

// kv_pack_item, kv_pack_row and kv_page_copy of pbx_kv_plan.h
struct PackItem {
  int page, sub, pos0, rows, at, raw, pad[2];
};
struct PackRow {
  int page, pos;
};
struct PageCopy {
  int from, to, blocks, pad;
};
struct KvPack {
  uint8_t *codes;  // of layer 0
  float *scales;
  int64_t layer_codes, layer_scales;
  const void *items;
  const PackRow *rows;
  int n_items, kv_heads, head_dim, page_shift;  // (copying: head_dim is a block's bytes)
};

__device__ __forceinline__ int64_t block_index(const KvPack &a, int page, int head, int sub) {
  return (((int64_t)page * a.kv_heads + head) << a.page_shift) + sub;
}

// Compaction: workgroup (layer, block of new rows, some KV heads).  A block's rows come
// from up to 32 old blocks; each code stands for code * s, keys turn back by the distance
// that they move down, and the block is coded as a new one is, quotients and largest
// magnitude as in 64 bits.  Both are looked for in f32 first: a magnitude is off by less
// than 2^-18 of the largest, a quotient of at most 127 by less than 10^-4, so only what
// comes as near to the largest, or to a border between codes, is computed in 64 bits.
// A row's keys lie side by side and are fetched as they are.  Its values lie 64 bytes
// apart for consecutive dims, so one row takes as many cache lines as the whole block:
// the blocks' values are fetched whole, PACK_BLOCKS at a time, into LDS, where the 64
// bytes of a dim take 68, so that dims fall in banks of their own.
// Half of 30,600 positions, kept here and there, 8 KV heads of 128, two layers: 109 us,
// where the codes read and written (156 MB) take 32; vector instructions fill 60% of the
// issue slots, and a workgroup waits for its chain of list, scales, codes and largest
// magnitudes.  A window of 1,000 of 5,000 positions, heads of 64: 8 us.
constexpr int PACK_BLOCKS = 4;
constexpr int pack_threads(int hdp) { return hdp <= 64 ? 256 : 2 * hdp; }
__device__ __forceinline__ int spread_byte(int key, int dim) {
  const int slot = 8 * ((key >> 2) & 3) + 4 * (key >> 4) + (key & 3);
  return (dim >> 5) * 1088 + (dim & 15) * 68 + (slot >> 3) * 16 + ((dim >> 4) & 1) * 8 + (slot & 7);
}
constexpr float LARGEST = 3.402823466e38f, NEAR_LARGEST = 1.f - 0x1p-17f, NEAR_BORDER = 2e-4f;

// y / s rounded half to even from q, which is it in f32 to 10^-4: where q is near the
// border k + 1/2, by 2 |y| against (2 k + 1) s, which are exact.
__device__ __forceinline__ float border_code(double y, float s, float q) {
  const float k = floorf(fabsf(q));
  if (fabsf(fabsf(q) - k - 0.5f) >= NEAR_BORDER) return rintf(q);
  const double t = (double)(2.f * k + 1.f) * (double)s, z = 2.0 * fabs(y);
  const float up = k + 1.f, r = z > t ? up : z < t ? k : ((int)k & 1 ? up : k);
  return copysignf(r, q);
}

template <int HDP>
__device__ __forceinline__ void pack_body(const KvPack &a, const KvRope &r) {
  constexpr int T = pack_threads(HDP), UNITS = BLK * HDP / 4 / T, BYTES = 2 * BLK * HDP, QUADS = HDP / 4;
  constexpr int SPREAD = HDP / 32 * 1088;  // a block's values in LDS
  __shared__ __attribute__((aligned(16))) uint8_t img[BYTES];
  __shared__ __attribute__((aligned(16))) unsigned val[PACK_BLOCKS * SPREAD / 4];
  __shared__ float red[2][T / 64];
  __shared__ uint64_t red_exact[2];
  __shared__ int64_t src[BLK], of[BLK];  // the rows' old blocks; the different ones among them
  __shared__ int val_at[BLK], nth[BLK];  // a row's place in an old block's values; which of the different ones
  __shared__ float sk[BLK], sv[BLK];
  __shared__ unsigned bads;  // rows of blocks that read as NaN: 1 keys, 2 values
  const int tid = threadIdx.x;
  const int per_layer = a.n_items * a.kv_heads;
  const int layer = blockIdx.x / per_layer, in_layer = blockIdx.x % per_layer;
  const PackItem it = reinterpret_cast<const PackItem *>(a.items)[in_layer / a.kv_heads];
  const int head = in_layer % a.kv_heads;
  uint8_t *codes = a.codes + layer * a.layer_codes;
  float *scales = a.scales + layer * a.layer_scales;
  const int64_t bi = block_index(a, it.page, head, it.sub);
  if (it.raw >= 0) {
    const int64_t from = block_index(a, it.raw, head, it.sub);
    for (int i = tid; i < BYTES / 16; i += T)
      reinterpret_cast<uintx4 *>(codes + bi * BYTES)[i] = reinterpret_cast<const uintx4 *>(codes + from * BYTES)[i];
    if (tid == 0) *reinterpret_cast<float2 *>(scales + 2 * bi) = *reinterpret_cast<const float2 *>(scales + 2 * from);
    return;
  }
  // unit i of a thread: 4 dims of row kw (keys), 4 rows from vw on at dim vd (values)
  auto kw = [&](int i) { return (tid + T * i) / QUADS; };
  auto ku = [&](int i) { return (tid + T * i) % QUADS; };
  auto vw = [&](int i) { return (tid + T * i) / HDP * 4; };
  auto vd = [&](int i) { return (tid + T * i) % HDP; };
  int pos[UNITS];
  bool kon[UNITS], von[UNITS];
  float cs[UNITS][4];  // cos and sin of the unit's two pairs
  auto angles = [&](int i) {
    KvRope q = r;
    asm volatile("" : "+s"(q.table));  // read again where they are needed, not kept in registers
    Angles x = angles_of(q, ku(i), pos[i] - (it.pos0 + kw(i)));
    x.p.y = -x.p.y;
    x.q.y = -x.q.y;
    return x;
  };
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    kon[i] = kw(i) < it.rows && 4 * ku(i) < a.head_dim;
    von[i] = vw(i) < it.rows && vd(i) < a.head_dim;
    pos[i] = 0;
    if (!kon[i]) continue;
    pos[i] = a.rows[it.at + kw(i)].pos;
    const Angles x = angles(i);
    cs[i][0] = (float)x.p.x, cs[i][1] = (float)x.p.y, cs[i][2] = (float)x.q.x, cs[i][3] = (float)x.q.y;
  }
  if (tid < BLK) {
    const PackRow row = a.rows[it.at + min(tid, it.rows - 1)];  // (the last one again past the rows)
    const int64_t from = block_index(a, row.page, head, row.pos / BLK & ((1 << a.page_shift) - 1));
    // positions rise: a row is the first of its old block where the row before is of another
    const int blk = row.pos / BLK;
    const bool first = tid == 0 || __shfl_up(blk, 1) != blk;
    const unsigned firsts = (unsigned)__ballot(first);
    const int n = __popc(firsts & (0xFFFFFFFFu >> (31 - tid))) - 1;
    src[tid] = from;
    nth[tid] = n;
    val_at[tid] = spread_byte(row.pos % BLK, 0) + n % PACK_BLOCKS * SPREAD;
    if (first) of[n] = from;
    const float2 s = *reinterpret_cast<const float2 *>(scales + 2 * from);
    sk[tid] = s.x;
    sv[tid] = s.y;
    const unsigned any = (__ballot(!(s.x < INFINITY)) ? 1u : 0u) | (__ballot(!(s.y < INFINITY)) ? 2u : 0u);
    if (tid == 0) bads = any;
  }
  if (tid < 2) red_exact[tid] = 0;
  __syncthreads();
  unsigned kc[UNITS];
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    if (!kon[i]) continue;
    const uint8_t *from = codes + src[kw(i)] * BYTES;
    int da, db;
    unit_dims(r, ku(i), da, db);
    kc[i] = *reinterpret_cast<const uint16_t *>(from + key_byte<HDP>(pos[i] % BLK, da)) |
            (unsigned)*reinterpret_cast<const uint16_t *>(from + key_byte<HDP>(pos[i] % BLK, db)) << 16;
  }
  if (it.rows < BLK || a.head_dim < HDP)
    for (int i = tid; i < BYTES / 4; i += T) reinterpret_cast<unsigned *>(img)[i] = 0x80808080u;
  const int blocks = nth[BLK - 1] + 1;
  float vc[UNITS][4];  // codes
  for (int b0 = 0; b0 < blocks; b0 += PACK_BLOCKS) {
    if (b0) __syncthreads();  // the blocks before have been read
    const int here = min(PACK_BLOCKS, blocks - b0);
#pragma unroll
    for (int i = 0; i < (PACK_BLOCKS * HDP * 2 + T - 1) / T; ++i) {
      const int c = tid + T * i, blk = c / (2 * HDP), at = c % (2 * HDP);  // 16-byte pieces
      if (blk < here) {
        const uintx4 x = reinterpret_cast<const uintx4 *>(codes + of[b0 + blk] * BYTES + BLK * HDP)[at];
        unsigned *y = val + blk * (SPREAD / 4) + (at >> 6) * 272 + (at >> 2 & 15) * 17 + (at & 3) * 4;
        y[0] = x.x, y[1] = x.y, y[2] = x.z, y[3] = x.w;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      const uint8_t *at = reinterpret_cast<const uint8_t *>(val) + spread_byte(0, vd(i));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int w = vw(i) + e;
        const float c = (float)at[val_at[w]] - 128.f;
        if (blocks <= PACK_BLOCKS || (nth[w] >= b0 && nth[w] < b0 + PACK_BLOCKS)) vc[i][e] = c;
      }
    }
  }
  // largest magnitudes in f32 (of numbers: a row of a block that reads as NaN is seen to below)
  float xk[UNITS][4], pk[UNITS], pv[UNITS], mk = 0.f, mv = 0.f;
  auto most4 = [](const float x[4]) { return fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))); };
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    pk[i] = pv[i] = 0.f;
    if (kon[i]) {
      const float c0 = (float)(kc[i] & 255) - 128.f, c1 = (float)(kc[i] >> 8 & 255) - 128.f;
      const float c2 = (float)(kc[i] >> 16 & 255) - 128.f, c3 = (float)(kc[i] >> 24) - 128.f, s = sk[kw(i)];
      // the pairs are (0, 2) and (1, 3) where halves turn, else (0, 1) and (2, 3)
      const bool halves = r.style == 2;
      const float d1 = halves ? c2 : c1, d2 = halves ? c1 : c2;
      const float y0 = (c0 * cs[i][0] - d1 * cs[i][1]) * s, y1 = (c0 * cs[i][1] + d1 * cs[i][0]) * s;
      const float y2 = (d2 * cs[i][2] - c3 * cs[i][3]) * s, y3 = (d2 * cs[i][3] + c3 * cs[i][2]) * s;
      xk[i][0] = y0, xk[i][1] = halves ? y2 : y1, xk[i][2] = halves ? y1 : y2, xk[i][3] = y3;
      pk[i] = most4(xk[i]);
      mk = fmaxf(mk, pk[i]);
    }
    if (von[i]) {
#pragma unroll
      for (int e = 0; e < 4; ++e) vc[i][e] *= sv[vw(i) + e];  // (from here on values, to a rounding)
      pv[i] = most4(vc[i]);
      mv = fmaxf(mv, pv[i]);
    }
  }
  mk = wave_max(mk);
  mv = wave_max(mv);
  if ((tid & 63) == 0) {
    red[0][tid >> 6] = mk;
    red[1][tid >> 6] = mv;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < T / 64; ++w) {
    mk = fmaxf(mk, red[0][w]);
    mv = fmaxf(mv, red[1][w]);
  }
  // (127 times the scale of f32's largest number rounds past it)
  if (!(mv < INFINITY)) {
    mv = LARGEST;
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      pv[i] = fminf(pv[i], LARGEST);
#pragma unroll
      for (int e = 0; e < 4; ++e) vc[i][e] = fminf(fmaxf(vc[i][e], -LARGEST), LARGEST);
    }
  }
  auto exact_keys = [&](int i, double x[4]) {
    const double s = sk[kw(i)];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = (double)((int)(kc[i] >> (8 * e) & 255) - 128) * s;
    turn(r, ku(i), angles(i), x);
  };
  // (the code again, as a product of at most 127 and s is off by a rounding)
  auto exact_value = [&](int i, int e) {
    const float s = sv[vw(i) + e];
    return s > 0.f ? (double)rintf(vc[i][e] / s) * (double)s : 0.0;
  };
  // what may be the largest, in 64 bits
  const float near_k = fminf(mk, LARGEST) * NEAR_LARGEST, near_v = mv * NEAR_LARGEST;
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    if (mk > 0.f && pk[i] >= near_k) {
      double x[4];
      exact_keys(i, x);
      atomicMax((unsigned long long *)&red_exact[0],
                magnitude(fmax(fmax(fabs(x[0]), fabs(x[1])), fmax(fabs(x[2]), fabs(x[3])))));
    }
    if (mv > 0.f && pv[i] >= near_v) {
      double x = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) x = fmax(x, fabs(exact_value(i, e)));
      atomicMax((unsigned long long *)&red_exact[1], magnitude(x));
    }
  }
  __syncthreads();
  const float none = __uint_as_float(0x7fc00000u);
  const float nk = bads & 1 ? none : scale_of(red_exact[0]), nv = bads & 2 ? none : scale_of(red_exact[1]);
  const bool ok_k = nk > 0.f && nk < INFINITY, ok_v = nv > 0.f && nv < INFINITY;  // else codes are 0
  const float ik = ok_k ? 1.f / nk : 0.f, iv = ok_v ? 1.f / nv : 0.f;
  // codes of 4 quotients + 128; how far the nearest one is from a border
  auto code4 = [](const float x[4], float inv, unsigned &w) {
    float gap = 1.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float q = x[e] * inv;
      gap = fminf(gap, fabsf(__builtin_amdgcn_fractf(q) - 0.5f));
      w = __builtin_amdgcn_cvt_pk_u8_f32(rintf(q) + 128.f, e, w);
    }
    return gap;
  };
  auto mend = [](unsigned w, int e, float code) {
    return (w & ~(255u << (8 * e))) | (unsigned)((int)code + 128) << (8 * e);
  };
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    if (kon[i]) {
      unsigned w = 0;
      // (past f32's range nothing above holds)
      if (code4(xk[i], ik, w) < NEAR_BORDER || !(mk < INFINITY)) {
        double x[4];
        exact_keys(i, x);
#pragma unroll 1
        for (int e = 0; e < 4; ++e) {
          const double y = e == 0 ? x[0] : e == 1 ? x[1] : e == 2 ? x[2] : x[3];
          w = mend(w, e, (float)rint(y / (double)nk));
        }
      }
      if (!ok_k) w = 0x80808080u;
      int da, db;
      unit_dims(r, ku(i), da, db);
      *reinterpret_cast<uint16_t *>(img + key_byte<HDP>(kw(i), da)) = (uint16_t)w;
      *reinterpret_cast<uint16_t *>(img + key_byte<HDP>(kw(i), db)) = (uint16_t)(w >> 16);
    }
    if (von[i]) {
      unsigned w = 0;
      if (code4(vc[i], iv, w) < NEAR_BORDER) {
#pragma unroll
        for (int e = 0; e < 4; ++e) w = mend(w, e, border_code(exact_value(i, e), nv, vc[i][e] * iv));
      }
      if (!ok_v) w = 0x80808080u;
      const int rest = it.rows - vw(i);  // positions past the rows hold code 0
      if (rest < 4) w = (w & ((1u << (8 * rest)) - 1)) | 0x80808080u << (8 * rest);
      *reinterpret_cast<unsigned *>(img + BLK * HDP + value_byte(vw(i), vd(i))) = w;
    }
  }
  __syncthreads();
  for (int i = tid; i < BYTES / 16; i += T)
    reinterpret_cast<uintx4 *>(codes + bi * BYTES)[i] = reinterpret_cast<const uintx4 *>(img)[i];
  if (tid == 0) *reinterpret_cast<float2 *>(scales + 2 * bi) = make_float2(nk, nv);
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
// A row's probabilities in a block are taken against the block's own largest
// score, rounded up to a whole number of powers of two, and times 2^LIFT: an fp16
// pair then keeps 22 bits of them down to 2^-9 of the block's largest and resolves
// 2^-30 of it below (more would cost the exponentials' arguments bits).  The block
// joins the row's sums in f32 with its weight, a power of two, so keys far below
// the row's largest keep their bits and add up, however many they are.
// A row's maximum follows the blocks' only when they pass it by 2^SLACK: a new
// maximum rescales all sums, and in some row of a tile nearly every block brings one.
// (All of a row against one maximum took 2 to 4 % less on prompts of heads up to 128,
// as much elsewhere, and lost what lay below 2^-31 of it: a quarter of a tail of 4,000
// keys behind one strong one.)
// Scores past 2^28 (in powers of two) are so coarse in f32 that an exponent's rounding
// would leave fp16's range.
constexpr float LIFT = 6.f, SLACK = 12.f;

// Codes reach LDS by DMA (global_load_lds: lane i's 16 bytes land at the
// instruction's LDS base + 16 i), without registers in between; waits are
// counted by hand, so every wave issues the same number of them for a block.
// M0 is the compiler's own (no asm may name it as clobbered): it writes it right
// before each use, and nothing else in these kernels uses it.
__device__ __forceinline__ unsigned lds_address(const void *p) {
  return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) void *)p;
}
__device__ __forceinline__ void dma16(const uint8_t *base, unsigned offset, unsigned lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               ::"v"(offset), "s"(base), "s"(lds) : "memory");
}
// Waits until at most N of the wave's vector memory operations are under way.
template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// The wave's LDS reads so far have their values: what they read may be fetched over.
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// A constant that the compiler cannot see through.
__device__ __forceinline__ float opaque(float x) {
  asm("" : "+s"(x));
  return x;
}

// hi = fp16(x), lo = fp16(x - hi) of 8 values: a packed conversion for two, and a
// mixed-precision fma each, which a visible -1 would be taken out of (three
// instructions then).
__device__ __forceinline__ void split8(const float x[8], float minus_one, half8 &hi, half8 &lo) {
  typedef float float2t __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float2t v = {x[e], x[e + 1]};
    const half2t h = __builtin_convertvector(v, half2t);
    hi[e] = h[0];
    hi[e + 1] = h[1];
    lo[e] = (_Float16)fmaf((float)h[0], minus_one, x[e]);
    lo[e + 1] = (_Float16)fmaf((float)h[1], minus_one, x[e + 1]);
  }
}

// Partial results cross workgroups (and XCDs, whose L2 caches do not see each
// other's lines) inside a launch: stores and loads at the device's coherence
// point, 8 bytes each.
__device__ __forceinline__ void put2(float *p, float x, float y) {
  const uint64_t v = (uint64_t)__float_as_uint(y) << 32 | __float_as_uint(x);
  __hip_atomic_store(reinterpret_cast<uint64_t *>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get2(const float *p) {
  const uint64_t v =
      __hip_atomic_load(reinterpret_cast<const uint64_t *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float((unsigned)v), __uint_as_float((unsigned)(v >> 32)));
}

// Attention: workgroup (item, KV head), four waves that take the item's blocks
// in turn.  A wave holds NQ tiles of 16 query rows (token, head of the group),
// each as the columns of its products: scores S = K Q^T of 32 keys (two 16-key
// tiles), a softmax step whose maxima and sums stay within a column (lanes c,
// c + 16, c + 32, c + 48), and O^T += V^T P^T with P taken from the score
// registers as they lie.  Codes are exact in fp16; queries (divided by a power
// of two near the row's largest) and probabilities enter as fp16 pairs, two
// products each, summed in f32.  The block's key scale joins the row's factor,
// its value scale weighs the block's products as they are added up.
// Every wave keeps a ring of RING blocks' codes in LDS; a block is asked for
// RING - 1 blocks ahead (RING 1: its keys after the scores of the one before, its
// values after that one's).  The counted waits allow for what was asked for later,
// but the compiler adds one: `scales` may have just been loaded in a branch of the
// loop, and it waits for all vector memory before each block's use of them.  So
// whatever is under way as a block begins is waited for, the block fetched ahead
// (RING 3) or its own values (RING 1) too.
// Where a tile's blocks are split over several workgroups, the one that finishes
// last puts their states together, in the order of the keys.
// Single tokens are bound by the codes' bytes: 64 sequences of 64 to 8,000
// positions, 32 / 8 heads of 64, 58 us (4.97 TB/s); one of 131,001 positions 35 us
// (3.9 TB/s; with 96 or 128 parts for 64 it took 38 and 43); one of 129 4.9 us, a
// launch's.  Prompts are bound by issue: a vector instruction does not run beside a
// 16x16x32 product (a loop of 8 products and 32 fmas a wave, four waves a SIMD:
// 358 ns, the products alone 226, the fmas 142), and 32 rows times 32 keys of 64
// dims are 36 products (576 cycles) and about 275 vector instructions, so what
// counts is fewer of either: 2,000 rows, 32 / 8 heads of 64, 52 us (635 TFLOP/s
// of products); 1,183 rows on pasts of up to 2,000, 32 / 8 heads of 128, 96 us
// (760 TFLOP/s); 2,000 rows, 16 / 8 heads of 192, 76 us (650), 8 / 1 of 256, 60 us
// (540).  Clocks rise over the first 600 launches or so (the first 60 of these
// prompts take 60 and 114 us); the figures are those after.
template <int HDP, int NQ, int KW, int RING>
__device__ __forceinline__ void attn_body(const KvArgs &a, const AttnItem *items, const int *table, const float *Q,
                                          int64_t qs, float scale, float *O, int64_t os, float *part,
                                          unsigned *arrived) {
  constexpr int HC = HDP / 32, PAIRS = HDP / 64, DT = HDP / 16;
  constexpr int U = NQ * 4 / KW;        // 16-row tiles of the workgroup
  constexpr int UNIT = 16 * (HDP + 2);  // floats of 16 rows' partial state
  constexpr int HALF = BLK * HDP, NI = HALF / 1024;  // bytes of a block's keys (or values), DMA instructions for them
  constexpr int MERGE = 4 * NQ * DT * 1024, LDS = 4 * RING * 2 * HALF;
  // the waves' rings, and the merge of their states after them
  __shared__ __attribute__((aligned(16))) uint8_t lds[LDS > MERGE ? LDS : MERGE];
  static_assert(LDS >= 256 * 8 * 4, "room for the join's shares");
  // (in place, too: the merge's barriers stand between the waves' query reads and the stores)
  static_assert(KW > 1, "waves with the same rows, whose states are merged");
  float(*mrg)[NQ * DT][256] = reinterpret_cast<float(*)[NQ * DT][256]>(lds);
  __shared__ float mrg_m[4][NQ][16], mrg_l[4][NQ][16];
  __shared__ unsigned order;
  const AttnItem &it = items[blockIdx.x / a.kv_heads];
  const int head = (int)(blockIdx.x % a.kv_heads);
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int blk0 = it.blk0, blk1 = it.blk1, start = it.start, count = it.count, tile = it.tile;
  const int sub_mask = (1 << a.page_shift) - 1;
  const int tab = it.tab, parts = it.parts, row0 = it.row0;
  const int part_at = it.slot + it.part * U, slot0 = it.slot, join = it.join;
  auto block_at = [&](int page, int b) { return block_index(a, page, head, b & sub_mask); };
  // wave (qw, kw): query tiles qw NQ .., blocks b0, b0 + KW, ..: page ids one a lane, 64 at a time; the
  // first one's comes with the item
  const int qw = wave / KW, kw = wave % KW;
  // query row r of the workgroup: token first_tok + k and head of the group; the
  // quotient of numbers this small is exact in f32
  const int first_tok = tile * 16 * U / a.groups, skip = tile * 16 * U % a.groups;
  const float per_group = 1.f / (float)a.groups;
  auto token_of = [&](int r) { return (int)(((float)(skip + r) + 0.5f) * per_group); };
  const int rows = min(16 * U, count * a.groups - tile * 16 * U);  // that are there
  const int first_pos = start + (tile * 16 * U + 16 * NQ * qw) / a.groups;  // of the wave's rows
  const int b0 = blk0 + kw;
  const int n = 16 * NQ * qw < rows ? (blk1 - b0 + KW - 1) / KW : 0;  // <= 0: none
  // the larger of two raw products is their median with infinity: fmaxf puts a
  // canonicalising move before each (of numbers; a NaN travels with the sums)
  const float inf = opaque(INFINITY), minus_one = opaque(-1.f);
  uint8_t *ring = lds + wave * (RING * 2 * HALF);
  const unsigned ring_at = __builtin_amdgcn_readfirstlane((int)lds_address(ring));
  // lane (c, g) fetches what it reads: 64 dims' 16 g .. of key c of each tile,
  // or 16 bytes g of value dim c; the last 32 dims' keys as they lie
  const unsigned mine16 = c * 64 + 16 * g;
  auto fetch_keys = [&](const uint8_t *p, int slot) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
      dma16(p, i * 1024 + (i < 2 * PAIRS ? mine16 : 16u * lane), ring_at + slot * (2 * HALF) + i * 1024);
  };
  auto fetch_values = [&](const uint8_t *p, int slot) {
#pragma unroll
    for (int i = 0; i < NI; ++i) dma16(p, HALF + i * 1024 + mine16, ring_at + slot * (2 * HALF) + HALF + i * 1024);
  };
  // 64 blocks' places and scales from `base` on, one a lane; the first block's page comes
  // with the item, so its codes are on their way before the page table is read
  constexpr int AHEAD = RING > 1 ? RING - 1 : 1;
  int base = 0, slot = 0;
  int64_t place = 0;
  float2 scales = make_float2(0.f, 0.f);
  auto look_up = [&](int i) {
    const int b = min(b0 + KW * (i + lane), blk1 - 1);
    place = block_at(table[tab + (b >> a.page_shift)], b);
    scales = *reinterpret_cast<const float2 *>(a.scales + 2 * place);
  };
  auto codes_of = [&](int i) {
    const unsigned lo = __builtin_amdgcn_readlane((unsigned)place, i - base);
    const unsigned hi = __builtin_amdgcn_readlane((unsigned)(place >> 32), i - base);
    return a.codes + (int64_t)((uint64_t)hi << 32 | lo) * (2 * HALF);
  };
  if (n > 0) {
    const int j = (b0 >> a.page_shift) - (blk0 >> a.page_shift);
    const int page = j == 0 ? it.pages[0] : j == 1 ? it.pages[1] : j == 2 ? it.pages[2] : it.pages[3];
    const uint8_t *p = a.codes + block_at(page, b0) * (2 * HALF);
    fetch_keys(p, 0);
    fetch_values(p, 0);
    look_up(0);
#pragma unroll
    for (int i = 1; i < RING - 1; ++i)
      if (i < n) {
        fetch_keys(codes_of(i), i);
        fetch_values(codes_of(i), i);
      }
  }
  half8 qh[NQ][HC], ql[NQ][HC];
  float factor[NQ];  // of the products: the row's power of two, scale, log2(e)
  int pos[NQ];
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int r = 16 * (qw * NQ + q) + c, k = token_of(r), tok = first_tok + k;
    const bool live = r < rows;
    pos[q] = live ? start + tok : -1;
    // (rows past the end load the last one's: no load waits behind a branch)
    const float *src = Q + ((int64_t)row0 + min(tok, count - 1)) * qs +
                       (int64_t)(head * a.groups + skip + r - k * a.groups) * a.head_dim;
    float x[HC][8];
    unsigned peak = 0;
#pragma unroll
    for (int i = 0; i < HC; ++i)
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const int d = i < 2 * PAIRS ? 64 * (i >> 1) + 16 * g + 8 * (i & 1) + e : 32 * i + 8 * g + e;
        const bool in = live && d < a.head_dim;
        const float4 v = *reinterpret_cast<const float4 *>(src + min(d, a.head_dim - 4));
        x[i][e] = in ? v.x : 0.f; x[i][e + 1] = in ? v.y : 0.f;
        x[i][e + 2] = in ? v.z : 0.f; x[i][e + 3] = in ? v.w : 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) peak = max(peak, __float_as_uint(x[i][e + k]) & 0x7fffffffu);
      }
    peak = max(peak, (unsigned)__shfl_xor((int)peak, 16, 64));
    peak = max(peak, (unsigned)__shfl_xor((int)peak, 32, 64));
    const unsigned ex = min(max(peak >> 23, 1u), 253u);
    // 2^(127 - ex), with scale's sign so that the factor keeps the scores' order
    const float down = copysignf(__uint_as_float((254u - ex) << 23), scale);
    factor[q] = __uint_as_float(ex << 23) * (fabsf(scale) * 1.44269504f);
#pragma unroll
    for (int i = 0; i < HC; ++i) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] *= down;
      split8(x[i], minus_one, qh[q][i], ql[q][i]);
    }
  }
  const floatx4 zero = {0.f, 0.f, 0.f, 0.f};
  floatx4 acc[NQ][DT];
  float m[NQ], l[NQ];
  half8 ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) ones[e] = (_Float16)1.f;
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    m[q] = NONE;
    l[q] = 0.f;
#pragma unroll
    for (int i = 0; i < DT; ++i) acc[q][i] = zero;
  }
  for (int i = 0; i < n; ++i) {
    const int b = b0 + KW * i, ahead = i + AHEAD;
    if (ahead - base > 63) {
      look_up(i);
      base = i;
    }
    const float sk = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(scales.x), i - base));
    const float svb = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(scales.y), i - base));
    const uint8_t *next = codes_of(min(ahead, n - 1));
    const uint8_t *codes = ring + (RING > 1 ? slot * (2 * HALF) : 0);
    // the block is there when at most what was fetched after it is under way
    if (RING > 1 ? RING > 2 && ahead - 1 < n : i > 0)
      wait_vm<RING == 1 ? NI : (RING - 2) * 2 * NI>();
    else
      wait_vm<0>();
    if constexpr (RING > 1) {
      // into the slot of the block before, which has been read
      if (ahead < n) {
        wait_lds();
        const int to = slot ? slot - 1 : RING - 1;
        fetch_keys(next, to);
        fetch_values(next, to);
      }
      slot = slot + 1 < RING ? slot + 1 : 0;
    }
    floatx4 s[NQ][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int q = 0; q < NQ; ++q) s[q][t] = zero;
#pragma unroll
      for (int p = 0; p < HC; p += 2) {
        uintx4 w;
        if (p < 2 * PAIRS) {
          w = *reinterpret_cast<const uintx4 *>(codes + (p + t) * 1024 + 16 * lane);
        } else {
          const uintx2 x = *reinterpret_cast<const uintx2 *>(codes + 2 * PAIRS * 1024 + (16 * t + c) * 32 + 8 * g);
          w[0] = x[0];
          w[1] = x[1];
        }
#pragma unroll
        for (int j = 0; j < (p < 2 * PAIRS ? 2 : 1); ++j) {
          const half8 k = halves(w[2 * j], w[2 * j + 1]);
#pragma unroll
          for (int q = 0; q < NQ; ++q)
            s[q][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh[q][p + j], s[q][t], 0, 0, 0);
#pragma unroll
          for (int q = 0; q < NQ; ++q)
            s[q][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql[q][p + j], s[q][t], 0, 0, 0);
        }
      }
    }
    if constexpr (RING == 1) {
      wait_lds();
      if (ahead < n) fetch_keys(next, 0);
    }
    half8 ph[NQ], pl[NQ];
    float mn[NQ], sv[NQ], wt[NQ];
    bool moved = false;
    const bool whole = b * BLK + BLK - 1 <= first_pos;  // every live row sees the block
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      // never 0, so that masked scores stay -inf (a block of zeros has scale 0)
      float f = factor[q] * sk;
      f = f < 1e-30f ? 1e-30f : f;
      sv[q] = svb;
      if (!whole) {
        // a row that sees nothing of the block takes nothing of its scales either
        const bool none = b * BLK > pos[q];
        f = none ? 1e-30f : f;
        sv[q] = none ? 0.f : sv[q];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (b * BLK + 4 * g + 16 * (e >> 2) + (e & 3) > pos[q]) s[q][e >> 2][e & 3] = -INFINITY;
      }
      float mx = s[q][0][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) mx = __builtin_amdgcn_fmed3f(mx, s[q][e >> 2][e & 3], inf);
      mx = pair_max<32>(pair_max<16>(mx));
      // (a row that sees nothing of the block has -inf here)
      mx = __builtin_amdgcn_fmed3f(__builtin_ceilf(mx * f), NONE, inf);
      const bool up = mx > m[q] + SLACK;
      mn[q] = up ? mx : m[q];
      moved = moved || up;
      const float base = mx - LIFT;  // whole numbers: exact, as the weight is
      wt[q] = __builtin_amdgcn_exp2f(base - mn[q]);
      sv[q] *= wt[q];
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(s[q][e >> 2][e & 3], f, -base));
      split8(p, minus_one, ph[q], pl[q]);
    }
    if (__any(moved)) {
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        const float al = __builtin_amdgcn_exp2f(m[q] - mn[q]);
        m[q] = mn[q];
        l[q] *= al;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[q][d] *= al;
      }
    }
    floatx4 bl[NQ];  // a column's sum in every row: products with ones
#pragma unroll
    for (int q = 0; q < NQ; ++q) bl[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, ph[q], zero, 0, 0, 0);
#pragma unroll
    for (int q = 0; q < NQ; ++q) bl[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pl[q], bl[q], 0, 0, 0);
#pragma unroll
    for (int q = 0; q < NQ; ++q) l[q] = fmaf(bl[q][0], wt[q], l[q]);
    if constexpr (RING == 1) {
      if (ahead < n)
        wait_vm<NI>();
      else
        wait_vm<0>();
    }
#pragma unroll
    for (int h = 0; h < HC; ++h) {
      const uintx4 w = *reinterpret_cast<const uintx4 *>(codes + HALF + h * 1024 + 16 * lane);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const half8 v = halves(w[2 * j], w[2 * j + 1]);
        floatx4 o[NQ];
#pragma unroll
        for (int q = 0; q < NQ; ++q) o[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph[q], zero, 0, 0, 0);
#pragma unroll
        for (int q = 0; q < NQ; ++q) o[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl[q], o[q], 0, 0, 0);
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[q][2 * h + j][e] = fmaf(o[q][e], sv[q], acc[q][2 * h + j][e]);
      }
    }
    if constexpr (RING == 1) {
      wait_lds();
      if (ahead < n) fetch_values(next, 0);
    }
  }
  // the states of the waves with the same rows put together: one maximum, then
  // the sums, each wave a share of the 16 x 16 output tiles
#pragma unroll
  for (int q = 0; q < NQ; ++q)
    if (g == 0) mrg_m[wave][q][c] = m[q];
  __syncthreads();  // (and every wave is done with its ring)
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    float M = mrg_m[qw * KW][q][c];
#pragma unroll
    for (int w = 1; w < KW; ++w) M = fmaxf(M, mrg_m[qw * KW + w][q][c]);
    const float f = __builtin_amdgcn_exp2f(m[q] - M);
    if (g == 0) mrg_l[wave][q][c] = l[q] * f;
    m[q] = M;
#pragma unroll
    for (int d = 0; d < DT; ++d)
      *reinterpret_cast<floatx4 *>(&mrg[wave][q * DT + d][4 * lane]) = acc[q][d] * f;
  }
  __syncthreads();
  auto out_row = [&](int r) {
    const int k = token_of(r);
    return O + ((int64_t)row0 + first_tok + k) * os + (int64_t)(head * a.groups + skip + r - k * a.groups) * a.head_dim;
  };
  float *mine = part + ((int64_t)part_at * a.kv_heads + head * U) * UNIT;
#pragma unroll
  for (int u = 0; u < NQ * DT; ++u) {
    if (u % KW != kw) continue;
    const int q = u / DT, d = 16 * (u % DT) + 4 * g, r = 16 * (qw * NQ + q) + c;
    floatx4 o = zero;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      o += *reinterpret_cast<const floatx4 *>(&mrg[qw * KW + w][u][4 * lane]);
      sum += mrg_l[qw * KW + w][q][c];
    }
    if (r >= rows) continue;
    if (parts > 1) {
      float *p = mine + (qw * NQ + q) * UNIT;
      put2(p + c * HDP + d, o[0], o[1]);
      put2(p + c * HDP + d + 2, o[2], o[3]);
      if (u % DT == 0 && g == 0) put2(p + 16 * HDP + 2 * c, m[q], sum);
    } else if (d < a.head_dim) {
      const float inv = 1.f / sum;
      *reinterpret_cast<float4 *>(out_row(r) + d) =
          make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
    }
  }
  if (parts == 1) return;
  // this part's state is at the coherence point before its workgroup counts
  // itself in; the workgroup that completes the count reads the others' from there
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0)
    order = __hip_atomic_fetch_add(&arrived[32 * (join * a.kv_heads + head)], 1u, __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (order != (unsigned)parts - 1) return;
  if (threadIdx.x == 0)
    __hip_atomic_store(&arrived[32 * (join * a.kv_heads + head)], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const int64_t step = (int64_t)a.kv_heads * U * UNIT;  // from part to part
  const float *first = part + ((int64_t)slot0 * a.kv_heads + head * U) * UNIT;
  // unit: four dims of a row; the parts in `ways` shares where there are few
  // units.  Eight parts' loads are under way at once: they come from the
  // coherence point, one round trip after the other took 14 us for 64 parts
  const int units = rows * (HDP / 4);
  int ways = 1;
  while (ways < 16 && 2 * ways * units <= 256) ways *= 2;
  float(*shares)[8] = reinterpret_cast<float(*)[8]>(lds);
  for (int u0 = 0; u0 < units; u0 += 256 / ways) {
    const int u = u0 + (int)threadIdx.x / ways, way = (int)threadIdx.x % ways;
    const int r = min(u, units - 1) / (HDP / 4), d = 4 * (min(u, units - 1) % (HDP / 4));
    float M = NONE, sum = 0.f;
    floatx4 o = zero;
    const float *p = first + (r >> 4) * UNIT;
    const int rr = r & 15;
    for (int k0 = way; k0 < parts; k0 += 8 * ways) {
      float2 ml[8], x[8], y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float *at = p + (int64_t)min(k0 + j * ways, parts - 1) * step;
        ml[j] = get2(at + 16 * HDP + 2 * rr);
        x[j] = get2(at + rr * HDP + d);
        y[j] = get2(at + rr * HDP + d + 2);
      }
      float mn = M;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (k0 + j * ways >= parts) ml[j] = make_float2(NONE, 0.f), x[j] = y[j] = make_float2(0.f, 0.f);
        mn = fmaxf(mn, ml[j].x);
      }
      const float f = __builtin_amdgcn_exp2f(M - mn);
      M = mn;
      sum *= f;
      o *= f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float h = __builtin_amdgcn_exp2f(ml[j].x - mn);
        sum = fmaf(ml[j].y, h, sum);
        o[0] = fmaf(x[j].x, h, o[0]);
        o[1] = fmaf(x[j].y, h, o[1]);
        o[2] = fmaf(y[j].x, h, o[2]);
        o[3] = fmaf(y[j].y, h, o[3]);
      }
    }
    if (ways > 1) {  // (one pass: the units fit)
      __syncthreads();
      float *s = shares[threadIdx.x];
      *reinterpret_cast<floatx4 *>(s) = o;
      s[4] = M;
      s[5] = sum;
      __syncthreads();
      if (way) continue;
      for (int w = 1; w < ways; ++w) {
        const float *t = s + 8 * w;
        const float mn = fmaxf(M, t[4]);
        const float f = __builtin_amdgcn_exp2f(M - mn), h = __builtin_amdgcn_exp2f(t[4] - mn);
        M = mn;
        sum = fmaf(t[5], h, sum * f);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(t[e], h, o[e] * f);
      }
    }
    if (u < units && d < a.head_dim) {
      const float inv = 1.f / sum;
      *reinterpret_cast<float4 *>(out_row(r) + d) =
          make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
    }
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

// Pages that sequences shared: the filled blocks of one page and KV head (which lie side
// by side) and their scales, a workgroup (layer, page, head).  48 pages of 32 to 128
// positions, 8 heads of 128: 4 us, a launch's own time.
extern "C" __global__ void __launch_bounds__(256) pbx_kv_copy(KvPack a) {
  const int per_layer = a.n_items * a.kv_heads;
  const int layer = blockIdx.x / per_layer, in_layer = blockIdx.x % per_layer;
  const PageCopy it = reinterpret_cast<const PageCopy *>(a.items)[in_layer / a.kv_heads];
  const int head = in_layer % a.kv_heads;
  const int64_t from = block_index(a, it.from, head, 0), to = block_index(a, it.to, head, 0);
  uint8_t *codes = a.codes + layer * a.layer_codes;
  float *scales = a.scales + layer * a.layer_scales;
  const uintx4 *x = reinterpret_cast<const uintx4 *>(codes + from * a.head_dim);
  uintx4 *y = reinterpret_cast<uintx4 *>(codes + to * a.head_dim);
  const int n = it.blocks * (a.head_dim / 16);
  for (int i = threadIdx.x; i < n; i += 256) y[i] = x[i];
  if ((int)threadIdx.x < 2 * it.blocks) scales[2 * to + threadIdx.x] = scales[2 * from + threadIdx.x];
}

#define PBX_KV_KERNELS(HDP)                                                                                        \
  extern "C" __global__ void __launch_bounds__(append_threads(HDP))                                                \
      pbx_kv_append_##HDP(KvArgs a, KvRope r, const BlockItem *items, int n_blocks, const int *row_pos,            \
                          const float *K, int64_t ks, const float *V, int64_t vs, const float *Q, int64_t qs,      \
                          float *Qout, int64_t qos) {                                                              \
    append_body<HDP>(a, r, items, n_blocks, row_pos, K, ks, V, vs, Q, qs, Qout, qos);                              \
  }                                                                                                                \
  extern "C" __global__ void __launch_bounds__(append_threads(HDP))                                                \
      pbx_kv_read_##HDP(KvArgs a, const BlockItem *items, float *K, int64_t ks, float *V, int64_t vs) {            \
    read_body<HDP>(a, items, K, ks, V, vs);                                                                        \
  }                                                                                                                \
  extern "C" __global__ void __launch_bounds__(pack_threads(HDP)) pbx_kv_pack_##HDP(KvPack a, KvRope r) {        \
    pack_body<HDP>(a, r);                                                                                          \
  }
#define PBX_KV_ATTN(HDP, U, NQ, KW, RING, WAVES)                                                                   \
  extern "C" __global__ void __launch_bounds__(256, WAVES)                                                         \
      pbx_kv_attn_##HDP##_##U(KvArgs a, const AttnItem *items, const int *table, const float *Q, int64_t qs,       \
                              float scale, float *O, int64_t os, float *part, unsigned *arrived) {                 \
    static_assert(U == NQ * 4 / KW, "16-row tiles of the workgroup");                                              \
    attn_body<HDP, NQ, KW, RING>(a, items, table, Q, qs, scale, O, os, part, arrived);                             \
  }
PBX_KV_KERNELS(32)
PBX_KV_KERNELS(64)
PBX_KV_KERNELS(96)
PBX_KV_KERNELS(128)
PBX_KV_KERNELS(192)
PBX_KV_KERNELS(256)
PBX_KV_ATTN(32, 1, 1, 4, 3, 4)
PBX_KV_ATTN(32, 2, 2, 4, 3, 4)
PBX_KV_ATTN(32, 4, 2, 2, 3, 4)
PBX_KV_ATTN(64, 1, 1, 4, 3, 3)
PBX_KV_ATTN(64, 2, 2, 4, 2, 3)
PBX_KV_ATTN(64, 4, 2, 2, 1, 3)
PBX_KV_ATTN(96, 1, 1, 4, 2, 3)
PBX_KV_ATTN(96, 2, 2, 4, 2, 2)
PBX_KV_ATTN(128, 1, 1, 4, 2, 2)
PBX_KV_ATTN(128, 2, 2, 4, 2, 2)
PBX_KV_ATTN(192, 1, 1, 4, 1, 2)
PBX_KV_ATTN(192, 2, 1, 2, 1, 2)
PBX_KV_ATTN(256, 1, 1, 4, 1, 2)
PBX_KV_ATTN(256, 2, 1, 2, 1, 2)
