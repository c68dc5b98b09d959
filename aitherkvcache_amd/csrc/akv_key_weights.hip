// The attention weight that every cached key gets from a chunk's tokens, summed over the tokens and over the query heads of a kv head:
//
//   w[seq, kv head, key] = sum over rows (token, head of the group) of exp(s[row, key] - lse[row]),   s = scale q . k,  causal
//
// over plain rows (akv_key_weights) or packed ones (akv_packed_key_weights).  The sum over rows needs each row's normalisation first, so
// the scores are made twice: kw_stats leaves maximum and sum of every row over each part of the keys, kw_join joins the parts, and
// kw_sum makes the scores again with the operands exchanged, which puts a key into a lane and the rows side by side in its registers, where
// their weights are added.  A part's keys stay in registers while the rows go by through LDS.  Every sum has its order, nothing is added
// atomically.
//
// Weights are float32 and as near as that lets them be: products of 16-bit numbers are exact, packed levels and rotated queries are two
// float16 terms each (three products, 2^-22).
#include "akv_batch.h"
#include "akv_device_once.h"

#define KW_F16 0
#define KW_BF16 1                       // 2, 3, 4: packed codes of so many bits

struct kw_args {
  ab_batch b;
  const void* q; int64_t qs_tok, qs_head; int dtype;
  const uint8_t* k; int64_t k_blk, k_pos, k_head;     // bytes
  const float* kn; int64_t kn_blk, kn_pos, kn_head;   // packed: norms, elements
  const float* centroids;
  const float* turn;                    // Pi^T, row-major
  uint16_t* turned; float* turned_by;   // packed: queries of the slab [token - t0][QH][2][D], and what undoes their scale (times that of the scores)
  float2* part;                         // [parts][KVH][rows] maximum and sum
  float2* stat;                         // [KVH][rows] maximum and inverse sum
  float* out; int64_t os_seq, os_head;
  int64_t length;                       // floats of a row of the result
  int KVH, QH, G, t0, t1, add;
  int parts;
  float scale2;
};

template <int D, int KIND> struct kw_plan {
  static constexpr bool PACKED = KIND >= 2;
  static constexpr int DT = KIND == KW_BF16 ? AKV_BF16 : AKV_F16, KS = D / 16, TERMS = PACKED ? 2 : 1;
  static constexpr int KT = D * TERMS <= 128 ? 2 : 1, N = 4 * 32 * KT;      // tiles of 32 keys a wavefront; keys of a part
  static constexpr int CHUNKS = TERMS * D / 8, ROW = 16 * CHUNKS;           // of a row of queries in LDS
  static __device__ __forceinline__ int f(int r) { return D == 64 ? (r >> 1) & 7 : r & 15; }
};

// ---- rows of queries
struct kw_rows {                        // of a sequence, as far as the slab has them: row r is token first + r / G, head kvh G + r % G
  int first, rows, pos0;                // pos0: position of token `first`
};
__device__ __forceinline__ kw_rows kw_rows_of(const kw_args& a, int seq, int ctx) {
  const int s0 = ab_start(a.b, seq), s1 = ab_start(a.b, seq + 1);
  kw_rows r;
  r.first = max(s0, a.t0);
  r.rows = max(0, min(s1, a.t1) - r.first) * a.G;
  r.pos0 = ctx - (s1 - r.first);
  return r;
}
// 32 rows from r0 on into LDS: sixteen bytes c of row r lie at c ^ f(r); rows past the last are zero
template <int D, int KIND> __device__ __forceinline__ void kw_stage(const kw_args& a, const kw_rows& R, int r0, int kvh, unsigned char* lds) {
  typedef kw_plan<D, KIND> P;
  for (int i = threadIdx.x; i < 32 * P::CHUNKS; i += 256) {
    const int r = i / P::CHUNKS, c = i % P::CHUNKS, row = r0 + r;
    ab_u4 v = {0u, 0u, 0u, 0u};
    if (row < R.rows) {
      const int t = row / a.G, token = R.first + t, head = kvh * a.G + row - t * a.G;
      if constexpr (P::PACKED) v = *(const ab_u4*)(a.turned + ((int64_t)(token - a.t0) * a.QH + head) * (2 * D) + 8 * c);
      else v = *(const ab_u4*)((const uint16_t*)a.q + (int64_t)token * a.qs_tok + (int64_t)head * a.qs_head + 8 * c);
    }
    *(ab_u4*)(lds + r * P::ROW + 16 * (c ^ P::f(r))) = v;
  }
}

// ---- keys of a wavefront as operands
template <int BITS> struct kw_levels {                // level of a code: float16 terms, the first in the lower half
  uint32_t level[16];
};
// scale of the levels: the largest to [2^7, 2^8)
template <int BITS> __device__ __forceinline__ float kw_fill(kw_levels<BITS>& t, const float* __restrict__ centroids) {
  const float c = centroids[threadIdx.x & ((1 << BITS) - 1)];
  const uint32_t e = akv_row_exponent(akv_wave_max(fabsf(c)));
  if (threadIdx.x < 16) {
    const float x = c * akv_row_scale(e) * 128.f;
    const _Float16 hi = (_Float16)x;
    t.level[threadIdx.x] = ab_math<AKV_F16>::pair((float)hi, x - (float)hi);
  }
  return akv_row_unscale(e) * (1.f / 128.f);
}
// eight codes (the first on top) of run g of a half row
template <int BITS, int W> __device__ __forceinline__ uint32_t kw_code(const uint32_t (&w)[W], int g, int j) {
  if constexpr (BITS == 4) return (w[g] >> (8 * (j >> 1) + 4 * (1 - (j & 1)))) & 15u;
  else if constexpr (BITS == 2) return (w[g >> 1] >> (16 * (g & 1) + 8 * (j >> 2) + 2 * (3 - (j & 3)))) & 3u;
  else {
    const int b = 3 * g, i = b >> 2, o = b & 3;
    const uint32_t x = __builtin_amdgcn_perm(i + 1 < W ? w[i + 1 < W ? i + 1 : 0] : 0u, w[i], (uint32_t)(o + 2) | (uint32_t)(o + 1) << 8 | (uint32_t)o << 16 | 0x0c000000u);
    return (x >> (21 - 3 * j)) & 7u;
  }
}
template <int D, int KIND> struct kw_keys {
  typedef kw_plan<D, KIND> P;
  ab_u4 hi[P::KT][P::KS], lo[P::PACKED ? P::KT : 1][P::PACKED ? P::KS : 1];
  float norm[P::KT];                    // packed: of the lane's key
  // keys base .. base + 32 KT - 1 of a sequence of ctx > base tokens (those past the last: the last)
  __device__ __forceinline__ void load(const kw_args& a, int seq, int kvh, int base, int ctx, const uint32_t* levels) {
    const int lane = threadIdx.x & 63, h = lane >> 5, col = lane & 31;
#pragma unroll
    for (int t = 0; t < P::KT; ++t) {
      const int key = min(base + 32 * t + col, ctx - 1);
      uint32_t place;
      const uint32_t c = akv_div32((uint32_t)key, (uint32_t)a.b.block_size, a.b.bs_recip, place);
      const int64_t blk = ab_block(a.b, seq, c);
      const uint8_t* p = a.k + blk * a.k_blk + (int64_t)place * a.k_pos + (int64_t)kvh * a.k_head;
      if constexpr (!P::PACKED) {
#pragma unroll
        for (int ks = 0; ks < P::KS; ++ks) hi[t][ks] = *(const ab_u4*)(p + 32 * ks + 16 * h);
      } else {
        constexpr int BITS = KIND, W = D * BITS / 64;      // words of half a row
        uint32_t w[W];
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = *(const uint32_t*)(p + 4 * (W * h + i));
        norm[t] = a.kn[blk * a.kn_blk + (int64_t)place * a.kn_pos + (int64_t)kvh * a.kn_head];
#pragma unroll
        for (int ks = 0; ks < P::KS; ++ks)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t x = levels[kw_code<BITS>(w, ks, 2 * i)], y = levels[kw_code<BITS>(w, ks, 2 * i + 1)];
            hi[t][ks][i] = __builtin_amdgcn_perm(y, x, 0x05040100u);
            lo[t][ks][i] = __builtin_amdgcn_perm(y, x, 0x07060302u);
          }
      }
    }
  }
  // products of tile t with the 32 rows in LDS; KEYS_FIRST: a key's are in the registers, a row's in a lane
  template <bool KEYS_FIRST> __device__ __forceinline__ ab_f16 product(int t, const unsigned char* rows) const {
    typedef ab_math<P::DT> M;
    const int lane = threadIdx.x & 63, h = lane >> 5, col = lane & 31;
    const unsigned char* r = rows + col * P::ROW;
    ab_f16 y = (ab_f16)(0.f);
#pragma unroll
    for (int ks = 0; ks < P::KS; ++ks) {
      // (packed: a lane has the half row h, plain: half of every sixteen coordinates)
      const int c = P::PACKED ? P::KS * h + ks : 2 * ks + h;
      const ab_u4 q = *(const ab_u4*)(r + 16 * (c ^ P::f(col)));
      if constexpr (P::PACKED) {
        const ab_u4 q_lo = *(const ab_u4*)(r + 16 * ((D / 8 + c) ^ P::f(col)));
        if constexpr (KEYS_FIRST) {
          y = M::mfma32(lo[t][ks], q, y);
          y = M::mfma32(hi[t][ks], q_lo, y);
        } else {
          y = M::mfma32(q, lo[t][ks], y);
          y = M::mfma32(q_lo, hi[t][ks], y);
        }
      }
      y = KEYS_FIRST ? M::mfma32(hi[t][ks], q, y) : M::mfma32(q, hi[t][ks], y);
    }
    return y;
  }
};

// ---- queries of packed rows: turned, scaled and as two terms; a workgroup takes 8 rows
template <int D> __global__ __launch_bounds__(256) void kw_turn_kernel(kw_args a) {
  constexpr int PER = 256 / D > 0 ? 256 / D : 1, LANES = D < 256 ? D : 256, R = 8 / PER;      // threads of a row; rows of a thread
  __shared__ float x[8][D];
  __shared__ float top[8][4];
  const int64_t rows = (int64_t)(a.t1 - a.t0) * a.QH, r0 = (int64_t)blockIdx.x * 8;
  for (int i = threadIdx.x; i < 8 * D; i += 256) {
    const int64_t r = r0 + i / D;
    float v = 0.f;
    if (r < rows) {
      const int64_t at = (r / a.QH + a.t0) * a.qs_tok + (r % a.QH) * a.qs_head + i % D;
      v = a.dtype == AKV_F16 ? akv_elem<AKV_F16>::load(a.q, at) : akv_elem<AKV_BF16>::load(a.q, at);
    }
    x[i / D][i % D] = v;
  }
  __syncthreads();
  const int d = threadIdx.x % LANES, who = threadIdx.x / LANES;
  float y[R][2] = {};
  for (int j = 0; j < D; j += 2) {
    const float p = a.turn[(size_t)j * D + d], p1 = a.turn[(size_t)(j + 1) * D + d];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      y[i][0] = fmaf(p, x[who * R + i][j], y[i][0]);
      y[i][1] = fmaf(p1, x[who * R + i][j + 1], y[i][1]);
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const float t = akv_wave_max(fabsf(y[i][0] + y[i][1]));
    if ((threadIdx.x & 63) == 0) top[who * R + i][(threadIdx.x % LANES) / 64] = t;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int64_t r = r0 + who * R + i;
    if (r >= rows) break;
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < LANES / 64; ++w) t = fmaxf(t, top[who * R + i][w]);
    const uint32_t e = akv_row_exponent(t);
    const float v = (y[i][0] + y[i][1]) * akv_row_scale(e) * 8192.f;      // the largest to [2^13, 2^14)
    const _Float16 hi = (_Float16)v, lo = (_Float16)(v - (float)hi);
    a.turned[r * (2 * D) + d] = __builtin_bit_cast(uint16_t, hi);
    a.turned[r * (2 * D) + D + d] = __builtin_bit_cast(uint16_t, lo);
    if (d == 0) a.turned_by[r] = akv_row_unscale(e) * (1.f / 8192.f) * a.scale2;
  }
}

// ---- maxima and sums of the rows over a part of the keys
template <int D, int KIND> __global__ __launch_bounds__(256, 2) void kw_stats_kernel(kw_args a) {
  typedef kw_plan<D, KIND> P;
  __shared__ __align__(16) unsigned char rows[32 * P::ROW];
  __shared__ float2 ml[4][32];
  __shared__ __align__(16) float norms[P::PACKED ? P::N : 4];
  __shared__ kw_levels<P::PACKED ? KIND : 4> levels;
  const int part = blockIdx.x, kvh = blockIdx.y, seq = blockIdx.z;
  const int ctx = ab_ctx(a.b, seq), from = part * P::N;
  if (from >= ctx) return;
  const kw_rows R = kw_rows_of(a, seq, ctx);
  if (R.rows == 0 || R.pos0 + (R.rows - 1) / a.G < from) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, col = lane & 31;
  const int base = from + 32 * P::KT * wave;
  kw_keys<D, KIND> K;
  float unit = 1.f;
  if constexpr (P::PACKED) {
    unit = kw_fill(levels, a.centroids);
    __syncthreads();
  }
  const bool any = base < ctx;
  if (any) K.load(a, seq, kvh, base, ctx, levels.level);
  if constexpr (P::PACKED) {
    if (any && h == 0)
#pragma unroll
      for (int t = 0; t < P::KT; ++t) norms[32 * (P::KT * wave + t) + col] = K.norm[t] * unit;
  }
  const int64_t all = (int64_t)(a.t1 - a.t0) * a.G, at = (int64_t)(R.first - a.t0) * a.G;
  float2* to = a.part + ((int64_t)part * a.KVH + kvh) * all + at;
  const int skip = max(0, from - R.pos0) * a.G / 32 * 32;      // rows before see nothing of the part
  for (int r0 = skip; r0 < R.rows; r0 += 32) {
    __syncthreads();
    kw_stage<D, KIND>(a, R, r0, kvh, rows);
    __syncthreads();
    const int row = r0 + col, pos = row < R.rows ? R.pos0 + row / a.G : -1;
    float m = -INFINITY, l = 0.f;
    if (any) {
      float c = a.scale2;
      if constexpr (P::PACKED) c = row < R.rows ? a.turned_by[(int64_t)(R.first - a.t0 + row / a.G) * a.QH + kvh * a.G + row % a.G] : 0.f;
      ab_f16 s[P::KT];
      const bool edge = base + 32 * P::KT - 1 > R.pos0 + r0 / a.G;
#pragma unroll
      for (int t = 0; t < P::KT; ++t) {
        s[t] = K.template product<true>(t, rows);
        if constexpr (P::PACKED) {
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const float4 n = *(const float4*)(norms + 32 * (P::KT * wave + t) + 8 * b + 4 * h);
            s[t][4 * b] *= n.x; s[t][4 * b + 1] *= n.y; s[t][4 * b + 2] *= n.z; s[t][4 * b + 3] *= n.w;
          }
        }
        if (edge) {
#pragma unroll
          for (int i = 0; i < 16; ++i) s[t][i] = base + 32 * t + 8 * (i >> 2) + 4 * h + (i & 3) <= pos ? s[t][i] : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) m = fmaxf(m, s[t][i]);
      }
      m = fmaxf(m, akv_lane_xor<32>(m)) * c;
      const float ref = m == -INFINITY || m != m ? 0.f : m;
#pragma unroll
      for (int t = 0; t < P::KT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) l += __builtin_amdgcn_exp2f(fmaf(s[t][i], c, -ref));
      l += akv_lane_xor<32>(l);
      if (m != m) m = -INFINITY, l = 0.f;      // (-inf times 0: a row that is none)
    }
    if (h == 0) ml[wave][col] = make_float2(m, l);
    __syncthreads();
    if (tid < 32 && row < R.rows) {
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, ml[w][tid].x);
#pragma unroll
      for (int w = 0; w < 4; ++w) sum += ml[w][tid].x == -INFINITY ? 0.f : ml[w][tid].y * __builtin_amdgcn_exp2f(ml[w][tid].x - top);
      to[row] = make_float2(top, sum);
    }
  }
}

// ---- the parts of a row together, a wavefront a row
template <int N> __global__ __launch_bounds__(256) void kw_join_kernel(kw_args a) {
  const int lane = threadIdx.x & 63;
  const int64_t all = (int64_t)(a.t1 - a.t0) * a.G, x = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (x >= all * a.KVH) return;
  const int64_t kvh = x / all, row = x - kvh * all;
  const int token = a.t0 + (int)(row / a.G);
  const int seq = ab_last(a.b.S, token, [&](int i) { return (int64_t)ab_start(a.b, i); });
  if (seq < 0) return;
  const int s1 = ab_start(a.b, seq + 1), pos = ab_ctx(a.b, seq) - (s1 - token);
  if (token >= s1) return;
  float m = -INFINITY, l = 0.f;
  for (int p = lane; pos >= 0 && p <= pos / N; p += 64) {
    const float2 e = a.part[((int64_t)p * a.KVH + kvh) * all + row];
    const float top = fmaxf(m, e.x);
    if (top == -INFINITY) continue;
    l = l * __builtin_amdgcn_exp2f(m - top) + e.y * __builtin_amdgcn_exp2f(e.x - top);
    m = top;
  }
  const float top = akv_wave_max(m);
  l = akv_wave_sum(m == -INFINITY ? 0.f : l * __builtin_amdgcn_exp2f(m - top));
  if (lane == 0) a.stat[kvh * all + row] = l > 0.f ? make_float2(top, 1.f / l) : make_float2(0.f, 0.f);
}

// ---- weights of a part's keys, summed over the rows
template <int D, int KIND> __global__ __launch_bounds__(256, 2) void kw_sum_kernel(kw_args a) {
  typedef kw_plan<D, KIND> P;
  __shared__ __align__(16) unsigned char rows[32 * P::ROW];
  __shared__ __align__(16) float ref[32], inv[32], by[32];
  __shared__ kw_levels<P::PACKED ? KIND : 4> levels;
  const int part = blockIdx.x, kvh = blockIdx.y, seq = blockIdx.z;
  const int ctx = ab_ctx(a.b, seq);
  const int64_t from = (int64_t)part * P::N;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, col = lane & 31;
  float* to = a.out + (int64_t)seq * a.os_seq + (int64_t)kvh * a.os_head;
  const kw_rows R = kw_rows_of(a, seq, ctx);
  if (from >= ctx || R.rows == 0 || R.pos0 + (R.rows - 1) / a.G < from) {
    if (!a.add)
      for (int64_t i = from + tid; i < from + P::N && i < a.length; i += 256) to[i] = 0.f;
    return;
  }
  const int base = (int)from + 32 * P::KT * wave;
  kw_keys<D, KIND> K;
  float unit = 1.f;
  if constexpr (P::PACKED) {
    unit = kw_fill(levels, a.centroids);
    __syncthreads();
  }
  const bool any = base < ctx;
  if (any) K.load(a, seq, kvh, base, ctx, levels.level);
  float w[P::KT] = {};
  const int64_t all = (int64_t)(a.t1 - a.t0) * a.G;
  const float2* stat = a.stat + (int64_t)kvh * all + (int64_t)(R.first - a.t0) * a.G;
  const int skip = max(0, (int)from - R.pos0) * a.G / 32 * 32;
  for (int r0 = skip; r0 < R.rows; r0 += 32) {
    __syncthreads();
    kw_stage<D, KIND>(a, R, r0, kvh, rows);
    if (tid < 32) {
      const int row = r0 + tid;
      float2 e = make_float2(0.f, 0.f);
      float c = 0.f;
      if (row < R.rows) {
        e = stat[row];
        c = a.scale2;
        if constexpr (P::PACKED) c = a.turned_by[(int64_t)(R.first - a.t0 + row / a.G) * a.QH + kvh * a.G + row % a.G];
      }
      ref[tid] = e.x;
      inv[tid] = e.y;
      by[tid] = c;
    }
    __syncthreads();
    if (!any) continue;
    const bool edge = base + 32 * P::KT - 1 > R.pos0 + r0 / a.G;
#pragma unroll
    for (int t = 0; t < P::KT; ++t) {
      const ab_f16 s = K.template product<false>(t, rows);
      float n = 1.f;
      if constexpr (P::PACKED) n = K.norm[t] * unit;
      const int key = base + 32 * t + col;
      float sum = 0.f;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const float4 m4 = *(const float4*)(ref + 8 * b + 4 * h), i4 = *(const float4*)(inv + 8 * b + 4 * h), c4 = *(const float4*)(by + 8 * b + 4 * h);
        const float m[4] = {m4.x, m4.y, m4.z, m4.w}, iv[4] = {i4.x, i4.y, i4.z, i4.w}, c[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float e = __builtin_amdgcn_exp2f(fmaf(P::PACKED ? s[4 * b + i] * n : s[4 * b + i], c[i], -m[i]));
          if (edge) e = key <= R.pos0 + (r0 + 8 * b + 4 * h + i) / a.G ? e : 0.f;
          sum = fmaf(e, iv[i], sum);
        }
      }
      w[t] += sum;
    }
  }
#pragma unroll
  for (int t = 0; t < P::KT; ++t) {
    const float sum = w[t] + akv_lane_xor<32>(w[t]);
    const int64_t key = (int64_t)base + 32 * t + col;
    if (h == 0 && key < a.length) {
      if (key < ctx) to[key] = a.add ? to[key] + sum : sum;
      else if (!a.add) to[key] = 0.f;
    }
  }
}

// ---- launches
#define KW_SCRATCH (256ll << 20)
struct kw_scratch { int64_t tokens; size_t stat, part, turned, by, bytes; int parts; };
// scratch of a call, its tokens in slabs of what KW_SCRATCH holds (a multiple of 32, or all)
static inline kw_scratch kw_layout(int64_t T, int QH, int D, bool packed, int keys, int64_t length) {
  kw_scratch w = {};
  w.parts = (int)((length + keys - 1) / keys);
  const int64_t per = (int64_t)QH * (8 + 8 * (int64_t)w.parts + (packed ? 4 * D + 4 : 0));
  w.tokens = KW_SCRATCH / per / 32 * 32;
  if (w.tokens < 32) w.tokens = 32;
  if (w.tokens > T) w.tokens = T;
  const int64_t rows = w.tokens * QH;
  w.stat = 0;
  w.part = akv_align256((size_t)rows * 8);
  w.turned = w.part + akv_align256((size_t)rows * 8 * w.parts);
  w.by = w.turned + (packed ? akv_align256((size_t)rows * 4 * D) : 0);
  w.bytes = w.by + (packed ? akv_align256((size_t)rows * 4) : 0);
  return w;
}
static inline int kw_part(int D, bool packed) { return D * (packed ? 2 : 1) <= 128 ? 256 : 128; }
static inline size_t kw_bytes(int64_t T, int QH, int D, bool packed, int64_t length) {
  return T <= 0 || QH <= 0 || length <= 0 || !ab_head_size(D) ? 0 : kw_layout(T, QH, D, packed, kw_part(D, packed), length).bytes;
}
extern "C" size_t akv_key_weights_workspace_bytes(int64_t num_tokens, int num_q_heads, int d, int64_t length) { return kw_bytes(num_tokens, num_q_heads, d, false, length); }
extern "C" size_t akv_packed_key_weights_workspace_bytes(int64_t num_tokens, int num_q_heads, int d, int64_t length) { return kw_bytes(num_tokens, num_q_heads, d, true, length); }

template <int D, int KIND> static int kw_launch(kw_args a, int64_t T, void* scratch, hipStream_t stream) {
  typedef kw_plan<D, KIND> P;
  static_assert(P::N == (D * P::TERMS <= 128 ? 256 : 128), "kw_part");
  const kw_scratch w = kw_layout(T, a.QH, D, P::PACKED, P::N, a.length);
  a.stat = (float2*)((char*)scratch + w.stat);
  a.part = (float2*)((char*)scratch + w.part);
  a.turned = (uint16_t*)((char*)scratch + w.turned);
  a.turned_by = (float*)((char*)scratch + w.by);
  a.parts = w.parts;
  const int add = a.add;
  const dim3 grid((uint32_t)w.parts, (uint32_t)a.KVH, (uint32_t)a.b.S);
  int64_t t = 0;
  do {                                  // (without a token: zeros)
    a.t0 = (int)t;
    a.t1 = (int)(t + w.tokens < T ? t + w.tokens : T);
    a.add = add || t > 0;
    const int64_t rows = (int64_t)(a.t1 - a.t0) * a.QH;
    if (rows > 0) {
      if constexpr (P::PACKED) {
        kw_turn_kernel<D><<<(uint32_t)((rows + 7) / 8), 256, 0, stream>>>(a);
        AKV_LAUNCH_CHECK("kw_turn_kernel");
      }
      kw_stats_kernel<D, KIND><<<grid, 256, 0, stream>>>(a);
      AKV_LAUNCH_CHECK("kw_stats_kernel");
      kw_join_kernel<P::N><<<(uint32_t)((rows + 3) / 4), 256, 0, stream>>>(a);
      AKV_LAUNCH_CHECK("kw_join_kernel");
    }
    kw_sum_kernel<D, KIND><<<grid, 256, 0, stream>>>(a);
    AKV_LAUNCH_CHECK("kw_sum_kernel");
    t += w.tokens;
  } while (t < T);
  return AKV_OK;
}
static inline int kw_check(const char* name, const kw_args& a, int dtype, int64_t T, int d, int64_t max_blocks, float scale, void* workspace, size_t workspace_bytes, bool packed) {
  AKV_REQUIRE(akv_valid_dtype(dtype), "%s: bad dtype %d", name, dtype);
  AKV_REQUIRE(a.QH > 0 && a.QH % a.KVH == 0, "%s: %d query heads on %d kv heads", name, a.QH, a.KVH);
  AKV_REQUIRE(scale > 0.f && scale < INFINITY, "%s: scale must be positive and finite", name);
  if (dtype == AKV_F32) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: float32 queries are not supported; use float16 or bfloat16", name);
  if (!ab_head_size(d)) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: head_dim %d; kernels are built for 64, 128 and 256", name, d);
  AKV_REQUIRE(a.length >= 0 && (a.length >= max_blocks * a.b.block_size || a.length >= AB_MOST_TOKENS), "%s: rows of %lld weights for tables of %lld tokens", name, (long long)a.length, (long long)max_blocks * a.b.block_size);
  if (a.KVH > 65535 || a.b.S > 65535) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: more than 65535 sequences or kv heads", name);
  if (a.length > AB_MOST_TOKENS) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: rows of 2^31 weights", name);
  if (a.b.S == 0 || a.length == 0) return AKV_OK;
  AKV_REQUIRE(a.out && (T == 0 || a.q) && a.b.starts, "%s: null pointer", name);
  if (T * (int64_t)a.QH > 0x7fffffff) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: more than 2^31 rows", name);
  if (!ab_aligned(a.q, 16) || ((a.qs_tok | a.qs_head) & 7)) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: queries must lie at multiples of 16 bytes", name);
  const size_t need = kw_bytes(T, a.QH, d, packed, a.length);
  if (need && (!workspace || workspace_bytes < need || !ab_aligned(workspace, 256))) return akv_fail(AKV_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", name, need);
  return AKV_OK;
}

extern "C" int akv_key_weights(const void* query, int dtype, int64_t qs_tok, int64_t qs_head, const void* key_cache, int64_t ks_blk, int64_t ks_pos, int64_t ks_head, const void* block_tables,
                               int bt_itype, int64_t bt_stride, const void* context_lens, int cl_itype, const void* query_starts, int qs_itype, float* weights, int64_t ws_seq, int64_t ws_head,
                               int64_t length, int accumulate, int num_seqs, int64_t num_tokens, int num_q_heads, int num_kv_heads, int d, int block_size, int64_t num_blocks,
                               int64_t max_blocks_per_seq, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  const char* name = "akv_key_weights";
  int rc = ab_check(name, block_tables, bt_itype, context_lens, cl_itype, query_starts, qs_itype, num_seqs, num_tokens, num_kv_heads, block_size, num_blocks, max_blocks_per_seq);
  if (rc) return rc;
  kw_args a = {};
  a.b = ab_make(block_tables, bt_itype, bt_stride, context_lens, cl_itype, query_starts, qs_itype, num_seqs, num_tokens, block_size, num_blocks, max_blocks_per_seq);
  a.q = query; a.qs_tok = qs_tok; a.qs_head = qs_head; a.dtype = dtype;
  a.k = (const uint8_t*)key_cache; a.k_blk = 2 * ks_blk; a.k_pos = 2 * ks_pos; a.k_head = 2 * ks_head;
  a.out = weights; a.os_seq = ws_seq; a.os_head = ws_head; a.length = length; a.add = accumulate;
  a.KVH = num_kv_heads; a.QH = num_q_heads; a.G = num_q_heads / num_kv_heads; a.scale2 = scale * 1.44269504088896341f;
  if ((rc = kw_check(name, a, dtype, num_tokens, d, max_blocks_per_seq, scale, workspace, workspace_bytes, false))) return rc;
  if (num_seqs == 0 || length == 0) return AKV_OK;
  AKV_REQUIRE(num_blocks == 0 || max_blocks_per_seq == 0 || key_cache, "%s: null pointer", name);
  if (!ab_aligned(key_cache, 16) || ((ks_blk | ks_pos | ks_head) & 7)) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: rows must lie at multiples of 16 bytes", name);
  const hipStream_t s = (hipStream_t)stream;
#define KW_CASE(DIM) if (d == DIM) return dtype == AKV_F16 ? kw_launch<DIM, KW_F16>(a, num_tokens, workspace, s) : kw_launch<DIM, KW_BF16>(a, num_tokens, workspace, s);
  KW_CASE(64) KW_CASE(128) KW_CASE(256)
#undef KW_CASE
  return AKV_ERR_UNSUPPORTED;
}

extern "C" int akv_packed_key_weights(const void* query, int dtype, int64_t qs_tok, int64_t qs_head, const uint8_t* k_packed, int64_t kps_blk, int64_t kps_pos, int64_t kps_head,
                                      const float* k_norms, int64_t kns_blk, int64_t kns_pos, int64_t kns_head, const void* block_tables, int bt_itype, int64_t bt_stride,
                                      const void* context_lens, int cl_itype, const void* query_starts, int qs_itype, const void* rot_prep, const float* centroids, int bits, float* weights,
                                      int64_t ws_seq, int64_t ws_head, int64_t length, int accumulate, int num_seqs, int64_t num_tokens, int num_q_heads, int num_kv_heads, int d, int block_size,
                                      int64_t num_blocks, int64_t max_blocks_per_seq, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  const char* name = "akv_packed_key_weights";
  int rc = ab_check(name, block_tables, bt_itype, context_lens, cl_itype, query_starts, qs_itype, num_seqs, num_tokens, num_kv_heads, block_size, num_blocks, max_blocks_per_seq);
  if (rc) return rc;
  AKV_REQUIRE(bits >= 2 && bits <= 4, "%s: bits must be 2, 3 or 4, got %d", name, bits);
  kw_args a = {};
  a.b = ab_make(block_tables, bt_itype, bt_stride, context_lens, cl_itype, query_starts, qs_itype, num_seqs, num_tokens, block_size, num_blocks, max_blocks_per_seq);
  a.q = query; a.qs_tok = qs_tok; a.qs_head = qs_head; a.dtype = dtype;
  a.k = k_packed; a.k_blk = kps_blk; a.k_pos = kps_pos; a.k_head = kps_head;
  a.kn = k_norms; a.kn_blk = kns_blk; a.kn_pos = kns_pos; a.kn_head = kns_head;
  a.centroids = centroids;
  a.turn = (const float*)rot_prep + (size_t)d * d;
  a.out = weights; a.os_seq = ws_seq; a.os_head = ws_head; a.length = length; a.add = accumulate;
  a.KVH = num_kv_heads; a.QH = num_q_heads; a.G = num_q_heads / num_kv_heads; a.scale2 = scale * 1.44269504088896341f;
  if ((rc = kw_check(name, a, dtype, num_tokens, d, max_blocks_per_seq, scale, workspace, workspace_bytes, true))) return rc;
  if (num_seqs == 0 || length == 0) return AKV_OK;
  AKV_REQUIRE(rot_prep && centroids, "%s: null pointer", name);
  AKV_REQUIRE(num_blocks == 0 || max_blocks_per_seq == 0 || (k_packed && k_norms), "%s: null pointer", name);
  if (!ab_aligned(k_packed, 4) || ((kps_blk | kps_pos | kps_head) & 3)) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: packed rows must lie at multiples of 4 bytes", name);
  const hipStream_t s = (hipStream_t)stream;
#define KW_CASE(DIM)                                                                                                                       \
  if (d == DIM) return bits == 4 ? kw_launch<DIM, 4>(a, num_tokens, workspace, s) : bits == 3 ? kw_launch<DIM, 3>(a, num_tokens, workspace, s) \
                                                                                              : kw_launch<DIM, 2>(a, num_tokens, workspace, s);
  KW_CASE(64) KW_CASE(128) KW_CASE(256)
#undef KW_CASE
  return AKV_ERR_UNSUPPORTED;
}
