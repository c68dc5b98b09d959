// Attention of a chunk of new tokens over a paged cache of float16 or bfloat16 rows, or of packed codes (akv_chunk.h: how the work is
// cut).
//
//   S^T[key, row] = K[key, :] . Q[row, :]          v_mfma_f32_32x32x16, A = 32 keys, B = 32 rows
//   O^T[d, row] = sum_key V[key, d] P^T[key, row]  A = 32 coordinates, B = 32 rows
//
// With the rows on the column side of both products a lane holds one row, and of its scores every second group of four keys (the
// other half of the wavefront the others): maximum and sum of the softmax are taken in the lane, one exchange between the halves
// a tile joins the maxima, the running rescale is a factor per lane, and the weights of the first product ARE the operand of the second: its k
// axis takes the keys in the order in which a lane holds them, 4h .. 4h + 3 and 8 + 4h .. 8 + 4h + 3 of sixteen.  V^T comes out of
// LDS by transposing reads (ds_read_b64_tr_b16: four keys of a coordinate a lane).
//
// Packed rows are attended in the rotated domain: queries are rotated before (ck_rotate_q_kernel), outputs after
// (ck_rotate_out_kernel), and in between a key is its norm times levels of the codebook.  Levels are float16 in units of a power of
// two (relative precision 2^-11 whatever the codebook's size); a key's norm multiplies its score in float32; a value's norm v goes into the
// exponent, w = 2^(s + log2 v - M), with M the running maximum of s + log2 v, so weights stay in [0, 1] for norms of any size,
// and the sum of the softmax takes w / v.
#pragma once
#include "akv_chunk.h"
#include "akv_device_once.h"

typedef _Float16 ck_half8 __attribute__((ext_vector_type(8)));
typedef __bf16 ck_bf8 __attribute__((ext_vector_type(8)));
typedef short ck_s4 __attribute__((ext_vector_type(4)));
typedef float ck_f16v __attribute__((ext_vector_type(16)));
typedef uint32_t ck_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t ck_u2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) ck_s4 ck_lds_s4;
typedef __attribute__((address_space(3))) ck_u4 ck_lds_u4;

#define CK_F16 0
#define CK_BF16 1                 // 2, 3, 4: packed codes of so many bits

// Smallest value norm that counts (its inverse, summed over a cache, is finite).  A smaller one, such as 0, has weight 1 in the
// frame of the exponents, as if its logarithm were 0, and its key is taken out of the product (ck_drop).  Norms of one sequence may
// lie 2^120 apart: weights are float32 until the sum of the softmax has taken them.
#define CK_TINY 0x1p-90f

__device__ __forceinline__ float ck_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

template <int KIND> struct ck_math {
  static constexpr bool packed = KIND >= 2;
  static __device__ __forceinline__ ck_f16v mfma(ck_u4 a, ck_u4 b, ck_f16v c) {
    if constexpr (KIND == CK_BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(ck_bf8, a), __builtin_bit_cast(ck_bf8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(ck_half8, a), __builtin_bit_cast(ck_half8, b), c, 0, 0, 0);
  }
  // two weights in [0, 1] to the type of the values (one rounding, to nearest)
  static __device__ __forceinline__ uint32_t pair(float x, float y) {
    if constexpr (KIND == CK_BF16) {
      typedef __bf16 b2 __attribute__((ext_vector_type(2)));
      b2 r = {(__bf16)x, (__bf16)y};
      return __builtin_bit_cast(uint32_t, r);
    } else {
      typedef _Float16 h2 __attribute__((ext_vector_type(2)));
      h2 r = {(_Float16)x, (_Float16)y};
      return __builtin_bit_cast(uint32_t, r);
    }
  }
};

// ---- packed codes -> float16 levels -----------------------------------------------------------------------------
// The codebook as bytes: low and high bytes of the levels of codes 0..3, 4..7, 8..11, 12..15, for v_perm.
template <int BITS> struct ck_table {
  static constexpr int N = BITS == 4 ? 4 : BITS == 3 ? 2 : 1;
  uint32_t lo[N], hi[N];
  float up;                 // the levels are in units of 1 / up ... value = level x unit
  __device__ __forceinline__ void load(const float* __restrict__ centroids) {
    float c[1 << BITS], m = 0.f;
#pragma unroll
    for (int i = 0; i < (1 << BITS); ++i) {
      c[i] = centroids[i];
      m = fmaxf(m, fabsf(c[i]));
    }
    const uint32_t e = akv_row_exponent(m);
    const float down = akv_row_scale(e);
    up = akv_row_unscale(e);
#pragma unroll
    for (int w = 0; w < N; ++w) {
      lo[w] = hi[w] = 0u;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const uint32_t h = __builtin_bit_cast(unsigned short, (_Float16)(c[4 * w + b] * down));
        lo[w] |= (h & 255u) << (8 * b);
        hi[w] |= (h >> 8) << (8 * b);
      }
    }
  }
  // four codes, a byte each, to two words of two levels
  __device__ __forceinline__ void four(uint32_t sel, uint32_t& w0, uint32_t& w1) const {
    uint32_t l, h;
    if constexpr (BITS == 4) {
      const uint32_t s = sel & 0x07070707u, t = (sel >> 3) & 0x01010101u, m = (t << 8) - t;
      const uint32_t l0 = __builtin_amdgcn_perm(lo[1], lo[0], s), l1 = __builtin_amdgcn_perm(lo[3], lo[2], s);
      const uint32_t h0 = __builtin_amdgcn_perm(hi[1], hi[0], s), h1 = __builtin_amdgcn_perm(hi[3], hi[2], s);
      l = (l1 & m) | (l0 & ~m);
      h = (h1 & m) | (h0 & ~m);
    } else if constexpr (BITS == 3) {
      l = __builtin_amdgcn_perm(lo[1], lo[0], sel);
      h = __builtin_amdgcn_perm(hi[1], hi[0], sel);
    } else {
      l = __builtin_amdgcn_perm(0u, lo[0], sel);
      h = __builtin_amdgcn_perm(0u, hi[0], sel);
    }
    w0 = __builtin_amdgcn_perm(h, l, 0x05010400u);
    w1 = __builtin_amdgcn_perm(h, l, 0x07030602u);
  }
};
// Group g (eight coordinates) of a run of codes that starts at word 0 of `w`, as eight levels in the order ck_order.
template <int BITS, int W> __device__ __forceinline__ ck_u4 ck_levels(const ck_table<BITS>& t, const uint32_t (&w)[W], int g) {
  uint32_t s0, s1;
  if constexpr (BITS == 4) {
    s0 = (w[g] >> 4) & 0x0f0f0f0fu;
    s1 = w[g] & 0x0f0f0f0fu;
  } else if constexpr (BITS == 3) {
    // 24 bits, the first coordinate on top: bytes 3g, 3g + 1, 3g + 2
    const int b = 3 * g, i = b >> 2, o = b & 3;
    const uint32_t sel = (uint32_t)(o + 2) | (uint32_t)(o + 1) << 8 | (uint32_t)o << 16 | 0x0c000000u;
    const uint32_t x = __builtin_amdgcn_perm(i + 1 < W ? w[i + 1 < W ? i + 1 : 0] : 0u, w[i], sel);
    const uint32_t a = x >> 12, c = x & 0xfffu;
    const uint32_t a2 = (a | a << 10) & 0x003f003fu, c2 = (c | c << 10) & 0x003f003fu;
    s0 = (a2 | a2 << 5) & 0x07070707u;
    s1 = (c2 | c2 << 5) & 0x07070707u;
  } else {
    const uint32_t x = g & 1 ? w[g >> 1] >> 16 : w[g >> 1];
    const uint32_t a = x & 0xffu, c = (x >> 8) & 0xffu;
    const uint32_t a2 = (a | a << 12) & 0x000f000fu, c2 = (c | c << 12) & 0x000f000fu;
    s0 = (a2 | a2 << 6) & 0x03030303u;
    s1 = (c2 | c2 << 6) & 0x03030303u;
  }
  ck_u4 r;
  uint32_t r0, r1, r2, r3;
  t.four(s0, r0, r1);
  t.four(s1, r2, r3);
  r[0] = r0; r[1] = r1; r[2] = r2; r[3] = r3;
  return r;
}
// place of coordinate c (of eight) in such a group, and the coordinate at a place
template <int BITS> __host__ __device__ constexpr int ck_place(int c) { return BITS == 4 ? (c >> 1) + 4 * (c & 1) : (c & 4) + 3 - (c & 3); }
template <int BITS> __host__ __device__ constexpr int ck_coord(int p) { return BITS == 4 ? 2 * (p & 3) + (p >> 2) : (p & 4) + 3 - (p & 3); }

// ---- one step of the softmax ----------------------------------------------------------------------------------------
// A row's running state; l is the sum over the lane's own keys (the halves are added at the end).
struct ck_row { float m, l; };
// Scores s of NT tiles of 32 keys to weights, in place; returns what the sums so far have to be multiplied with.  Dense: s is a raw product
// and m a maximum of such, c = scale x log2 e.  Packed: s are exponents already (norms in them), c = 1, `inv` the inverse value norms.
template <int NT, bool PACKED>
__device__ __forceinline__ float ck_softmax(ck_f16v (&s)[NT], ck_row& r, float c, const float* __restrict__ inv) {
  float mx = s[0][0];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[t][i]);
  mx = fmaxf(mx, akv_lane_xor<32>(mx));
  const float mn = fmaxf(r.m, mx);
  const float ref = mn == -INFINITY ? 0.f : mn * c;
  const float alpha = ck_exp2(fmaf(r.m, c, -ref));
  r.m = mn;
  float l = 0.f;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float w = ck_exp2(PACKED ? s[t][i] - ref : fmaf(s[t][i], c, -ref));
      s[t][i] = w;
      if constexpr (!PACKED) l += w;
    }
  if constexpr (PACKED) {
    const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const float4 v = *(const float4*)(inv + 32 * t + 8 * b + 4 * h);
        l = fmaf(s[t][4 * b], v.x, l); l = fmaf(s[t][4 * b + 1], v.y, l);
        l = fmaf(s[t][4 * b + 2], v.z, l); l = fmaf(s[t][4 * b + 3], v.w, l);
      }
  }
  r.l = fmaf(r.l, alpha, l);
  return alpha;
}
// products to exponents: norms of 32 NT keys from LDS, f = the row's factor
template <int NT>
__device__ __forceinline__ void ck_norms(ck_f16v (&s)[NT], float f, const float* __restrict__ kn, const float* __restrict__ lg) {
  const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const float4 k = *(const float4*)(kn + 32 * t + 8 * b + 4 * h), g = *(const float4*)(lg + 32 * t + 8 * b + 4 * h);
      s[t][4 * b] = fmaf(s[t][4 * b] * k.x, f, g.x);
      s[t][4 * b + 1] = fmaf(s[t][4 * b + 1] * k.y, f, g.y);
      s[t][4 * b + 2] = fmaf(s[t][4 * b + 2] * k.z, f, g.z);
      s[t][4 * b + 3] = fmaf(s[t][4 * b + 3] * k.w, f, g.w);
    }
}
// weights of keys whose value norm counts as nothing
template <int NT> __device__ __forceinline__ void ck_drop(ck_f16v (&s)[NT], const float* __restrict__ keep) {
  const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const float4 k = *(const float4*)(keep + 32 * t + 8 * b + 4 * h);
      s[t][4 * b] *= k.x; s[t][4 * b + 1] *= k.y; s[t][4 * b + 2] *= k.z; s[t][4 * b + 3] *= k.w;
    }
}
// keys that the row at position `pos` does not see: from `base` on, NT x 32 of them
template <int NT> __device__ __forceinline__ void ck_mask(ck_f16v (&s)[NT], int base, int pos, int window) {
  const int h = (threadIdx.x & 63) >> 5;
  const int oldest = window > 0 ? pos - window : -1;      // the last key that is too old
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int key = base + 32 * t + 8 * (i >> 2) + 4 * h + (i & 3);
      s[t][i] = key <= pos && key > oldest ? s[t][i] : -INFINITY;
    }
}

// ---- rows and outputs of a tile -----------------------------------------------------------------------------------------
struct ck_lane {                 // the row of a lane
  int token, head, pos;          // query token of the call, query head, position (-1: no row, sees nothing)
  bool valid;
};
__device__ __forceinline__ ck_lane ck_row_of(const ck_args& a, const ck_seq& s, int t0, int t1, int head, int row) {
  // head: kv head x HS + group of query heads
  const int j = row / a.GC, g = (head % a.HS) * a.GC + row - j * a.GC;
  ck_lane r;
  r.valid = t0 + j < t1 && g < a.G;
  r.token = r.valid ? s.q0 + t0 + j : 0;
  r.head = r.valid ? (head / a.HS) * a.G + g : 0;
  r.pos = r.valid ? s.ctx - s.n + t0 + j : -1;
  return r;
}
// quad c of a row's outputs: coordinates 32 (c / 4) + 8 (c % 4) + 4 h .. + 3, finished
template <int D, int KIND>
__device__ __forceinline__ void ck_store(const ck_args& a, int token, int head, int c, float x, float y, float z, float w) {
  const int d = 8 * c + 4 * ((threadIdx.x & 63) >> 5);
  if constexpr (ck_math<KIND>::packed) {
    *(float4*)((float*)a.out + (int64_t)token * a.os_tok + (int64_t)head * a.os_head + d) = make_float4(x, y, z, w);
  } else {
    ck_u2 v;
    v[0] = ck_math<KIND>::pair(x, y);
    v[1] = ck_math<KIND>::pair(z, w);
    *(ck_u2*)((uint16_t*)a.out + (int64_t)token * a.os_tok + (int64_t)head * a.os_head + d) = v;
  }
}
// what the sums of a row are multiplied with in the end
template <int KIND> __device__ __forceinline__ float ck_finish(float l, float unit) { return l == 0.f ? 0.f : (ck_math<KIND>::packed ? unit / l : 1.f / l); }

// bytes of a cache row of D coordinates
template <int D, int KIND> constexpr int ck_row_bytes() { return KIND >= 2 ? D * KIND / 8 : 2 * D; }

// byte or element offsets of a key: its block (clamped into the cache) and place there
struct ck_place_of { int64_t blk; int pos; };
__device__ __forceinline__ ck_place_of ck_key(const ck_args& a, int seq, int key, bool there) {
  ck_place_of p = {0, 0};
  if (there) {
    uint32_t rem;
    const uint32_t b = akv_div32((uint32_t)key, (uint32_t)a.block_size, a.bs_recip, rem);
    p.blk = akv_clamp_block(akv_load_index(a.tables, a.tables_it, (int64_t)seq * a.bt_stride + b), a.num_blocks);
    p.pos = (int)rem;
  }
  return p;
}

template <int W> __device__ __forceinline__ void ck_load_words(uint32_t (&w)[W], const uint8_t* __restrict__ p) {
  // rows lie at multiples of four bytes
  struct __attribute__((packed, aligned(4))) words { uint32_t v[W]; };
  const words x = *(const words*)p;
#pragma unroll
  for (int i = 0; i < W; ++i) w[i] = x.v[i];
}

// ---- few rows a sequence ---------------------------------------------------------------------------------------------------
// A tile is 32 rows, a unit 128 keys: each of the four wavefronts takes 32 of them on its own, keys straight from memory into the
// operand, values through its own part of LDS; what the four hold of the tile is added at the end of the tile or range.  No barrier
// inside.  Reading the cache bounds it.
template <int D, int KIND> struct ck_narrow {
  static constexpr int ROWS = 32, N = 128, THREADS = 256;
  static constexpr int KS = D / 16, DT = D / 32, QUADS = D / 8;
  static constexpr int PITCH = 2 * D + 32;                            // bytes of a value row in LDS: eight rows meet all banks
  static constexpr int V_BYTES = 32 * PITCH;
  static constexpr int MERGE_BYTES = 4 * QUADS * 64 * 16;             // the sums of four wavefronts
  static constexpr int LDS = 4 * V_BYTES > MERGE_BYTES ? 4 * V_BYTES : MERGE_BYTES;
};

template <int D, int KIND>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void ck_narrow_kernel(ck_args a) {
  typedef ck_narrow<D, KIND> P;
  typedef ck_math<KIND> M;
  constexpr bool PACKED = M::packed;
  constexpr int BITS = PACKED ? KIND : 4;
  constexpr int KS = P::KS, DT = P::DT;
  constexpr int HW = D * BITS / 64;                // packed: words of half a row
  __shared__ __align__(16) unsigned char lds[P::LDS];
  __shared__ ck_lengths<256> L;
  __shared__ float ml[4][64][2];
  __shared__ __align__(16) float nrm[PACKED ? 4 : 1][4][32];     // per wavefront: key norms, log2 and inverse of value norms, whether they count
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, col = lane & 31;
  const int G = gridDim.x;
  const int g = G % 8 == 0 ? (int)(blockIdx.x % 8) * (G / 8) + (int)(blockIdx.x / 8) : (int)blockIdx.x;
  const int TM = P::ROWS / a.GC;

  ck_load_lengths(a, L);
  const int per_head = ck_total<256, P::N>(a, L, TM);
  const int heads = a.KVH * a.HS;
  const int64_t total = (int64_t)per_head * heads;
  int64_t at = ck_begin(total, g, G);
  const int64_t end = ck_begin(total, g + 1, G);
  if (tid == 0) a.rec[g].valid = 0;
  if (at >= end) return;
  int head = (int)(at / per_head), seq, tile, first;
  ck_find<256, P::N>(a, L, TM, (int)(at - (int64_t)head * per_head), seq, tile, first);
  int64_t tile_at = (int64_t)head * per_head + first;        // the tile's first unit on the axis

  ck_table<BITS> table;
  if constexpr (PACKED) table.load(a.centroids);

  for (;;) {
    const ck_seq s = ck_sequence(a, L, seq);
    const ck_range keys = ck_keys<P::N>(a, s, tile, TM);
    const int t0 = tile * TM, t1 = min(s.n, t0 + TM);
    const int u0 = (int)(at - tile_at), u1 = (int)min((int64_t)keys.units, end - tile_at);
    const ck_lane row = ck_row_of(a, s, t0, t1, head, col);
    const int kvh = head / a.HS;
    const int pos_first = s.ctx - s.n + t0, pos_last = s.ctx - s.n + t1 - 1;
    // the rows: columns of the operand
    ck_u4 q[KS];
    float fac = 1.f;
    {
      const uint16_t* p = (const uint16_t*)a.q + (int64_t)row.token * a.qs_tok + (int64_t)row.head * a.qs_head;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int grp = PACKED ? KS * h + ks : 2 * ks + h;
        q[ks] = row.valid ? *(const ck_u4*)(p + 8 * grp) : (ck_u4){0u, 0u, 0u, 0u};
      }
      if constexpr (PACKED) fac = row.valid ? a.qfac[(int64_t)row.token * a.QH + row.head] * table.up : 0.f;
    }
    ck_f16v o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = (ck_f16v)(0.f);
    ck_row st = {-INFINITY, 0.f};

    // 32 keys of the wavefront, a lane its half of one
    const int base0 = (keys.first + u0) * P::N + 32 * wave, steps = u1 - u0;
    ck_place_of at0 = ck_key(a, seq, base0 + col, steps > 0 && base0 + col < keys.hi);
    ck_u4 kd[PACKED ? 1 : KS], vd[PACKED ? 1 : KS];
    uint32_t kw[PACKED ? HW : 1], vw[PACKED ? HW : 1];
    float kn = 0.f, vn = 0.f;
    auto request = [&](const ck_place_of& p, bool there) {
      if constexpr (PACKED) {
        if (there) {
          ck_load_words(kw, a.k + p.blk * a.k_blk + p.pos * a.k_pos + kvh * a.k_head + 4 * HW * h);
          ck_load_words(vw, a.v + p.blk * a.v_blk + p.pos * a.v_pos + kvh * a.v_head + 4 * HW * h);
          kn = a.kn[p.blk * a.kn_blk + p.pos * a.kn_pos + kvh * a.kn_head];
          vn = a.vn[p.blk * a.vn_blk + p.pos * a.vn_pos + kvh * a.vn_head];
        } else {
#pragma unroll
          for (int i = 0; i < HW; ++i) kw[i] = vw[i] = 0u;
          kn = 0.f;
          vn = 1.f;
        }
      } else {
        const uint8_t* k = a.k + p.blk * a.k_blk + p.pos * a.k_pos + kvh * a.k_head + 16 * h;
        const uint8_t* v = a.v + p.blk * a.v_blk + p.pos * a.v_pos + kvh * a.v_head + 16 * h;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          kd[ks] = there ? *(const ck_u4*)(k + 32 * ks) : (ck_u4){0u, 0u, 0u, 0u};
          vd[ks] = there ? *(const ck_u4*)(v + 32 * ks) : (ck_u4){0u, 0u, 0u, 0u};
        }
      }
    };
    request(at0, base0 + col < keys.hi);
    ck_place_of next = ck_key(a, seq, base0 + P::N + col, steps > 1 && base0 + P::N + col < keys.hi);
    unsigned char* vl = lds + wave * P::V_BYTES;
    __syncthreads();               // (LDS of the tile before has been read)
    for (int u = 0; u < steps; ++u) {
      const int base = base0 + u * P::N;
      // ---- values to LDS, products of keys and rows
      ck_f16v sc[1];
      sc[0] = (ck_f16v)(0.f);
      bool drop = false;
      if constexpr (PACKED) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          *(ck_u4*)(vl + col * P::PITCH + 16 * (KS * h + ks)) = ck_levels<BITS>(table, vw, ks);
          sc[0] = M::mfma(ck_levels<BITS>(table, kw, ks), q[ks], sc[0]);
        }
        drop = __ballot(vn < CK_TINY) != 0;
        if (h == 0) {
          const float v = vn < CK_TINY ? 1.f : vn;
          nrm[wave][0][col] = kn;
          nrm[wave][1][col] = __log2f(v);
          nrm[wave][2][col] = 1.f / v;
          nrm[wave][3][col] = vn < CK_TINY ? 0.f : 1.f;
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          *(ck_u4*)(vl + col * P::PITCH + 16 * (2 * ks + h)) = vd[ks];
          sc[0] = M::mfma(kd[ks], q[ks], sc[0]);
        }
      }
      // ---- the next keys fly from here on
      if (u + 1 < steps) {
        request(next, base + P::N + col < keys.hi);
        next = ck_key(a, seq, base + 2 * P::N + col, u + 2 < steps && base + 2 * P::N + col < keys.hi);
      }
      akv_wave_sync();
      if (base < keys.hi) {
        if constexpr (PACKED) ck_norms(sc, fac, nrm[wave][0], nrm[wave][1]);
        if (base + 31 > pos_first || (a.window > 0 && base <= pos_last - a.window)) ck_mask(sc, base, row.pos, a.window);
        const float alpha = ck_softmax<1, PACKED>(sc, st, PACKED ? 1.f : a.scale2, PACKED ? nrm[wave][2] : nullptr);
        if constexpr (PACKED)
          if (drop) ck_drop(sc, nrm[wave][3]);
        if (__ballot(alpha != 1.f)) {
#pragma unroll
          for (int i = 0; i < DT; ++i) o[i] *= alpha;
        }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          ck_u4 p;
#pragma unroll
          for (int i = 0; i < 4; ++i) p[i] = M::pair(sc[0][8 * kb + 2 * i], sc[0][8 * kb + 2 * i + 1]);
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            // keys 16 kb + 4 h .. + 3 and + 8, coordinate 32 dt + lane % 32
            unsigned char* at_v = vl + (16 * kb + 4 * h + (lane & 15) / 4) * P::PITCH + 64 * dt + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
            const ck_s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ck_lds_s4*)at_v);
            const ck_s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ck_lds_s4*)(at_v + 8 * P::PITCH));
            const ck_u2 xu = __builtin_bit_cast(ck_u2, x), yu = __builtin_bit_cast(ck_u2, y);
            o[dt] = M::mfma((ck_u4){xu[0], xu[1], yu[0], yu[1]}, p, o[dt]);
          }
        }
      }
      akv_wave_sync();             // (the next values go where these are)
    }

    // ---- the four wavefronts' sums of the tile: wavefront w ends up with a quarter of the coordinates
    st.l += akv_lane_xor<32>(st.l);
    ml[wave][lane][0] = st.m;
    ml[wave][lane][1] = st.l;
    __syncthreads();
    float m = ml[0][lane][0];
#pragma unroll
    for (int w = 1; w < 4; ++w) m = fmaxf(m, ml[w][lane][0]);
    const float c = PACKED ? 1.f : a.scale2, ref = m == -INFINITY ? 0.f : m * c;
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) l += ml[w][lane][1] * ck_exp2(fmaf(ml[w][lane][0], c, -ref));
    const float mine = ck_exp2(fmaf(st.m, c, -ref));
    float4* merge = (float4*)lds;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        merge[(wave * P::QUADS + 4 * dt + b) * 64 + lane] = make_float4(o[dt][4 * b] * mine, o[dt][4 * b + 1] * mine, o[dt][4 * b + 2] * mine, o[dt][4 * b + 3] * mine);
    __syncthreads();
    const bool whole = u0 == 0 && u1 == keys.units;
    const float f = ck_finish<KIND>(l, PACKED ? table.up : 1.f);
    const int64_t slot = 2 * (int64_t)g + (u0 == 0 ? 1 : 0);
#pragma unroll
    for (int i = 0; i < P::QUADS / 4; ++i) {
      const int cq = (P::QUADS / 4) * wave + i;
      float4 x = merge[cq * 64 + lane];
#pragma unroll
      for (int w = 1; w < 4; ++w) {
        const float4 y = merge[(w * P::QUADS + cq) * 64 + lane];
        x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
      }
      if (whole) {
        if (row.valid) ck_store<D, KIND>(a, row.token, row.head, cq, x.x * f, x.y * f, x.z * f, x.w * f);
      } else {
        ((float4*)a.part)[(slot * P::QUADS + cq) * 64 + lane] = x;
      }
    }
    if (!whole && wave == 0) {
      a.part_ml[slot * 64 + lane] = make_float2(m, l);
      if (u0 == 0 && lane == 0) a.rec[g] = {tile_at + keys.units, total, 1, head, s.q0 + t0, t1 - t0};
    }
    // ---- on to the next tile
    at = tile_at + u1;
    if (at >= end) return;
    tile_at += keys.units;
    ++tile;
    int n = s.n;
    while ((int64_t)tile * TM >= n) {
      tile = 0;
      if (++seq > a.S) { seq = 0; ++head; }
      n = ck_sequence(a, L, seq).n;
    }
  }
}

// ---- many rows a sequence -----------------------------------------------------------------------------------------------------
// A tile is 32 rows a wavefront, a unit 64 keys, which the wavefronts of the workgroup share in LDS, in two buffers: while one is multiplied the
// next is requested into registers.  Matrix cores and the vector work of the softmax bound it.
template <int D, int KIND> struct ck_wide {
  static constexpr int WAVES = 4, THREADS = 64 * WAVES, ROWS = 32 * WAVES, N = 64;
  static constexpr int KS = D / 16, DT = D / 32, QUADS = D / 8;
  static constexpr int PITCH = 2 * D + 32;
  static constexpr int TILE = N * PITCH;
  static constexpr int NORMS = KIND >= 2 ? 4 * N * 4 : 0;
  static constexpr int BUF = 2 * TILE + NORMS;
  static constexpr int LDS = 2 * BUF;
};

template <int D, int KIND>
__global__ __launch_bounds__((ck_wide<D, KIND>::THREADS), D == 256 ? 1 : 2) void ck_wide_kernel(ck_args a) {
  typedef ck_wide<D, KIND> P;
  typedef ck_math<KIND> M;
  constexpr bool PACKED = M::packed;
  constexpr int BITS = PACKED ? KIND : 4;
  constexpr int KS = P::KS, DT = P::DT, N = P::N, T = P::THREADS;
  constexpr int CPR = D / 8;                                  // dense: pieces of 16 bytes a row
  constexpr int NP = N * CPR / T;                             // pieces of K, and of V, a thread
  constexpr int TPR = D / 32, TASKS = N * TPR, NT = (TASKS + T - 1) / T;      // packed: 32 codes a task
  extern __shared__ __align__(16) unsigned char lds[];
  __shared__ ck_lengths<T> L;
  __shared__ int64_t place_blk[2][N];
  __shared__ int place_pos[2][N];
  __shared__ int drops[2];                                    // packed: value norms of the unit that count as nothing
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, col = lane & 31;
  const int G = gridDim.x;
  const int g = G % 8 == 0 ? (int)(blockIdx.x % 8) * (G / 8) + (int)(blockIdx.x / 8) : (int)blockIdx.x;
  const int TM = P::ROWS / a.GC;

  ck_load_lengths(a, L);
  const int per_head = ck_total<T, N>(a, L, TM);
  const int heads = a.KVH * a.HS;
  const int64_t total = (int64_t)per_head * heads;
  int64_t at = ck_begin(total, g, G);
  const int64_t end = ck_begin(total, g + 1, G);
  if (tid == 0) a.rec[g].valid = 0;
  if (at >= end) return;
  int head = (int)(at / per_head), seq, tile, first;
  ck_find<T, N>(a, L, TM, (int)(at - (int64_t)head * per_head), seq, tile, first);
  int64_t tile_at = (int64_t)head * per_head + first;

  ck_table<BITS> table;
  if constexpr (PACKED) table.load(a.centroids);

  for (;;) {
    const ck_seq s = ck_sequence(a, L, seq);
    const ck_range keys = ck_keys<N>(a, s, tile, TM);
    const int t0 = tile * TM, t1 = min(s.n, t0 + TM);
    const int u0 = (int)(at - tile_at), u1 = (int)min((int64_t)keys.units, end - tile_at), steps = u1 - u0;
    const ck_lane row = ck_row_of(a, s, t0, t1, head, 32 * wave + col);
    const int kvh = head / a.HS;
    // positions of the wavefront's rows
    const int w0 = t0 + 32 * wave / a.GC, w1 = min(t1, t0 + (32 * wave + 31) / a.GC + 1);
    const int pos_first = s.ctx - s.n + w0, pos_last = w0 < t1 ? s.ctx - s.n + w1 - 1 : -1;
    ck_u4 q[KS];
    float fac = 1.f;
    {
      const uint16_t* p = (const uint16_t*)a.q + (int64_t)row.token * a.qs_tok + (int64_t)row.head * a.qs_head;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) q[ks] = row.valid ? *(const ck_u4*)(p + 8 * (2 * ks + h)) : (ck_u4){0u, 0u, 0u, 0u};
      if constexpr (PACKED) fac = row.valid ? a.qfac[(int64_t)row.token * a.QH + row.head] * table.up : 0.f;
    }
    ck_f16v o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = (ck_f16v)(0.f);
    ck_row st = {-INFINITY, 0.f};

    const int base0 = (keys.first + u0) * N;
    ck_u4 kd[PACKED ? 1 : NP], vd[PACKED ? 1 : NP];
    uint32_t kw[PACKED ? NT : 1][BITS], vw[PACKED ? NT : 1][BITS];
    float kn = 0.f, vn = 1.f;
    // places of a unit's keys, by the first threads
    auto look = [&](int u) { return ck_key(a, seq, base0 + u * N + tid, tid < N && u < steps && base0 + u * N + tid < keys.hi); };
    auto note = [&](int u, const ck_place_of& p) {
      if (tid < N) {
        place_blk[u & 1][tid] = p.blk;
        place_pos[u & 1][tid] = p.pos;
      }
    };
    auto request = [&](int u) {
      const int b = u & 1, limit = keys.hi - (base0 + u * N);
      if constexpr (PACKED) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const int task = tid + T * i, r = task / TPR, part = task % TPR;
          if (task < TASKS && r < limit) {
            const int64_t blk = place_blk[b][r];
            const int pos = place_pos[b][r];
            ck_load_words(kw[i], a.k + blk * a.k_blk + pos * a.k_pos + kvh * a.k_head + 4 * BITS * part);
            ck_load_words(vw[i], a.v + blk * a.v_blk + pos * a.v_pos + kvh * a.v_head + 4 * BITS * part);
          } else {
#pragma unroll
            for (int j = 0; j < BITS; ++j) kw[i][j] = vw[i][j] = 0u;
          }
        }
        kn = 0.f;
        vn = 1.f;
        if (tid < N && tid < limit) {
          const int64_t blk = place_blk[b][tid];
          const int pos = place_pos[b][tid];
          kn = a.kn[blk * a.kn_blk + pos * a.kn_pos + kvh * a.kn_head];
          vn = a.vn[blk * a.vn_blk + pos * a.vn_pos + kvh * a.vn_head];
        }
      } else {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int c = tid + T * i, r = c / CPR, part = c % CPR;
          if (r < limit) {
            const int64_t blk = place_blk[b][r];
            const int pos = place_pos[b][r];
            kd[i] = *(const ck_u4*)(a.k + blk * a.k_blk + pos * a.k_pos + kvh * a.k_head + 16 * part);
            vd[i] = *(const ck_u4*)(a.v + blk * a.v_blk + pos * a.v_pos + kvh * a.v_head + 16 * part);
          } else {
            kd[i] = vd[i] = (ck_u4){0u, 0u, 0u, 0u};
          }
        }
      }
    };
    auto put = [&](int u) {
      unsigned char* kt = lds + (u & 1) * P::BUF;
      unsigned char* vt = kt + P::TILE;
      if constexpr (PACKED) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const int task = tid + T * i, r = task / TPR, part = task % TPR;
          if (TASKS % T == 0 || task < TASKS) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              *(ck_u4*)(kt + r * P::PITCH + 64 * part + 16 * j) = ck_levels<BITS>(table, kw[i], j);
              *(ck_u4*)(vt + r * P::PITCH + 64 * part + 16 * j) = ck_levels<BITS>(table, vw[i], j);
            }
          }
        }
        if (tid < N) {
          float* nr = (float*)(vt + P::TILE);
          const float v = vn < CK_TINY ? 1.f : vn;
          nr[tid] = kn;
          nr[N + tid] = __log2f(v);
          nr[2 * N + tid] = 1.f / v;
          nr[3 * N + tid] = vn < CK_TINY ? 0.f : 1.f;
          const int drop = __ballot(vn < CK_TINY) != 0;      // (the N threads are the first wavefront)
          if (tid == 0) drops[u & 1] = drop;
        }
      } else {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int c = tid + T * i, r = c / CPR, part = c % CPR;
          *(ck_u4*)(kt + r * P::PITCH + 16 * part) = kd[i];
          *(ck_u4*)(vt + r * P::PITCH + 16 * part) = vd[i];
        }
      }
    };
    __syncthreads();               // (LDS of the tile before has been read)
    note(0, look(0));
    note(1, look(1));
    __syncthreads();
    request(0);
    put(0);
    __syncthreads();
    for (int u = 0; u < steps; ++u) {
      const int base = base0 + u * N;
      ck_place_of ahead = {0, 0};
      if (u + 1 < steps) {
        request(u + 1);
        ahead = look(u + 2);
      }
      if (base <= pos_last && !(a.window > 0 && base + N - 1 <= pos_first - a.window)) {
        const unsigned char* kt = lds + (u & 1) * P::BUF;
        unsigned char* vt = (unsigned char*)kt + P::TILE;
        const float* nr = (const float*)(vt + P::TILE);
        ck_f16v sc[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          sc[t] = (ck_f16v)(0.f);
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) sc[t] = M::mfma(*(const ck_u4*)(kt + (32 * t + col) * P::PITCH + 16 * (2 * ks + h)), q[ks], sc[t]);
        }
        if constexpr (PACKED) ck_norms(sc, fac, nr, nr + N);
        if (base + N - 1 > pos_first || (a.window > 0 && base <= pos_last - a.window)) ck_mask(sc, base, row.pos, a.window);
        const float alpha = ck_softmax<2, PACKED>(sc, st, PACKED ? 1.f : a.scale2, PACKED ? nr + 2 * N : nullptr);
        if constexpr (PACKED)
          if (drops[u & 1]) ck_drop(sc, nr + 3 * N);
        if (__ballot(alpha != 1.f)) {
#pragma unroll
          for (int i = 0; i < DT; ++i) o[i] *= alpha;
        }
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
          ck_u4 p;
#pragma unroll
          for (int i = 0; i < 4; ++i) p[i] = M::pair(sc[kb / 2][8 * (kb & 1) + 2 * i], sc[kb / 2][8 * (kb & 1) + 2 * i + 1]);
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            unsigned char* at_v = vt + (16 * kb + 4 * h + (lane & 15) / 4) * P::PITCH + 64 * dt + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
            const ck_s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ck_lds_s4*)at_v);
            const ck_s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ck_lds_s4*)(at_v + 8 * P::PITCH));
            const ck_u2 xu = __builtin_bit_cast(ck_u2, x), yu = __builtin_bit_cast(ck_u2, y);
            o[dt] = M::mfma((ck_u4){xu[0], xu[1], yu[0], yu[1]}, p, o[dt]);
          }
        }
      }
      if (u + 1 < steps) put(u + 1);
      if (u + 2 < steps) note(u + 2, ahead);
      __syncthreads();
    }

    st.l += akv_lane_xor<32>(st.l);
    const bool whole = u0 == 0 && u1 == keys.units;
    if (whole) {
      const float f = ck_finish<KIND>(st.l, PACKED ? table.up : 1.f);
      if (row.valid) {
#pragma unroll
        for (int c = 0; c < P::QUADS; ++c)
          ck_store<D, KIND>(a, row.token, row.head, c, o[c / 4][4 * (c & 3)] * f, o[c / 4][4 * (c & 3) + 1] * f, o[c / 4][4 * (c & 3) + 2] * f, o[c / 4][4 * (c & 3) + 3] * f);
      }
    } else {
      const int64_t slot = (2 * (int64_t)g + (u0 == 0 ? 1 : 0)) * P::WAVES + wave;
#pragma unroll
      for (int c = 0; c < P::QUADS; ++c)
        ((float4*)a.part)[(slot * P::QUADS + c) * 64 + lane] = make_float4(o[c / 4][4 * (c & 3)], o[c / 4][4 * (c & 3) + 1], o[c / 4][4 * (c & 3) + 2], o[c / 4][4 * (c & 3) + 3]);
      a.part_ml[slot * 64 + lane] = make_float2(st.m, st.l);
      if (u0 == 0 && tid == 0) a.rec[g] = {tile_at + keys.units, total, 1, head, s.q0 + t0, t1 - t0};
    }
    at = tile_at + u1;
    if (at >= end) return;
    tile_at += keys.units;
    ++tile;
    int n = s.n;
    while ((int64_t)tile * TM >= n) {
      tile = 0;
      if (++seq > a.S) { seq = 0; ++head; }
      n = ck_sequence(a, L, seq).n;
    }
  }
}

// ---- the pieces of a tile that several ranges share --------------------------------------------------------------------------
// Workgroup (g, w): the 32 rows w of the tile that begins in range g and does not end there; its other pieces are the first ones of the
// ranges behind.
template <int D, int KIND, int WAVES>
__global__ __launch_bounds__(256) void ck_merge_kernel(ck_args a, int G) {
  constexpr int QUADS = D / 8, MINE = QUADS / 4;
  const int g = blockIdx.x, part = blockIdx.y;
  const ck_record rec = a.rec[g];
  if (!rec.valid) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31;
  const float c = ck_math<KIND>::packed ? 1.f : a.scale2;
  float m = -INFINITY, l = 0.f;
  float4 x[MINE];
#pragma unroll
  for (int i = 0; i < MINE; ++i) x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](int64_t slot) {
    const float2 e = a.part_ml[(slot * WAVES + part) * 64 + lane];
    const float mn = fmaxf(m, e.x), ref = mn == -INFINITY ? 0.f : mn * c;
    const float f0 = ck_exp2(fmaf(m, c, -ref)), f1 = ck_exp2(fmaf(e.x, c, -ref));
    l = l * f0 + e.y * f1;
    m = mn;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      const float4 y = ((const float4*)a.part)[((slot * WAVES + part) * QUADS + MINE * wave + i) * 64 + lane];
      x[i].x = x[i].x * f0 + y.x * f1; x[i].y = x[i].y * f0 + y.y * f1;
      x[i].z = x[i].z * f0 + y.z * f1; x[i].w = x[i].w * f0 + y.w * f1;
    }
  };
  add(2 * (int64_t)g + 1);
  for (int r = g + 1; r < G; ++r) {
    const int64_t b = ck_begin(rec.total, r, G), e = ck_begin(rec.total, r + 1, G);
    if (b >= rec.end) break;
    if (b < e) add(2 * (int64_t)r);
  }
  const int row = 32 * part + col, j = row / a.GC, gq = (rec.head % a.HS) * a.GC + row - j * a.GC;
  if (j >= rec.tokens || gq >= a.G) return;
  float unit = 1.f;
  if constexpr (ck_math<KIND>::packed) {
    ck_table<KIND> t;
    t.load(a.centroids);
    unit = t.up;
  }
  const float f = ck_finish<KIND>(l, unit);
#pragma unroll
  for (int i = 0; i < MINE; ++i)
    ck_store<D, KIND>(a, rec.token + j, (rec.head / a.HS) * a.G + gq, MINE * wave + i, x[i].x * f, x[i].y * f, x[i].z * f, x[i].w * f);
}


// ---- launches ---------------------------------------------------------------------------------------------------------------------
// Scratch of the main kernels: a record a workgroup, and the pieces of two tiles (the sums of 32 rows, QUADS x 64 x 16 bytes, and their
// maxima and sums of weights) a wavefront of rows.
static inline int ck_groups(int per_cu) {
  const int cus = akv_cached_cu_count();
  return (cus > 0 ? cus : 256) * per_cu;
}
struct ck_scratch { size_t rec, ml, part, bytes; };
static inline ck_scratch ck_scratch_layout(int D) {
  const size_t g = (size_t)ck_groups(2), slots = 2 * g * 4;          // (the wide kernel's: four times the narrow one's)
  ck_scratch w;
  w.rec = 0;
  w.ml = akv_align256(g * sizeof(ck_record));
  w.part = w.ml + akv_align256(slots * 64 * sizeof(float2));
  w.bytes = w.part + slots * (size_t)(D / 8) * 64 * 16;
  return w;
}
static inline uint32_t ck_reciprocal(int d) { return (uint32_t)(0xffffffffull / (uint32_t)d); }

template <int D, int KIND>
static int ck_launch(ck_args a, int most_new, void* scratch, hipStream_t stream) {
  typedef ck_wide<D, KIND> W;
  const ck_scratch w = ck_scratch_layout(D);
  a.rec = (ck_record*)((char*)scratch + w.rec);
  a.part_ml = (float2*)((char*)scratch + w.ml);
  a.part = (float*)((char*)scratch + w.part);
  // Few rows a sequence as far as the host can tell: the narrow kernel takes all of them.  One sequence of more: the wide one.  Otherwise
  // each takes its own, by the lengths on the device.
  const int64_t most = most_new > 0 && most_new < a.T ? most_new : a.T;
  const bool few = most * a.G <= CK_NARROW_ROWS, one = !few && a.S == 1;
  if (!one) {
    ck_args n = a;
    n.kind = few ? 0 : 1;
    n.HS = (a.G + 31) / 32;
    n.GC = (a.G + n.HS - 1) / n.HS;
    const int G = ck_groups(D == 256 ? 1 : 2);
    ck_narrow_kernel<D, KIND><<<G, 256, 0, stream>>>(n);
    AKV_LAUNCH_CHECK("ck_narrow_kernel");
    ck_merge_kernel<D, KIND, 1><<<dim3(G, 1), 256, 0, stream>>>(n, G);
    AKV_LAUNCH_CHECK("ck_merge_kernel");
  }
  if (!few) {
    ck_args n = a;
    n.kind = one ? 0 : 2;
    n.HS = (a.G + W::ROWS - 1) / W::ROWS;
    n.GC = (a.G + n.HS - 1) / n.HS;
    static akv_device_once once;
    int dev = 0;
    AKV_HIP(hipGetDevice(&dev));
    const int rc = once(dev, [&]() -> int {
      AKV_HIP(hipFuncSetAttribute((const void*)ck_wide_kernel<D, KIND>, hipFuncAttributeMaxDynamicSharedMemorySize, W::LDS));
      return AKV_OK;
    });
    if (rc) return rc;
    const int G = ck_groups(D == 256 ? 1 : 2);
    ck_wide_kernel<D, KIND><<<G, W::THREADS, W::LDS, stream>>>(n);
    AKV_LAUNCH_CHECK("ck_wide_kernel");
    ck_merge_kernel<D, KIND, W::WAVES><<<dim3(G, W::WAVES), 256, 0, stream>>>(n, G);
    AKV_LAUNCH_CHECK("ck_merge_kernel");
  }
  return AKV_OK;
}

static inline bool ck_aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
// what both entry points ask of a call's batch
static inline int ck_check_batch(const char* name, const void* query, int dtype, const void* tables, int tables_it, const void* lens, int lens_it,
                                 const void* starts, int starts_it, const void* out, int S, int64_t T, int QH, int KVH, int D, int block_size, int64_t num_blocks, int64_t max_blocks, float scale) {
  AKV_REQUIRE(akv_valid_dtype(dtype), "%s: bad dtype %d", name, dtype);
  AKV_REQUIRE(akv_valid_itype(tables_it) && akv_valid_itype(lens_it) && akv_valid_itype(starts_it), "%s: bad index type", name);
  AKV_REQUIRE(S >= 0 && T >= 0 && QH > 0 && KVH > 0 && QH % KVH == 0, "%s: %d sequences, %lld tokens, %d query heads on %d kv heads", name, S, (long long)T, QH, KVH);
  AKV_REQUIRE(block_size > 0 && num_blocks >= 0 && max_blocks >= 0, "%s: bad block_size %d, num_blocks %lld or max_blocks_per_seq %lld", name, block_size, (long long)num_blocks, (long long)max_blocks);
  AKV_REQUIRE(scale > 0.f && scale < INFINITY, "%s: scale must be positive and finite", name);
  if (T == 0) return AKV_OK;
  AKV_REQUIRE(query && out && starts, "%s: null pointer", name);
  AKV_REQUIRE(S == 0 || lens, "%s: null pointer", name);
  AKV_REQUIRE(S == 0 || max_blocks == 0 || num_blocks == 0 || tables, "%s: null pointer", name);
  if (dtype == AKV_F32) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: float32 queries are not supported; use float16 or bfloat16", name);
  if (D != 64 && D != 128 && D != 256) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: head_dim %d; kernels are built for 64, 128 and 256", name, D);
  if (T > 0x3fffffff || S > 0x3fffffff || T * (int64_t)QH > 0x7fffffff) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: more than 2^31 rows", name);
  return AKV_OK;
}
