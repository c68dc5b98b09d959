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
// Packed rows are attended in the rotated domain: queries are rotated on the way in, results on the way out (akv_chunk_rotate.h), and in
// between a key is its norm times levels of the codebook.  Levels are float16 in a unit that loses little of them (ck_unit_key); a key's
// norm multiplies its score in float32; a value's norm v goes into the exponent, w = 2^(s + log2 v - M), with M from the running maximum of
// s + log2 v, so weights stay in [0, 2^(CK_LIFT + CK_FRAME)] for norms of any size, and the sum of the softmax takes w / v.
//
// What is rounded to sixteen bits: the weights, once, as operand of the second product (relative 2^-11 or 2^-8, as of the values beside them;
// float16 ones, those over packed rows in either type, besides by 2^-30 of the row's largest); packed: the levels (2^-14) and the queries (many
// rows: one float16 term; few rows: two, 2^-22).  Scores, maxima, sums and results are float32.
#pragma once
#include "akv_chunk_rotate.h"
#include "akv_device_once.h"
#include <climits>
#include <type_traits>

// Smallest value norm that counts (its inverse times weights of 2^13, summed over a cache, is finite).  A value of a smaller one,
// such as 0, is zero, and in the exponents its norm is CK_NONE: far below those that come with it, or its score would lift the frame of the row
// past what the others have to give (as 1 it made float16 zeros of values 2^-26 in size); no further below than that weight times inverse,
// which the sum of the softmax still takes, are float32 numbers beside norms of up to 2^80.
#define CK_TINY 0x1p-80f
#define CK_NONE 0x1p-40f

// ---- packed codes -> float16 levels -----------------------------------------------------------------------------
// Value of the levels' last place, so to say: a level is a float16 number times this.  Any unit would do (scores take it with the key's norm,
// outputs in the end); of 64 N between two powers of two the one is picked whose float16 levels are nearest to the codebook.  With 64 the
// sixteen levels of four bits are off by a third of what a power of two leaves, 2^-13.6 of themselves instead of 2^-12; with 1024 by a quarter.
// `own`: level lane % 2^BITS.  ck_unit_key: the best of the units from..from + N - 1 of every lane of a wavefront, as a number that is less
// for a better one; ck_unit_of: the unit.
template <int BITS> __device__ __forceinline__ float ck_largest_level(float own, float (&c)[1 << BITS]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < (1 << BITS); ++i) {
    c[i] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(own), i));
    m = fmaxf(m, fabsf(c[i]));
  }
  return m;
}
template <int BITS, int N, int TOTAL> __device__ __forceinline__ uint32_t ck_unit_key(float own, int from) {
  float c[1 << BITS];
  // the largest to [16, 32) x (1 .. 2): levels down to 2^-18 of it are normal numbers
  const float up = akv_row_scale(akv_row_exponent(ck_largest_level<BITS>(own, c)));
  uint32_t best = 0xffffffffu;
#pragma unroll 1
  for (int n = from; n < from + N; ++n) {
    const float s = 16.f + (16.f / TOTAL) * (float)n;
    float off = 0.f;
#pragma unroll
    for (int i = 0; i < (1 << BITS); ++i) {
      const float x = c[i] * (up * s), e = (float)(_Float16)x - x;
      off = fmaf(e, e, off);
    }
    off *= __builtin_amdgcn_rcpf(s * s);
    // the least, of equal ones the first; a codebook that is not finite leaves the first
    best = min(best, (off < INFINITY ? __float_as_uint(off) & ~(uint32_t)(TOTAL - 1) : 0x7f800000u) | (uint32_t)n);
  }
  best = min(best, akv_lane_xor_u32<32>(best)); best = min(best, akv_lane_xor_u32<16>(best)); best = min(best, akv_lane_xor_u32<8>(best));
  best = min(best, akv_lane_xor_u32<4>(best)); best = min(best, akv_lane_xor_u32<2>(best)); best = min(best, akv_lane_xor_u32<1>(best));
  return best;
}
template <int BITS, int TOTAL> __device__ __forceinline__ float ck_unit_of(float own, uint32_t key) {
  float c[1 << BITS];
  const float s = 16.f + (16.f / TOTAL) * (float)(__builtin_amdgcn_readfirstlane((int)key) & (TOTAL - 1));
  return akv_row_unscale(akv_row_exponent(ck_largest_level<BITS>(own, c))) / s;
}
// Levels from a table in LDS, of two codes at a time (four where a byte holds them).  COPIES of 64: every lane has its own, so that no two
// meet a bank (a shared table of 256 entries cost 9 clocks a look-up: lanes meet banks, codes in the middle are frequent).
template <int BITS, int COPIES> struct ck_lut {
  static constexpr bool OWN = COPIES == 64;
  static constexpr int ENTRIES = BITS == 3 ? 64 : OWN && BITS == 2 ? 16 : 256, WORDS = BITS == 2 && !OWN ? 2 : 1;
  uint32_t level[ENTRIES * WORDS * COPIES];
  __device__ __forceinline__ void fill(const float* __restrict__ centroids, int tid, int threads, float unit) {
    constexpr int M = (1 << BITS) - 1;
    // (a lane a level, looked up across the wavefront: every entry would wait for memory otherwise)
    const uint32_t mine = __builtin_bit_cast(unsigned short, (_Float16)(centroids[tid & M] * (1.f / unit)));
    auto one = [&](int code) { return (uint32_t)__builtin_amdgcn_ds_bpermute(4 * code, (int)mine); };
    if constexpr (OWN) {
      // sixteen lanes an entry, sixteen bytes each
      for (int i = tid / 16; i < ENTRIES; i += threads / 16) {
        const uint32_t v = one(i >> BITS) | one(i & M) << 16;
        *(ck_u4*)(level + i * 64 + 4 * (tid & 15)) = (ck_u4){v, v, v, v};
      }
    } else {
      for (int i = tid; i < ENTRIES; i += threads) {
        if constexpr (BITS == 2) {
          level[2 * i] = one(i >> 6) | one((i >> 4) & 3) << 16;
          level[2 * i + 1] = one((i >> 2) & 3) | one(i & 3) << 16;
        } else {
          level[i] = one(i >> BITS) | one(i & M) << 16;
        }
      }
    }
  }
  // group g (eight coordinates) of a run of codes that starts at word 0 of `w`
  template <int W> __device__ __forceinline__ ck_u4 group(const uint32_t (&w)[W], int g) const {
    const unsigned char* t = (const unsigned char*)level;
    const uint32_t mine = 4 * (threadIdx.x & 63);
    // (a lane's own table begins where LDS does: the sum of entry and lane is the address)
    auto own = [](uint32_t at) { return *(const __attribute__((address_space(3))) uint32_t*)(uintptr_t)at; };
    ck_u4 r;
    if constexpr (BITS == 4) {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        if constexpr (OWN) r[b] = own(__builtin_amdgcn_perm(w[g], mine, 0x0c0c0000u | (uint32_t)(4 + b) << 8));
        else r[b] = *(const uint32_t*)(t + (b == 0 ? (w[g] << 2) & 0x3fcu : (w[g] >> (8 * b - 2)) & 0x3fcu));
      }
    } else if constexpr (BITS == 3) {
      const int b = 3 * g, i = b >> 2, o = b & 3;
      const uint32_t sel = (uint32_t)(o + 2) | (uint32_t)(o + 1) << 8 | (uint32_t)o << 16 | 0x0c000000u;
      const uint32_t x = __builtin_amdgcn_perm(i + 1 < W ? w[i + 1 < W ? i + 1 : 0] : 0u, w[i], sel);      // 24 bits, the first coordinate on top
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        constexpr int up = OWN ? 8 : 2;
        const int sh = 18 - 6 * p;
        const uint32_t v = (sh >= up ? x >> (sh - up) : x << (up - sh)) & (63u << up);
        if constexpr (OWN) r[p] = own(v | mine);
        else r[p] = *(const uint32_t*)(t + v);
      }
    } else if constexpr (OWN) {
      // nibbles: of a byte the upper first
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const int sh = 16 * (g & 1) + 8 * (p >> 1) + 4 * (1 - (p & 1));
        r[p] = own(((sh >= 8 ? w[g >> 1] >> (sh - 8) : w[g >> 1] << (8 - sh)) & 0xf00u) | mine);
      }
    } else {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int sh = 16 * (g & 1) + 8 * b;
        const ck_u2 v = *(const ck_u2*)(t + (sh < 3 ? (w[g >> 1] << 3) & 0x7f8u : (w[g >> 1] >> (sh - 3)) & 0x7f8u));
        r[2 * b] = v[0];
        r[2 * b + 1] = v[1];
      }
    }
    return r;
  }
};

// ---- one step of the softmax ----------------------------------------------------------------------------------------
// A row's running state: weights are 2^(exponent - m), and l is their sum over the lane's own keys (the halves are added at the end).  m is
// not the maximum so far but lies CK_LIFT to CK_LIFT + CK_FRAME below it: the sums are rescaled only when a row's maximum has outgrown that, and
// weights of up to 2^13 lose nothing, as their rounding is relative and float16 reaches 2^16 (the other 2^3: scores of 2^26 are rounded to
// steps of 8, of which a maximum may be off by half).  What lies far below the largest keeps the more: float16 weights are in steps of 2^-24
// at least, 2^-29 of the largest (with the largest at 1 keys 2^-26 below it were lost however many or large they were).  A frame of 4 under
// a lift of 7 rescales more often: a first chunk of 2048 tokens 75.2 us, this one 72.7.  bfloat16 weights have the range as they are, and
// values that may be of any size beside them: no lift.
#define CK_FRAME 8.f
template <int KIND> constexpr float CK_LIFT = KIND == CK_BF16 ? 0.f : 5.f;
struct ck_row { float m, l; };
// largest of NT tiles of 32 products, over both halves
template <int NT> __device__ __forceinline__ float ck_max(const ck_f16v (&s)[NT]) {
  float a = s[0][0], b = s[0][1];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = t == 0 ? 2 : 0; i < 16; i += 2) {
      a = fmaxf(a, s[t][i]);
      b = fmaxf(b, s[t][i + 1]);
    }
  a = fmaxf(a, b);
  return fmaxf(a, akv_lane_xor<32>(a));
}
// Whether some row's largest exponent has outgrown its frame; `alpha` is then what the row's sums are multiplied with.
template <int KIND> __device__ __forceinline__ bool ck_outgrown(ck_row& r, float mx, float& alpha) {
  const bool grown = mx - r.m > CK_LIFT<KIND> + CK_FRAME;      // (the difference of two numbers so near is exact)
  if (!__ballot(grown)) return false;
  const float m = grown ? mx - CK_LIFT<KIND> : r.m;
  alpha = grown ? ck_exp2(r.m - m) : 1.f;
  r.m = m;
  r.l *= alpha;
  return true;
}
// Products (packed: exponents) to weights, in place; c = scale x log2 e.
template <int NT, bool PACKED>
__device__ __forceinline__ void ck_weights(ck_f16v (&s)[NT], ck_row& r, float c, const float* __restrict__ inv) {
  const float ref = r.m == -INFINITY ? 0.f : r.m;
  const int h = (threadIdx.x & 63) >> 5;
  float l0 = 0.f, l1 = 0.f;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = ck_exp2(PACKED ? s[t][4 * b + e] - ref : fmaf(s[t][4 * b + e], c, -ref));
      if constexpr (PACKED) {
        const float4 v = *(const float4*)(inv + 32 * t + 8 * b + 4 * h);
        l0 = fmaf(w[0], v.x, l0); l1 = fmaf(w[1], v.y, l1);
        l0 = fmaf(w[2], v.z, l0); l1 = fmaf(w[3], v.w, l1);
      } else {
        l0 += w[0]; l1 += w[1];
        l0 += w[2]; l1 += w[3];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) s[t][4 * b + e] = w[e];
    }
  r.l += l0 + l1;
}
// Products to exponents: s x (key norm x unit of the levels) + log2 of the value norm, norms of 32 NT keys from LDS.
template <int NT>
__device__ __forceinline__ void ck_norms(ck_f16v (&s)[NT], const float* __restrict__ kn, const float* __restrict__ lg) {
  const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const float4 k = *(const float4*)(kn + 32 * t + 8 * b + 4 * h), g = *(const float4*)(lg + 32 * t + 8 * b + 4 * h);
      s[t][4 * b] = fmaf(s[t][4 * b], k.x, g.x);
      s[t][4 * b + 1] = fmaf(s[t][4 * b + 1], k.y, g.y);
      s[t][4 * b + 2] = fmaf(s[t][4 * b + 2], k.z, g.z);
      s[t][4 * b + 3] = fmaf(s[t][4 * b + 3], k.w, g.w);
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
  int token, head, pos;          // query token of the call, query head, position (below 0: no row, or one before the first key, sees nothing)
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
// quad c of a row's outputs: coordinates 8 c + 4 h .. + 3, finished
template <int KIND>
__device__ __forceinline__ void ck_store(const ck_args& a, int token, int head, int c, float x, float y, float z, float w) {
  const int d = 8 * c + 4 * ((threadIdx.x & 63) >> 5);
  ck_u2 v;
  if (ck_math<KIND>::packed && a.dtype == AKV_BF16) {
    v[0] = ck_math<CK_BF16>::pair(x, y);
    v[1] = ck_math<CK_BF16>::pair(z, w);
  } else {
    v[0] = ck_math<KIND>::pair(x, y);
    v[1] = ck_math<KIND>::pair(z, w);
  }
  *(ck_u2*)((uint16_t*)a.out + (int64_t)token * a.os_tok + (int64_t)head * a.os_head + d) = v;
}
// what the sums of a row are multiplied with in the end
__device__ __forceinline__ float ck_finish(float l) { return l == 0.f ? 0.f : 1.f / l; }

// Results of 32 rows whose coordinates are spread over the W wavefronts of a workgroup, QW quads each, times f.  Packed rows go
// through `rows` (LDS, 32 x (D + 4) floats, which has been read by others) and are turned back.
template <int D, int KIND, int W, int QW, class Matrix>
__device__ __forceinline__ void ck_results(const ck_args& a, const float4 (&x)[QW], float f, const Matrix& matrix, bool valid, int token, int head, float* __restrict__ rows) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, col = lane & 31;
  if constexpr (!ck_math<KIND>::packed) {
    if (valid) {
#pragma unroll
      for (int i = 0; i < QW; ++i) ck_store<KIND>(a, token, head, QW * wave + i, x[i].x * f, x[i].y * f, x[i].z * f, x[i].w * f);
    }
  } else {
    constexpr int ROW = D + 4, KS = D / 16, DT = D / 32;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < QW; ++i) *(float4*)(rows + col * ROW + 8 * (QW * wave + i) + 4 * h) = make_float4(x[i].x * f, x[i].y * f, x[i].z * f, x[i].w * f);
    __syncthreads();
    if (wave < DT) {
      float v[KS][8];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const float4 y = *(const float4*)(rows + col * ROW + 16 * ks + 8 * p + 4 * h);
          v[ks][4 * p] = y.x; v[ks][4 * p + 1] = y.y; v[ks][4 * p + 2] = y.z; v[ks][4 * p + 3] = y.w;
        }
      ck_u4 hi[KS], lo[KS];
      const float un = ck_result_operand<D>([&](int ks, int j) { return v[ks][j]; }, hi, lo) * a.turn_scale->up * (1.f / CK_TURN);
#pragma unroll
      for (int dt = wave; dt < DT; dt += W) {
        const ck_f16v y = matrix.turn(dt, hi, lo);
        if (valid) {
#pragma unroll
          for (int b = 0; b < 4; ++b) ck_store<KIND>(a, token, head, 4 * dt + b, y[4 * b] * un, y[4 * b + 1] * un, y[4 * b + 2] * un, y[4 * b + 3] * un);
        }
      }
    }
  }
}


// A key's entry in the block table, as it is requested (both words of a 64-bit one), and the key's place in the cache from it: the block is clamped
// into the cache.  (Taken apart so that nothing waits for the entry where it is requested.)
struct ck_entry { uint32_t lo, hi; };
__device__ __forceinline__ ck_entry ck_look(const ck_args& a, int seq, int key) {
  uint32_t rem;
  const int wide = a.tables_it == AKV_I64;
  const int64_t i = (int64_t)seq * a.bt_stride + akv_div32((uint32_t)key, (uint32_t)a.block_size, a.bs_recip, rem);
  const uint32_t* p = (const uint32_t*)a.tables + (i << wide);
  return {p[0], p[wide]};
}
struct ck_place { uint32_t blk, pos; };
__device__ __forceinline__ ck_place ck_place_of(const ck_args& a, int key, ck_entry e) {
  ck_place p;
  akv_div32((uint32_t)key, (uint32_t)a.block_size, a.bs_recip, p.pos);
  const int64_t id = a.tables_it == AKV_I64 ? (int64_t)((uint64_t)e.hi << 32 | e.lo) : (int64_t)(int32_t)e.lo;
  p.blk = (uint32_t)akv_clamp_block(id, a.num_blocks);
  return p;
}
__device__ __forceinline__ int64_t ck_offset(ck_place p, int64_t blk, int64_t pos) { return (int64_t)p.blk * blk + (int64_t)p.pos * pos; }

template <int W> __device__ __forceinline__ void ck_load_words(uint32_t (&w)[W], const uint8_t* __restrict__ p) {
  // rows lie at multiples of four bytes
  struct __attribute__((packed, aligned(4))) words { uint32_t v[W]; };
  const words x = *(const words*)p;
#pragma unroll
  for (int i = 0; i < W; ++i) w[i] = x.v[i];
}

// ---- few rows a sequence ---------------------------------------------------------------------------------------------------
// A tile is 32 rows, a unit 32 keys a wavefront: each takes its own, keys straight from memory into the operand, values through its
// part of LDS (sixteen bytes c of value t lie at c ^ f(t), which 16 rows written and 4 read at a time meet all banks with); what the
// wavefronts hold of the tile is added at the end of the tile or range.  No barrier inside.  Packed codes of two units are on their way at a
// time, of one for heads of 256, whose sums leave no registers (9 sequences of 162 tokens over 39562 keys, 4 bits: 5373 us with two, 2005).
// 16 users' drafts of four tokens over 1000 to 40000 keys of 4 bits, 350 MB: 151 us, 2.3 TB/s; the vector unit (46% of the time), the
// look-ups and operands in LDS (47%) and waits in turn bound it, besides what lies before the first unit and behind the last.  Heads of 256,
// bfloat16, a window of 1024 keys, 38 MB: 40 us, which is latency: lengths, table, keys, the second unit's keys, pieces, their join; and 19
// reloads of spilled registers and 176 moves of sums a unit.
template <int D, int KIND> struct ck_narrow {
  static constexpr bool PACKED = KIND >= 2;
  static constexpr int WAVES = PACKED && D < 256 ? 8 : 4, THREADS = 64 * WAVES, ROWS = 32, N = 32 * WAVES, START = 3;
  static constexpr int PER_CU = PACKED || D == 256 ? 1 : 2, PER_SIMD = D == 256 ? 1 : 2;
  // Of a unit, beside ck_wide's, where both share a launch.  Measured over 32 sequences of one full tile after 8000 to 25000 keys, us: plain heads
  // of 64 4.4 and 1.9, of 256 9.7 and 2.1; 4 bits, heads of 128 3.1 and 3.1, of 256 4.6 and 3.6; with keys of a few thousand, which
  // caches hold, packed rows of 128 took 2.7 and 3.6.
  static constexpr int COST = PACKED ? 3 : D == 256 ? 5 : 2;
  static constexpr int KS = D / 16, DT = D / 32, QUADS = D / 8, QW = QUADS / WAVES;
  static constexpr int V_BYTES = 32 * 2 * D, ROW = D + 4;            // (of a value; floats of a row that is turned)
  // sums of the wavefronts: the upper half's are added to the lower's first where not all fit
  static constexpr int LEFT = WAVES == 8 || D == 256 ? WAVES / 2 : WAVES;
  static constexpr int MERGE = LEFT * QUADS * 1024, TURN = 32 * ROW * 4;
  static constexpr int V0 = PACKED ? (int)sizeof(ck_lut<PACKED ? KIND : 4, 64>) : 0;
  static constexpr int AREA = MERGE > WAVES * V_BYTES ? MERGE : WAVES * V_BYTES, Q0 = V0 + (AREA > TURN ? AREA : TURN);
  static constexpr int ON = PACKED && D < 256 ? 2 : 1;               // units ahead of which keys are requested
  static constexpr bool Q_LDS = PACKED && (D < 256 || KIND < 4);                   // rows as operands in LDS: registers hold the keys on their way
  static constexpr int ML0 = Q0 + (Q_LDS ? 2 * KS * 1024 : 0), NRM0 = ML0 + WAVES * 512, UNDO0 = NRM0 + (PACKED ? WAVES * 3 * 128 : 0), L0 = UNDO0 + 128;
  static constexpr int LDS = L0 + (int)sizeof(ck_lengths<THREADS>);      // (nothing is static: the table of levels begins at 0)
  static_assert(L0 % 8 == 0 && LDS * PER_CU <= 160 * 1024, "fits");
  static __device__ __forceinline__ int f(int r) { return D == 64 ? 4 * ((r >> 1) & 1) + ((r >> 2) & 3) : 4 * (r & 3) + ((r >> 2) & 3); }
};

// What workgroup g of G does (workgroups 0 .. G - 1 of the launch), with `slots` pieces a tile in the scratch; `total`: length of one kv head's part of
// the axis.
template <int D, int KIND>
__device__ __forceinline__ void ck_narrow_work(const ck_args& a, unsigned char* const lds, ck_lengths<ck_narrow<D, KIND>::THREADS>& L, const int64_t total, const int g, const int G, const int slots) {
  typedef ck_narrow<D, KIND> P;
  typedef ck_math<KIND> M;
  constexpr bool PACKED = M::packed;
  constexpr int BITS = PACKED ? KIND : 4;
  constexpr int KS = P::KS, DT = P::DT, W = P::WAVES, T = P::THREADS;
  constexpr int HW = D * BITS / 64;                // packed: words of half a row
  float (*const ml)[64][2] = (float (*)[64][2])(lds + P::ML0);
  float (*const nrm)[3][32] = (float (*)[3][32])(lds + P::NRM0);     // packed, per wavefront: key norms, log2 and inverse of value norms
  float* const undo = (float*)(lds + P::UNDO0);    // packed: what undoes the scale of a row of queries
  typedef ck_lut<BITS, 64> lut_type;
  const lut_type& lut = *(const lut_type*)lds;
  unsigned char* const area = lds + P::V0;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, col = lane & 31;
  const int TM = P::ROWS / a.GC;

  // Ranges of one kv head's part of the axis, each taken by as many workgroups as there are heads, side by side on one die: they read the
  // same lines of the cache at the same time.  (A packed row is half a line or less, a norm a thirty-second of one; with the heads one
  // after the other on the axis, cut anywhere, a verification of 350 MB fetched 830.)
  const int heads = a.KVH * a.HS, head = g % heads, R = G / heads;
  const ck_share share = ck_share_of(total, R);
  int64_t at = ck_begin(share, g / heads, R);
  const int64_t end = ck_begin(share, g / heads + 1, R);
  if (tid == 0) a.rec[g].valid = 0;
  if (at >= end) return;
  int seq, tile;
  int64_t tile_at;                     // the tile's place on the axis
  ck_find<T, P::N, P::START>(a, L, TM, at, seq, tile, tile_at);

  float unit = 1.f, level = 0.f, turned = 0.f;      // of the levels; the lane's level; what undoes the matrix's scale, times the scale of the scores
  bool filled = false;

  for (;;) {
    const ck_seq s = ck_sequence(a, L, seq);
    const ck_range keys = ck_keys<P::N>(a, s, tile, TM);
    const int t0 = tile * TM, t1 = min(s.n, t0 + TM);
    const int64_t tile_end = tile_at + P::START + keys.units;
    const int u0 = max(0, (int)(at - tile_at) - P::START), u1 = min(keys.units, (int)min((int64_t)0x7fffffff, end - tile_at) - P::START);
    if (u1 <= 0) return;           // (nothing but the start of the tile: it begins in the next range)
    const ck_lane row = ck_row_of(a, s, t0, t1, head, col);
    const int kvh = head / a.HS;
    const int pos_first = s.ctx - s.n + t0, pos_last = s.ctx - s.n + t1 - 1;

    // ---- 32 keys of the wavefront, a lane its half of one (outside of what the tile sees: its first or last key, masked.  What else lies
    // there may be anything, and a weight of zero does not undo an infinity)
    const int base0 = (keys.first + u0) * P::N + 32 * wave;
    const int steps = keys.hi > base0 ? min(u1 - u0, (keys.hi - base0 + P::N - 1) / P::N) : 0;
    // (only the tile's first unit begins before its first key; packed rows have no windows)
    auto key_of = [&](int u, int oldest = INT_MIN) {
      const int key = min(base0 + u * P::N + col, keys.hi - 1);
      return PACKED ? key : max(key, oldest);
    };
    ck_u4 kd[PACKED ? 1 : KS], vd[PACKED ? 1 : KS];
    struct codes { uint32_t k[PACKED ? HW : 1], v[PACKED ? HW : 1]; float kn, vn; };
    codes even, odd;               // packed: those of two units (in turns, so that nothing in flight is ever moved)
    const uint8_t *const k_base = a.k + kvh * a.k_head + (PACKED ? 4 * HW : 16) * h, *const v_base = a.v + kvh * a.v_head + (PACKED ? 4 * HW : 16) * h;
    // (the entry after this unit's is requested first: what waits for it must not wait for the keys as well)
    ck_entry ahead = {0u, 0u};
    auto request = [&](int u, codes& w, int oldest = INT_MIN) {
      const ck_place p = ck_place_of(a, key_of(u, oldest), ahead);
      ahead = ck_look(a, seq, key_of(u + 1));
      const int64_t ko = ck_offset(p, a.k_blk, a.k_pos), vo = a.kv_alike ? ko : ck_offset(p, a.v_blk, a.v_pos);
      if constexpr (PACKED) {
        ck_load_words(w.k, k_base + ko);
        ck_load_words(w.v, v_base + vo);
        const int64_t kno = ck_offset(p, a.kn_blk, a.kn_pos), vno = a.kv_alike ? kno : ck_offset(p, a.vn_blk, a.vn_pos);
        w.kn = a.kn[kno + kvh * a.kn_head];
        w.vn = a.vn[vno + kvh * a.vn_head];
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          kd[ks] = *(const ck_u4*)(k_base + ko + 32 * ks);
          vd[ks] = *(const ck_u4*)(v_base + vo + 32 * ks);
        }
      }
    };
    if (steps > 0) {
      ahead = ck_look(a, seq, key_of(0, keys.lo));
      request(0, even, keys.lo);
      if constexpr (P::ON == 2) request(1, odd);
    }

    // ---- the rows: columns of the operand
    ck_u4 q[P::Q_LDS ? 1 : KS], ql[PACKED && !P::Q_LDS ? KS : 1];      // packed: two terms
    ck_u4* const q_lds = (ck_u4*)(lds + P::Q0) + lane;
    float fac = 1.f;
    {
      const uint16_t* p = (const uint16_t*)a.q + (int64_t)row.token * a.qs_tok + (int64_t)row.head * a.qs_head;
      if constexpr (PACKED) {
        float* rows = (float*)area;
        ck_u4 x[KS];
        float un = 1.f;
        if (wave < DT) {
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) x[ks] = row.valid ? *(const ck_u4*)(p + 8 * (2 * ks + h)) : (ck_u4){0u, 0u, 0u, 0u};
          un = ck_query_operand<D>(x, a.dtype);
        }
        if (!filled) {
          level = a.centroids[lane & ((1 << BITS) - 1)];
          ((uint32_t*)ml)[wave] = ck_unit_key<BITS, 16 / W, 1024>(level, 16 / W * (64 * wave + lane));
          turned = a.turn_scale->up * (1.f / CK_TURN) * a.scale2;
        }
        __syncthreads();           // (the area has been read)
        if (wave < DT) {
          if (wave == 0) undo[col] = un;
#pragma unroll
          for (int dt = wave; dt < DT; dt += W) {
            const ck_f16v y = ck_turn<D>(a.turn_in, dt, x);
#pragma unroll
            for (int b = 0; b < 4; ++b) *(float4*)(rows + col * P::ROW + 32 * dt + 8 * b + 4 * h) = make_float4(y[4 * b], y[4 * b + 1], y[4 * b + 2], y[4 * b + 3]);
          }
        }
        if (!filled) {
          uint32_t key = ((uint32_t*)ml)[0];
#pragma unroll
          for (int w = 1; w < W; ++w) key = min(key, ((uint32_t*)ml)[w]);
          unit = ck_unit_of<BITS, 1024>(level, key);
          ((lut_type*)lds)->fill(a.centroids, tid, T, unit);
          filled = true;
        }
        __syncthreads();
        // half h of a row: coordinates D / 2 h ..
        const float* from = rows + col * P::ROW + D / 2 * h;
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const float4 u = *(const float4*)(from + 4 * i);
          m = fmaxf(fmaxf(m, fmaxf(fabsf(u.x), fabsf(u.y))), fmaxf(fabsf(u.z), fabsf(u.w)));
        }
        m = fmaxf(m, akv_lane_xor<32>(m));
        const float f = ck_query_scale(m, undo[col] * turned, fac);
        auto piece = [&](int ks, ck_u4& hi, ck_u4& lo) {
          typedef _Float16 h2 __attribute__((ext_vector_type(2)));
          const float4 u = *(const float4*)(from + 8 * ks), v = *(const float4*)(from + 8 * ks + 4);
          const float y[8] = {u.x * f, u.y * f, u.z * f, u.w * f, v.x * f, v.y * f, v.z * f, v.w * f};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            hi[i] = M::pair(y[2 * i], y[2 * i + 1]);
            const h2 t = __builtin_bit_cast(h2, (uint32_t)hi[i]);
            lo[i] = M::pair(y[2 * i] - (float)t[0], y[2 * i + 1] - (float)t[1]);
          }
        };
        if constexpr (P::Q_LDS) {
          for (int ks = wave; ks < KS; ks += W) {      // (divided over the wavefronts; all read all of them)
            ck_u4 hi, lo;
            piece(ks, hi, lo);
            q_lds[64 * ks] = hi;
            q_lds[64 * (KS + ks)] = lo;
          }
        } else {
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) piece(ks, q[ks], ql[ks]);
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) q[ks] = row.valid ? *(const ck_u4*)(p + 8 * (2 * ks + h)) : (ck_u4){0u, 0u, 0u, 0u};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(q[ks]));
      }
    }
    const bool scaled = PACKED && __ballot(fac != 1.f) != 0;
    ck_f16v o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = (ck_f16v)(0.f);
    ck_row st = {-INFINITY, 0.f};
    unsigned char* vl = area + wave * P::V_BYTES;
    uint32_t v_at[DT];             // where the lane reads four coordinates of its value
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const int r = 4 * h + (lane & 15) / 4, c = 4 * dt + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
      v_at[dt] = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)vl + r * 2 * D + 16 * (c ^ P::f(r)) + 8 * (lane & 1);
    }
    __syncthreads();               // (the area has been read)
    auto unit_of = [&](int u, codes& w) {
      const int base = base0 + u * P::N;
      // ---- values to LDS, products of keys and rows
      ck_f16v sc[1];
      sc[0] = (ck_f16v)(0.f);
      if constexpr (PACKED) {
        const uint32_t keep = w.vn < CK_TINY ? 0u : 0xffffffffu;
        // look-ups of all keys, then of the values half at a time while the keys are multiplied
        ck_u4 k[KS], v[KS / 2];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) k[ks] = lut.group(w.k, ks);
#pragma unroll
        for (int p = 0; p < 2; ++p) {
#pragma unroll
          for (int i = 0; i < KS / 2; ++i) v[i] = lut.group(w.v, p * (KS / 2) + i);
#pragma unroll
          for (int i = 0; i < KS / 2; ++i) {
            const int ks = p * (KS / 2) + i;
            if constexpr (P::Q_LDS) {
              sc[0] = M::mfma(k[ks], q_lds[64 * (KS + ks)], sc[0]);
              sc[0] = M::mfma(k[ks], q_lds[64 * ks], sc[0]);
            } else {
              sc[0] = M::mfma(k[ks], ql[ks], sc[0]);
              sc[0] = M::mfma(k[ks], q[ks], sc[0]);
            }
          }
#pragma unroll
          for (int i = 0; i < KS / 2; ++i) *(ck_u4*)(vl + col * 2 * D + 16 * ((KS * h + p * (KS / 2) + i) ^ P::f(col))) = v[i] & keep;
        }
        if (h == 0) {
          const float v = w.vn < CK_TINY ? CK_NONE : w.vn;
          nrm[wave][0][col] = w.kn * unit;
          nrm[wave][1][col] = __log2f(v);
          nrm[wave][2][col] = 1.f / v;
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          *(ck_u4*)(vl + col * 2 * D + 16 * ((2 * ks + h) ^ P::f(col))) = vd[ks];
          sc[0] = M::mfma(kd[ks], q[ks], sc[0]);
        }
      }
      // ---- the next keys (packed: those two units on) fly from here on, and the entries of those behind them
      if (u + P::ON < steps) request(u + P::ON, w);
      akv_wave_sync();
      // keys 16 kb + 8 e + 4 h .. + 3, coordinate 32 dt + lane % 32 (eight rows on, f differs in its bit 1)
      auto value = [&](int kb, int dt, int e) {
        return __builtin_bit_cast(ck_u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ck_lds_s4*)(uintptr_t)((v_at[dt] ^ (32u * e)) + (16 * kb + 8 * e) * 2 * D)));
      };
      constexpr bool V_AHEAD = D == 64;      // read while the weights are computed, as far as there are registers
      ck_u2 vf[2][DT][2];
      if constexpr (V_AHEAD) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 2; ++e) vf[kb][dt][e] = value(kb, dt, e);
      }
      if (scaled) sc[0] *= fac;        // (a row far from the usual size)
      if constexpr (PACKED) ck_norms(sc, nrm[wave][0], nrm[wave][1]);
      if (base + 31 > pos_first || (a.window > 0 && base <= pos_last - a.window)) ck_mask(sc, base, row.pos, a.window);
      float alpha;
      if (ck_outgrown<KIND>(st, ck_max(sc) * (PACKED ? 1.f : a.scale2), alpha)) {
#pragma unroll
        for (int i = 0; i < DT; ++i) o[i] *= alpha;
      }
      ck_weights<1, PACKED>(sc, st, a.scale2, PACKED ? nrm[wave][2] : nullptr);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        ck_u4 p;
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = M::pair(sc[0][8 * kb + 2 * i], sc[0][8 * kb + 2 * i + 1]);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const ck_u2 x = V_AHEAD ? vf[kb][dt][0] : value(kb, dt, 0), y = V_AHEAD ? vf[kb][dt][1] : value(kb, dt, 1);
          o[dt] = M::mfma((ck_u4){x[0], x[1], y[0], y[1]}, p, o[dt]);
        }
      }
      akv_wave_sync();             // (the next values go where these are)
    };
    if constexpr (P::ON == 2) {
      for (int u = 0; u < steps; u += 2) {
        unit_of(u, even);
        if (u + 1 < steps) unit_of(u + 1, odd);
      }
    } else {
      for (int u = 0; u < steps; ++u) unit_of(u, even);
    }

    // ---- the wavefronts' sums of the tile, each in the frame of all; a wavefront ends up with QW quads of the coordinates
    st.l += akv_lane_xor<32>(st.l);
    ml[wave][lane][0] = st.m;
    ml[wave][lane][1] = st.l;
    __syncthreads();
    float m = ml[0][lane][0];
#pragma unroll
    for (int w = 1; w < W; ++w) m = fmaxf(m, ml[w][lane][0]);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) l += ml[w][lane][1] * ck_exp2(ml[w][lane][0] - ref);
    const float mine = ck_exp2(st.m - ref) * unit;
    float4* merge = (float4*)area;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] *= mine;
    auto dump = [&](int w) {
#pragma unroll
      for (int c = 0; c < P::QUADS; ++c)
        merge[(w * P::QUADS + c) * 64 + lane] = make_float4(o[c / 4][4 * (c & 3)], o[c / 4][4 * (c & 3) + 1], o[c / 4][4 * (c & 3) + 2], o[c / 4][4 * (c & 3) + 3]);
    };
    if (P::LEFT < W) {
      if (wave >= P::LEFT) dump(wave - P::LEFT);
      __syncthreads();
      if (wave < P::LEFT) {
#pragma unroll
        for (int c = 0; c < P::QUADS; ++c) {
          const float4 y = merge[(wave * P::QUADS + c) * 64 + lane];
          o[c / 4][4 * (c & 3)] += y.x; o[c / 4][4 * (c & 3) + 1] += y.y; o[c / 4][4 * (c & 3) + 2] += y.z; o[c / 4][4 * (c & 3) + 3] += y.w;
        }
      }
      __syncthreads();
    }
    if (wave < P::LEFT) dump(wave);
    __syncthreads();
    const bool whole = u0 == 0 && u1 == keys.units;
    const int64_t slot = (2 * (int64_t)g + (u0 == 0 ? 1 : 0)) * slots;
    float4 x[P::QW];
#pragma unroll
    for (int i = 0; i < P::QW; ++i) {
      const int cq = P::QW * wave + i;
      x[i] = merge[cq * 64 + lane];
#pragma unroll
      for (int w = 1; w < P::LEFT; ++w) {
        const float4 y = merge[(w * P::QUADS + cq) * 64 + lane];
        x[i].x += y.x; x[i].y += y.y; x[i].z += y.z; x[i].w += y.w;
      }
    }
    if (!whole) {
#pragma unroll
      for (int i = 0; i < P::QW; ++i) ((float4*)a.part)[(slot * P::QUADS + P::QW * wave + i) * 64 + lane] = x[i];
      if (wave == 0) {
        a.part_ml[slot * 64 + lane] = make_float2(m, l);
        if (u0 == 0 && lane == 0) a.rec[g] = {tile_end, total, CK_LEFT_NARROW, head, s.q0 + t0, t1 - t0, 0, G};
      }
    } else {
      ck_results<D, KIND, W, P::QW>(a, x, ck_finish(l), ck_turn_rows<D, false>(a.turn_out, wave), row.valid, row.token, row.head, (float*)area);
    }
    // ---- on to the next tile
    at = tile_at = tile_end;
    if (at >= end) return;
    ++tile;
    int n = s.n;
    while ((int64_t)tile * TM >= n) {
      tile = 0;
      if (++seq > a.S) return;         // (starts that go back: the axis has fewer tiles than the sequences)
      n = ck_sequence(a, L, seq).n;
    }
  }
}

// ---- many rows a sequence -----------------------------------------------------------------------------------------------------
// A tile is 32 rows a wavefront, a unit N keys, which the wavefronts of the workgroup share in LDS.  Work goes by steps of 32
// keys: while the weights of step x are computed (vector unit) the products of step x + 1 are (matrix cores), their operands read during the
// value products of step x - 1; then the values of step x are multiplied, their operands read during the first half.  The two units take
// turns instruction by instruction: left to two wavefronts a SIMD with both in blocks, they overlapped by a quarter (mean of 16
// products and 16 weights 1417 clocks, in turns 1071).  Keys of unit u + 2 and values of u + 1 are on their way during unit u; packed ones
// are put to LDS then, beside the value products, from codes that were requested a unit before (all at the end of a unit: 2000 rows over
// 8000 keys, 32 heads, 445 us instead of 422).
//
// The matrix cores bound it as far as the chip's power allows: 2048 rows over 31000 keys, 32 heads of 128 in bfloat16 take 1060 to 1120 us by the
// machine, 1000 TFLOP/s, where a large product of the library reaches 1280 (products 47% of the clocks; written out in turns by hand it is no
// faster).  Heads of 64 are bound by the vector unit, 60% of the clocks.  Packed rows of 128: 640 TFLOP/s; codes are looked up by every
// workgroup for its 256 rows, LDS is busy 47% and the vector unit 56% of the clocks, and registers leave no room for more in flight.  Heads of
// 256: the sums do not stay where the products leave them, a step of 32 products has some 630 moves between the two register files (one
// prompt of 2048 after 6000 keys 943 us, 480 TFLOP/s).
//
// Rows lie in LDS without padding, their pieces of sixteen bytes in an order that depends on the row, piece c at place c ^ f(row): sixteen
// lanes that read one piece of sixteen keys, and 32 that read four coordinates each of four values, meet all 64 banks once
// (245 and 216 bytes a clock; rows padded by 32 bytes gave 128 and 126).
template <int D, int KIND> struct ck_wide {
  static constexpr bool AHEAD = D == 64 || (D == 128 && KIND < 2);    // registers for the keys of the step after the next
  static constexpr int EARLY = AHEAD ? D / 16 : KIND >= 2 && D < 256 ? D / 32 : 0;     // pieces of a step's keys that are read during the step before
  static constexpr int WAVES = D == 128 ? 8 : 4, THREADS = 64 * WAVES, ROWS = 32 * WAVES, N = D == 256 ? 32 : 64, STEPS = N / 32;
  // What a tile costs besides its units, in units; both kernels', as it is | none | twice as much: 2048 tokens after nothing 78.7 | 102 | 80.4 us, 40
  // prompts of 30 to 200 67.7 | 74.4 | 67.9, 16 drafts over up to 40000 packed keys 175 | 182 | 175, 64 of 5 tokens after 20 to 400 30.1 | 32.7 | 29.6,
  // a window of 1024 at heads of 256 39.0 | 43.3 | 41.1.
  static constexpr int START = 192 / N;
  static constexpr int PER_CU = D == 256 || WAVES == 8 ? 1 : 2;       // workgroups a CU
  static constexpr int PER_SIMD = D == 256 ? 1 : 2;                   // wavefronts a SIMD
  static constexpr int KS = D / 16, DT = D / 32, QUADS = D / 8;
  static constexpr int ROW = 2 * D, TILE = N * ROW;
  // Units of keys held: of those read during a unit, and the one that is written (a unit on with AHEAD, or where a unit is a step)
  static constexpr int KRING = AHEAD || STEPS == 1 ? 2 : 3;
  static_assert(EARLY == 0 || STEPS == 2, "the step after the next lies in the next unit");
  static constexpr int UNROLL = KIND >= 2 ? 1 : STEPS;
  static constexpr int RING = 2 * WAVES;                              // units whose places and norms are held
  static constexpr int COST = KIND >= 2 ? 4 : 2;
  static constexpr int K0 = 0, V0 = KRING * TILE, PLACE0 = V0 + 2 * TILE, NORM0 = PLACE0 + RING * N * 16;
  static constexpr int LUT0 = NORM0 + (KIND >= 2 ? RING * N * 16 : 0), L0 = LUT0 + (KIND >= 2 ? (int)sizeof(ck_lut<KIND >= 2 ? KIND : 4, 1>) : 0);
  static constexpr int LDS = L0 + (int)sizeof(ck_lengths<THREADS>);
  static_assert(L0 % 8 == 0 && LDS * PER_CU <= 160 * 1024, "fits");
  static __device__ __forceinline__ int fk(int r) { return D == 64 ? (r >> 1) & 7 : r & 15; }
  static __device__ __forceinline__ int fv(int r) { return D == 64 ? 4 * ((r >> 1) & 1) + ((r >> 1) & 3) : 5 * (r & 3); }
};
// Sixteen bytes a lane from `src` into LDS at `at` + 16 x lane.  (The compiler does not see the request: who reads waits by
// ck_landed() and a barrier.  The wait states stand behind m0.)
__device__ __forceinline__ void ck_request(const uint8_t* src, uint32_t at) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "{m0}"(at) : "memory");
}
__device__ __forceinline__ void ck_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// What workgroup g of G does, number base + g of the launch; `per_head`: length of one kv head's part of the axis.
template <int D, int KIND>
__device__ __forceinline__ void ck_wide_work(const ck_args& a, unsigned char* const lds, ck_lengths<ck_wide<D, KIND>::THREADS>& L, const int64_t per_head, const int g, const int G, const int base) {
  typedef ck_wide<D, KIND> P;
  typedef ck_math<KIND> M;
  constexpr bool PACKED = M::packed;
  constexpr int BITS = PACKED ? KIND : 4;
  constexpr int KS = P::KS, DT = P::DT, N = P::N, T = P::THREADS;
  constexpr int CPR = D / 8;                                  // pieces of 16 bytes a row
  constexpr int RPI = 64 / CPR, NP = N / RPI / P::WAVES;      // dense: rows a request, requests a wavefront
  constexpr int TPR = D / 32, TASKS = N * TPR, NT = 2 * TASKS / T;      // packed: 32 codes a task, keys' then values'
  static_assert(NT * T == 2 * TASKS && NP * RPI * P::WAVES == N, "whole tasks and requests");
  typedef ck_lut<BITS, 1> lut_type;
  lut_type& lut = *(lut_type*)(lds + P::LUT0);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, col = lane & 31;
  const int TM = P::ROWS / a.GC;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;

  const int heads = a.KVH * a.HS;
  const int64_t total = per_head * heads;
  const ck_share share = ck_share_of(total, G);
  int64_t at = ck_begin(share, g, G);
  const int64_t end = ck_begin(share, g + 1, G);
  if (tid == 0) a.rec[base + g].valid = 0;
  if (at >= end) return;
  int head = total <= 0xffffffffll ? (int)((uint32_t)at / (uint32_t)per_head) : (int)(at / per_head), seq, tile;
  int64_t tile_at;
  ck_find<T, N, P::START>(a, L, TM, at - head * per_head, seq, tile, tile_at);
  tile_at += head * per_head;

  float unit = 1.f;                // of the levels
  if constexpr (PACKED) {
    const float level = a.centroids[lane & ((1 << BITS) - 1)];
    unit = ck_unit_of<BITS, 64>(level, ck_unit_key<BITS, 1, 64>(level, lane));
    lut.fill(a.centroids, tid, T, unit);
  }
  // where the lane reads its operands: a piece of a key, four coordinates of a value
  uint32_t k_at[KS], v_at[DT];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) k_at[ks] = lds0 + P::K0 + col * P::ROW + 16 * ((2 * ks + h) ^ P::fk(col));
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    const int r = 4 * h + (lane & 15) / 4, c = 4 * dt + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    v_at[dt] = lds0 + P::V0 + r * P::ROW + 16 * (c ^ P::fv(r)) + 8 * (lane & 1);
  }

  for (;;) {
    const ck_seq s = ck_sequence(a, L, seq);
    const ck_range keys = ck_keys<N>(a, s, tile, TM);
    const int t0 = tile * TM, t1 = min(s.n, t0 + TM);
    const int64_t tile_end = tile_at + P::START + keys.units;
    const int u0 = max(0, (int)(at - tile_at) - P::START), u1 = min(keys.units, (int)min((int64_t)0x7fffffff, end - tile_at) - P::START);
    if (u1 <= 0) return;           // (nothing but the start of the tile: it begins in the next range)
    const int units = keys.hi > 0 ? u1 - u0 : 0;
    const ck_lane row = ck_row_of(a, s, t0, t1, head, 32 * wave + col);
    const int kvh = head / a.HS;
    // positions of the wavefront's rows
    const int w0 = t0 + 32 * wave / a.GC, w1 = min(t1, t0 + (32 * wave + 31) / a.GC + 1);
    const int pos_first = s.ctx - s.n + w0, pos_last = w0 < t1 ? s.ctx - s.n + w1 - 1 : -1;
    ck_f16v o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = (ck_f16v)(0.f);
    ck_row st = {-INFINITY, 0.f};

    const int base0 = (keys.first + u0) * N;
    // Places of a unit's keys, by one wavefront, a lane a key: the table's entry is requested, and what the rows of keys and
    // values lie at is written a unit later.  Every wavefront does so for one unit of the next WAVES, all at the same time: one that did
    // it for the others would be what they wait for.  A key behind the last one that the tile sees has the last one's place, one before the
    // first the first one's: what is read for it is masked, and its value is as finite as that one's.
    // (Only the tile's first unit begins before its first key; packed rows have no windows.)
    auto key_of = [&](int u, int oldest = INT_MIN) {
      const int key = min(base0 + u * N + (lane & (N - 1)), keys.hi - 1);
      return PACKED ? key : max(key, oldest);
    };
    auto look = [&](int u, int oldest = INT_MIN) { return ck_look(a, seq, key_of(u, oldest)); };
    float kn = 0.f, vn = 1.f;      // packed: norms of the unit noted last
    auto note = [&](int u, const ck_entry& e, int oldest = INT_MIN) {
      const ck_place p = ck_place_of(a, key_of(u, oldest), e);
      int64_t* place = (int64_t*)(lds + P::PLACE0) + (u & (P::RING - 1)) * 2 * N;
      const int64_t k_at = ck_offset(p, a.k_blk, a.k_pos) + kvh * a.k_head;
      place[lane & (N - 1)] = k_at;
      place[N + (lane & (N - 1))] = a.kv_alike ? k_at : ck_offset(p, a.v_blk, a.v_pos) + kvh * a.v_head;
      if constexpr (PACKED) {
        const int64_t n_at = ck_offset(p, a.kn_blk, a.kn_pos) + kvh * a.kn_head;
        kn = a.kn[n_at];
        vn = a.vn[a.kv_alike ? n_at : ck_offset(p, a.vn_blk, a.vn_pos) + kvh * a.vn_head];
      }
    };
    auto note_norms = [&](int u) {
      if constexpr (PACKED) {
        float* nr = (float*)(lds + P::NORM0) + (u & (P::RING - 1)) * 4 * N;
        const float v = vn < CK_TINY ? CK_NONE : vn;
        const int key = lane & (N - 1);
        nr[key] = kn * unit;
        nr[N + key] = __log2f(v);
        nr[2 * N + key] = 1.f / v;
        ((uint32_t*)nr)[3 * N + key] = vn < CK_TINY ? 0u : 0xffffffffu;
      }
    };
    // dense: keys of one unit, values of another on their way to LDS
    auto request = [&](int uk, int k_slot, bool k_there, int uv, bool v_there) {
      const int64_t* pk = (const int64_t*)(lds + P::PLACE0) + (uk & (P::RING - 1)) * 2 * N;
      const int64_t* pv = (const int64_t*)(lds + P::PLACE0) + (uv & (P::RING - 1)) * 2 * N + N;
      int64_t ok[NP], ov[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int r = (wave * NP + i) * RPI + lane / CPR;
        ok[i] = pk[r] + 16 * ((lane % CPR) ^ P::fk(r));
        ov[i] = pv[r] + 16 * ((lane % CPR) ^ P::fv(r));
      }
      const uint32_t k_to = lds0 + P::K0 + k_slot * P::TILE + wave * NP * RPI * P::ROW, v_to = lds0 + P::V0 + (uv & 1) * P::TILE + wave * NP * RPI * P::ROW;
      if (k_there) {
#pragma unroll
        for (int i = 0; i < NP; ++i) ck_request(a.k + ok[i], __builtin_amdgcn_readfirstlane(k_to + i * 1024));
      }
      if (v_there) {
#pragma unroll
        for (int i = 0; i < NP; ++i) ck_request(a.v + ov[i], __builtin_amdgcn_readfirstlane(v_to + i * 1024));
      }
    };
    // packed: codes of the keys of one unit and the values of another to registers, and from there to LDS; a value whose norm counts as
    // nothing is zero
    struct codes { uint32_t w[PACKED ? NT : 1][BITS]; };
    codes words;
    // (the wavefront's own choice of the two, and by value: taken from the arguments' memory it made every request a generic one, for which reads
    // of LDS wait)
    const uint8_t *const k_base = a.k, *const v_base = a.v;
    auto fetch = [&](int uk, int uv, codes& c) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int task = tid + T * i, v = (64 * wave + T * i) / TASKS, r = task % TASKS / TPR, part = task % TPR;
        const int64_t* place = (const int64_t*)(lds + P::PLACE0) + ((v ? uv : uk) & (P::RING - 1)) * 2 * N + v * N;
        ck_load_words(c.w[i], (v ? v_base : k_base) + place[r] + 4 * BITS * part);
      }
    };
    // ... the part `step` of STEPS of them
    auto put = [&](int k_slot, int uv, int step) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int task = tid + T * i, v = (64 * wave + T * i) / TASKS, r = task % TASKS / TPR, part = task % TPR;
        unsigned char* to = lds + (v ? P::V0 + (uv & 1) * P::TILE : P::K0 + k_slot * P::TILE) + r * P::ROW;
        const int f = v ? P::fv(r) : P::fk(r);
        const uint32_t keep = ((const uint32_t*)(lds + P::NORM0))[(uv & (P::RING - 1)) * 4 * N + 3 * N + r] | (v ? 0u : 0xffffffffu);
        // (the step is no constant: its sixteen codes are moved to the front)
        uint32_t w[BITS];
#pragma unroll
        for (int b = 0; b < BITS; ++b) {
          w[b] = words.w[i][b];
          const uint32_t far = BITS == 3 ? (b == 0 ? __builtin_amdgcn_alignbyte(words.w[i][2], words.w[i][1], 2) : words.w[i][2] >> 16) : words.w[i][(b + BITS / 2) % BITS];
          if (P::STEPS == 2 && step == 1 && b < (BITS + 1) / 2) w[b] = far;
        }
#pragma unroll
        for (int n = 0; n < 4 / P::STEPS; n += 2) {
          const int j = 2 * (P::STEPS == 2 ? step : 0) + n;
          // (keys: the order of the turned rows; without branches, which the products could not be spread over)
          const ck_u4 x = lut.group(w, n), y = lut.group(w, n + 1);
          *(ck_u4*)(to + 16 * ((4 * part + j) ^ f)) = (ck_u4){x[0], x[1], v ? x[2] : y[0], v ? x[3] : y[1]} & keep;
          *(ck_u4*)(to + 16 * ((4 * part + j + 1) ^ f)) = (ck_u4){v ? y[0] : x[2], v ? y[1] : x[3], y[2], y[3]} & keep;
        }
      }
    };
    auto put_all = [&](int k_slot, int uv) {
#pragma unroll
      for (int t = 0; t < P::STEPS; ++t) put(k_slot, uv, t);
    };

    // (the rows of the tile are requested behind the first keys and values)
    ck_u4 q[KS];
    float fac = 1.f;
    auto rows = [&]() {
      const uint16_t* p = (const uint16_t*)a.q + (int64_t)row.token * a.qs_tok + (int64_t)row.head * a.qs_head;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) q[ks] = row.valid ? *(const ck_u4*)(p + 8 * (2 * ks + h)) : (ck_u4){0u, 0u, 0u, 0u};
    };
    // packed: turned, by the lane's own products: the coordinates of a step come out as 4 h .. + 3 and 8 + 4 h .. + 3 of sixteen, the
    // order that keys are put to LDS in
    auto turn_rows = [&]() {
      const float un = ck_query_operand<D>(q, a.dtype) * a.turn_scale->up * (1.f / CK_TURN) * a.scale2;
      ck_f16v y[DT];
      float m = 0.f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        y[dt] = ck_turn<D>(a.turn_in, dt, q);
#pragma unroll
        for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(y[dt][i]));
      }
      m = fmaxf(m, akv_lane_xor<32>(m));
      const float f = ck_query_scale(m, un, fac);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int i = 0; i < 4; ++i) q[ks][i] = M::pair(y[ks / 2][8 * (ks & 1) + 2 * i] * f, y[ks / 2][8 * (ks & 1) + 2 * i + 1] * f);
    };
    ck_entry ahead = {0u, 0u};
    __syncthreads();               // (LDS of the tile before has been read)
    if (units > 0) {
      note(wave, look(wave, keys.lo), keys.lo);
      note_norms(wave);
      __syncthreads();
      ahead = look(P::WAVES + wave);
      if constexpr (PACKED) {
        fetch(0, 0, words);
        rows();
        put_all(0, 0);
        fetch(1, 0, words);
        turn_rows();
        put_all(1, 0);
        fetch(2, 1, words);
      } else {
        request(0, 0, true, 0, true);
        request(1, 1, units > 1, 0, false);
        rows();
        ck_landed();
      }
    } else {
      rows();
      fac = 1.f;
    }
    // (the rows are there: without a use here the compiler waits for them in the loop, and so for what flies then)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(q[ks]));
    const bool scaled = PACKED && __ballot(fac != 1.f) != 0;
    __syncthreads();
    ck_u4 kf[KS];
    ck_f16v sc[1];
    auto read_keys = [&](uint32_t from, int first, int last) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        if (ks >= first && ks < last) kf[ks] = *(const ck_lds_u4*)(uintptr_t)(k_at[ks] + from);
    };
    if (units > 0) {
      read_keys(0, 0, KS);
      sc[0] = (ck_f16v)(0.f);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) sc[0] = M::mfma(kf[ks], q[ks], sc[0]);
      if (P::EARLY > 0) read_keys(32 * P::ROW, 0, P::EARLY);
      __syncthreads();             // (unit 2's keys may go where these were)
      const float* nr = (const float*)(lds + P::NORM0);
      if (scaled) sc[0] *= fac;
      if constexpr (PACKED) ck_norms(sc, nr, nr + N);
      if (base0 + 31 > pos_first || (a.window > 0 && base0 <= pos_last - a.window)) ck_mask(sc, base0, row.pos, a.window);
      float alpha;
      ck_outgrown<KIND>(st, ck_max(sc) * (PACKED ? 1.f : a.scale2), alpha);      // (nothing to rescale yet)
    }
    const bool busy = 32 * wave < (t1 - t0) * a.GC;      // (a wavefront behind the tile's last row only brings keys and values)
    int k_slot = 0;                // of unit u
    for (int u = 0; u < units; ++u) {
      // ---- on their way: places of the WAVES units behind the WAVES that this one belongs to; keys of u + 2, values of u + 1 (packed:
      // of units one further on, while the codes requested a unit ago are put to LDS beside the products).  Noted during unit k WAVES
      // they are read from k WAVES + 1 on, up to three units ahead: WAVES is at least four.
      static_assert(P::WAVES >= 4, "places are noted before they are read");
      const int turn = u & (P::WAVES - 1);
      if (turn == 0) note(u + P::WAVES + wave, ahead);
      if (turn == P::WAVES - 1) ahead = look(u + 1 + P::WAVES + wave);
      const int k_next = P::KRING == 2 ? k_slot ^ 1 : k_slot == 2 ? 0 : k_slot + 1, k_after = P::KRING == 2 ? k_slot : k_next == 2 ? 0 : k_next + 1;
      codes flying;
      if constexpr (PACKED) fetch(u + 3, u + 2, flying);
      else request(u + 2, k_after, u + 2 < units, u + 1, u + 1 < units);
      const float* nr = (const float*)(lds + P::NORM0) + (u & (P::RING - 1)) * 4 * N;
      const uint32_t v_from = (u & 1) * P::TILE;
      if (busy)
#pragma unroll P::UNROLL
      for (int t = 0; t < P::STEPS; ++t) {
        // ---- weights of these keys, products of the next 32 (behind the last: of whatever lies there, unused), values to registers
        if (!P::AHEAD) read_keys(t + 1 < P::STEPS ? k_slot * P::TILE + (t + 1) * 32 * P::ROW : k_next * P::TILE, P::EARLY, KS);
        ck_f16v next = (ck_f16v)(0.f);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) next = M::mfma(kf[ks], q[ks], next);
        ck_u2 vf[2][DT][2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 2; ++e)     // keys 16 kb + 8 e + 4 h .. + 3, coordinate 32 dt + lane % 32
              vf[kb][dt][e] = __builtin_bit_cast(ck_u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ck_lds_s4*)(uintptr_t)(v_at[dt] + v_from + (32 * t + 16 * kb + 8 * e) * P::ROW)));
        ck_weights<1, PACKED>(sc, st, a.scale2, PACKED ? nr + 2 * N + 32 * t : nullptr);
        ck_u4 p[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 4; ++i) p[kb][i] = M::pair(sc[0][8 * kb + 2 * i], sc[0][8 * kb + 2 * i + 1]);
        constexpr int READS = 4 * DT + KS - P::EARLY + (PACKED ? 4 : 0), FIRST = P::AHEAD ? 0 : 4;
        if (FIRST > 0) __builtin_amdgcn_sched_group_barrier(0x100, FIRST, 0);
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                                      // MFMA
          __builtin_amdgcn_sched_group_barrier(0x100, (READS - FIRST + KS - 1) / KS, 0);          // LDS read
          __builtin_amdgcn_sched_group_barrier(0x402, (PACKED ? 64 : 56) / KS + 1, 0);            // vector and transcendental
        }
        // (the weights stay on this side of the branch: behind it they would have no products to run beside)
        asm volatile("" : "+v"(p[0]), "+v"(p[1]), "+v"(st.l));
        if constexpr (PACKED) __builtin_amdgcn_sched_barrier(0);
        // ---- what the next step's rows do not see
        const int base = base0 + u * N + 32 * (t + 1);
        const float* nn = t + 1 < P::STEPS ? nr + 32 * (t + 1) : (const float*)(lds + P::NORM0) + ((u + 1) & (P::RING - 1)) * 4 * N;
        sc[0] = next;
        if (scaled) sc[0] *= fac;
        const bool hidden = base + 31 > pos_first || (a.window > 0 && base <= pos_last - a.window);
        if (!PACKED && hidden) ck_mask(sc, base, row.pos, a.window);
        // ---- values, the keys of the step after the next to registers, and the largest of the next step's scores (packed: their norms, and
        // codes to LDS; without a branch, over which the products could not be spread)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
            o[dt] = M::mfma((ck_u4){vf[kb][dt][0][0], vf[kb][dt][0][1], vf[kb][dt][1][0], vf[kb][dt][1][1]}, p[kb], o[dt]);
        if (P::AHEAD) read_keys(k_next * P::TILE + t * 32 * P::ROW, 0, KS);
        else if (P::EARLY > 0) read_keys(k_next * P::TILE + t * 32 * P::ROW, 0, P::EARLY);
        if constexpr (PACKED) {
          ck_norms(sc, nn, nn + N);
          put(k_after, u + 1, t);
        }
        constexpr int LOOK = PACKED ? 16 * NT / P::STEPS : 0;      // levels looked up
        float mx = PACKED ? 0.f : ck_max(sc) * a.scale2;
#pragma unroll
        for (int i = 0; i < 2 * DT; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          if (P::EARLY > 0) __builtin_amdgcn_sched_group_barrier(0x100, (P::EARLY + (PACKED ? 10 : 0) + LOOK + 2 * DT - 1) / (2 * DT), 0);
          __builtin_amdgcn_sched_group_barrier(0x002, (PACKED ? 32 + 4 * LOOK : 16) / (2 * DT) + 1, 0);
        }
        if constexpr (PACKED) {
          if (hidden) ck_mask(sc, base, row.pos, a.window);
          mx = ck_max(sc);
        }
        float alpha;
        if ((t + 1 < P::STEPS || u + 1 < units) && ck_outgrown<KIND>(st, mx, alpha)) {
#pragma unroll
          for (int i = 0; i < DT; ++i) o[i] *= alpha;
        }
      }
      // ---- what was requested is there
      if constexpr (PACKED) {
        if (!busy) put_all(k_after, u + 1);
        if (turn == 0) note_norms(u + P::WAVES + wave);
        words = flying;
      } else {
        ck_landed();
      }
      k_slot = k_next;
      __syncthreads();
    }

    st.l += akv_lane_xor<32>(st.l);
    const bool whole = u0 == 0 && u1 == keys.units;
    if (whole && PACKED) {
      const float f = ck_finish(st.l) * unit;
      ck_u4 hi[KS], lo[KS];
      const float un = ck_result_operand<D>([&](int ks, int j) { return o[ks / 2][8 * (ks & 1) + j] * f; }, hi, lo) * a.turn_scale->up * (1.f / CK_TURN);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const ck_f16v y = ck_turn<D>(a.turn_out, dt, hi, lo);
        if (row.valid) {
#pragma unroll
          for (int b = 0; b < 4; ++b) ck_store<KIND>(a, row.token, row.head, 4 * dt + b, y[4 * b] * un, y[4 * b + 1] * un, y[4 * b + 2] * un, y[4 * b + 3] * un);
        }
      }
    } else if (whole) {
      const float f = ck_finish(st.l);
      if (row.valid) {
#pragma unroll
        for (int c = 0; c < P::QUADS; ++c)
          ck_store<KIND>(a, row.token, row.head, c, o[c / 4][4 * (c & 3)] * f, o[c / 4][4 * (c & 3) + 1] * f, o[c / 4][4 * (c & 3) + 2] * f, o[c / 4][4 * (c & 3) + 3] * f);
      }
    } else {
      const int64_t slot = (2 * (int64_t)(base + g) + (u0 == 0 ? 1 : 0)) * P::WAVES + wave;
      if (busy) {
#pragma unroll
        for (int c = 0; c < P::QUADS; ++c)
          ((float4*)a.part)[(slot * P::QUADS + c) * 64 + lane] = make_float4(o[c / 4][4 * (c & 3)] * unit, o[c / 4][4 * (c & 3) + 1] * unit, o[c / 4][4 * (c & 3) + 2] * unit, o[c / 4][4 * (c & 3) + 3] * unit);
        a.part_ml[slot * 64 + lane] = make_float2(st.m, st.l);
      }
      if (u0 == 0 && tid == 0) a.rec[base + g] = {tile_end, total, CK_LEFT_WIDE, head, s.q0 + t0, t1 - t0, base, G};
    }
    at = tile_at = tile_end;
    if (at >= end) return;
    ++tile;
    int n = s.n;
    while ((int64_t)tile * TM >= n) {
      tile = 0;
      if (++seq > a.S) {
        seq = 0;
        if (++head >= heads) return;   // (starts that go back)
      }
      n = ck_sequence(a, L, seq).n;
    }
  }
}

// ---- kernels -------------------------------------------------------------------------------------------------------------------
// Nothing in LDS is static: the narrow kernel's table of levels begins at 0, the lengths lie behind everything.
template <class P> __device__ __forceinline__ ck_lengths<P::THREADS>& ck_lengths_at(unsigned char* lds, int at) { return *(ck_lengths<P::THREADS>*)(lds + at); }
// Workgroups in the order in which they lie on the dies.
__device__ __forceinline__ int ck_workgroup() {
  const int G = gridDim.x, b = blockIdx.x;
  return G % 8 == 0 ? b % 8 * (G / 8) + b / 8 : b;
}
template <int D, int KIND>
__global__ __launch_bounds__((ck_narrow<D, KIND>::THREADS), (ck_narrow<D, KIND>::PER_SIMD)) void ck_narrow_kernel(ck_args a) {
  typedef ck_narrow<D, KIND> P;
  extern __shared__ __align__(1024) unsigned char lds[];
  auto& L = ck_lengths_at<P>(lds, P::L0);
  ck_load_lengths(a, L);
  ck_clear_front(a, L, D);
  const int64_t total = ck_total<P::THREADS, P::N, P::START>(a, L, P::ROWS / a.GC);
  ck_narrow_work<D, KIND>(a, lds, L, total, ck_workgroup(), gridDim.x, 1);
}
template <int D, int KIND>
__global__ __launch_bounds__((ck_wide<D, KIND>::THREADS), (ck_wide<D, KIND>::PER_SIMD)) void ck_wide_kernel(ck_args a) {
  typedef ck_wide<D, KIND> P;
  extern __shared__ __align__(1024) unsigned char lds[];
  auto& L = ck_lengths_at<P>(lds, P::L0);
  ck_load_lengths(a, L);
  if (a.kind == 0) ck_clear_front(a, L, D);      // (the narrow kernel did otherwise)
  const int64_t per_head = ck_total<P::THREADS, P::N, P::START>(a, L, P::ROWS / a.GC);
  ck_wide_work<D, KIND>(a, lds, L, per_head, ck_workgroup(), gridDim.x, 0);
}
// Both at once: the workgroups are divided by what each has to do.  (One kernel after the other the few rows of a mixed batch take as long as
// a workgroup needs to begin and to end: 12 sequences of 1 to 90 tokens over 3 bits 152 us, together 122; 24 of 1 to 300 over plain heads of
// 64 119.5 and 118.)
template <int D, int KIND> struct ck_both {
  typedef ck_narrow<D, KIND> N;
  typedef ck_wide<D, KIND> W;
  static constexpr bool FITS = N::THREADS == W::THREADS && N::PER_CU == W::PER_CU;
  static constexpr int L0 = N::L0 > W::L0 ? N::L0 : W::L0, LDS = L0 + (int)sizeof(ck_lengths<W::THREADS>);
};
template <int D, int KIND>
__global__ __launch_bounds__((ck_wide<D, KIND>::THREADS), (ck_wide<D, KIND>::PER_SIMD)) void ck_both_kernel(ck_args few, ck_args many) {
  typedef ck_narrow<D, KIND> N;
  typedef ck_wide<D, KIND> W;
  extern __shared__ __align__(1024) unsigned char lds[];
  auto& L = ck_lengths_at<W>(lds, ck_both<D, KIND>::L0);
  ck_load_lengths(many, L);
  ck_clear_front(many, L, D);
  const int64_t few_total = ck_total<N::THREADS, N::N, N::START>(few, L, N::ROWS / few.GC), many_total = ck_total<W::THREADS, W::N, W::START>(many, L, W::ROWS / many.GC);
  const int G = gridDim.x, g = ck_workgroup(), few_heads = few.KVH * few.HS;
  const float few_cost = (float)N::COST * (float)few_heads * (float)few_total, many_cost = (float)W::COST * (float)(many.KVH * many.HS) * (float)many_total;
  int ranges = 0;
  if (few_total > 0) {
    ranges = (int)((float)G * few_cost / ((few_cost + many_cost) * (float)few_heads) + 0.5f);
    ranges = max(1, min(ranges, (many_total > 0 ? G - 1 : G) / few_heads));
  }
  const int taken = ranges * few_heads;
  if (g < taken) ck_narrow_work<D, KIND>(few, lds, L, few_total, g, taken, W::WAVES);
  else ck_wide_work<D, KIND>(many, lds, L, many_total, g - taken, G - taken, taken);
}

// ---- the pieces of a tile that several ranges share --------------------------------------------------------------------------
// Workgroup (g, w): the 32 rows w of the tile that begins in workgroup g's range and does not end there; its other pieces are the first ones
// of the ranges behind, which are a workgroup apart (many rows) or as many as there are heads (few).  Up to four pieces are on their way
// together, under a running maximum.  Reading the pieces bounds it (512 bytes a row of 128 and piece): 15 us after the first chunk of 2048
// tokens, of which 67 MB are pieces; after few rows it is one trip to memory, 6 us.
struct ck_cut { int HS, GC; };        // of the few rows' kernel
template <int D, int KIND, int WAVES>
__global__ __launch_bounds__(256, WAVES == 1 || D == 256 ? 2 : 4) void ck_merge_kernel(ck_args a, ck_cut few) {
  constexpr int QUADS = D / 8, MINE = QUADS / 4;
  __shared__ __align__(16) float rows[ck_math<KIND>::packed ? 32 * (D + 4) : 1];
  const int part = blockIdx.y;
  const ck_record rec = a.rec[blockIdx.x];
  if (rec.valid == 0) return;
  const bool narrow = WAVES == 1 || rec.valid == CK_LEFT_NARROW;
  const int HS = narrow ? few.HS : a.HS, GC = narrow ? few.GC : a.GC;
  if (32 * part >= rec.tokens * GC) return;      // (rows behind the tile's last: nothing was left of them)
  const int stride = narrow ? a.KVH * HS : 1, g = (int)blockIdx.x - rec.base, G = rec.count;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31;
  ck_turn_rows<D, ck_math<KIND>::packed && D < 256 && WAVES == 1> matrix(a.turn_out, wave);
  // ranges first + 1 .. last hold a piece each, unless they are empty
  const int R = G / stride, first = g / stride;
  const ck_share share = ck_share_of(rec.total, R);
  int next = first + 1;
  float m = -INFINITY, l = 0.f;
  float4 x[MINE];
#pragma unroll
  for (int i = 0; i < MINE; ++i) x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (bool more = true, begun = false; more; begun = true) {
    float2 e[4];
    float4 y[4][MINE];
    float top = m;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      int r = begun || k > 0 ? R : first;
      if (begun || k > 0) {
        while (next < R && share.whole == 0 && ck_begin(share, next, R) == ck_begin(share, next + 1, R)) ++next;
        if (next < R && ck_begin(share, next, R) < rec.end) r = next++;
      }
      const bool there = r < R;
      more = there;
      const int64_t slot = (2 * (int64_t)(rec.base + (there ? r : first) * stride + g % stride) + (!there || r == first ? 1 : 0)) * WAVES + part;
      e[k] = a.part_ml[slot * 64 + lane];
#pragma unroll
      for (int i = 0; i < MINE; ++i) y[k][i] = ((const float4*)a.part)[(slot * QUADS + MINE * wave + i) * 64 + lane];
      if (!there) e[k] = make_float2(-INFINITY, 0.f);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) top = fmaxf(top, e[k].x);
    const float ref = top == -INFINITY ? 0.f : top, old = ck_exp2(m - ref);
    l *= old;
#pragma unroll
    for (int i = 0; i < MINE; ++i) { x[i].x *= old; x[i].y *= old; x[i].z *= old; x[i].w *= old; }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (e[k].x == -INFINITY) continue;       // (no such piece, or nothing in it)
      const float f = ck_exp2(e[k].x - ref);
      l = fmaf(e[k].y, f, l);
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
        x[i].x = fmaf(y[k][i].x, f, x[i].x); x[i].y = fmaf(y[k][i].y, f, x[i].y);
        x[i].z = fmaf(y[k][i].z, f, x[i].z); x[i].w = fmaf(y[k][i].w, f, x[i].w);
      }
    }
    m = top;
  }
  const int row = 32 * part + col, j = row / GC, gq = (rec.head % HS) * GC + row - j * GC;
  ck_results<D, KIND, 4, MINE>(a, x, ck_finish(l), matrix, j < rec.tokens && gq < a.G, rec.token + j, (rec.head / HS) * a.G + gq, rows);
}

// ---- launches ---------------------------------------------------------------------------------------------------------------------
// Scratch of the main kernels: a record a workgroup, and the pieces of two tiles (the sums of 32 rows, QUADS x 64 x 16 bytes, and their
// maxima and sums of weights) a wavefront of rows.
static inline int ck_groups(int per_cu) {
  const int cus = akv_cached_cu_count();
  return (cus > 0 ? cus : 256) * per_cu;
}
#define CK_GROUPS 2048            // workgroups of a launch at most
struct ck_scratch { size_t rec, ml, part, bytes; };
static inline ck_scratch ck_scratch_layout(int D) {
  const size_t wide = 2 * (size_t)ck_groups(1) * 8, slots = wide > 2 * CK_GROUPS ? wide : 2 * CK_GROUPS;      // (either kernel's)
  ck_scratch w;
  w.rec = 0;
  w.ml = akv_align256(CK_GROUPS * sizeof(ck_record));
  w.part = w.ml + akv_align256(slots * 64 * sizeof(float2));
  w.bytes = w.part + slots * (size_t)(D / 8) * 64 * 16;
  return w;
}
static inline uint32_t ck_reciprocal(int d) { return (uint32_t)(0xffffffffull / (uint32_t)d); }

static inline int ck_lds(const void* kernel, int bytes) {
  AKV_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  return AKV_OK;
}
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
  // Packed rows and float16: all of them as well.  The wide kernel has no registers for the queries' second term, without which float16
  // outputs are off by 4.2e-4 to 5.4e-4 of their size instead of 2.2e-4 (their own rounding is 2.1e-4) to 2.9e-4.  Time with this rule | without,
  // us, 4 bits, 32 heads: 12 turns of 1 to 90 tokens at heads of 64 75 | 94, of 128 126 | 117, of 256 312 | 444; two prompts of 1000 after 7000
  // 482 | 349, 768 | 459, 2117 | 1762.
  const bool few = most * a.G <= CK_NARROW_ROWS || (KIND >= 2 && a.dtype == AKV_F16), one = !few && a.S == 1;
  typedef ck_narrow<D, KIND> N;
  typedef ck_both<D, KIND> B;
  ck_args n = a, m = a;
  n.kind = few ? 0 : 1;
  n.HS = (a.G + 31) / 32;
  n.GC = (a.G + n.HS - 1) / n.HS;
  m.kind = one ? 0 : 2;
  m.HS = (a.G + W::ROWS - 1) / W::ROWS;
  m.GC = (a.G + m.HS - 1) / m.HS;
  const ck_cut cut = {n.HS, n.GC};
  const int heads = n.KVH * n.HS, most_groups = ck_groups(W::PER_CU);
  int dev = 0;
  AKV_HIP(hipGetDevice(&dev));
  if constexpr (B::FITS) {
    if (!few && !one && 2 * heads <= most_groups) {
      static akv_device_once once;
      if (const int rc = once(dev, [&]() -> int { return ck_lds((const void*)ck_both_kernel<D, KIND>, B::LDS); })) return rc;
      ck_both_kernel<D, KIND><<<most_groups, W::THREADS, B::LDS, stream>>>(n, m);
      AKV_LAUNCH_CHECK("ck_both_kernel");
      ck_merge_kernel<D, KIND, W::WAVES><<<dim3(most_groups, W::WAVES), 256, 0, stream>>>(m, cut);
      AKV_LAUNCH_CHECK("ck_merge_kernel");
      return AKV_OK;
    }
  }
  if (!one) {
    static akv_device_once once;
    if (const int rc = once(dev, [&]() -> int { return ck_lds((const void*)ck_narrow_kernel<D, KIND>, N::LDS); })) return rc;
    const int ranges = ck_groups(N::PER_CU) / heads, G = heads * (ranges > 1 ? ranges : 1);
    if (G > CK_GROUPS) return akv_fail(AKV_ERR_UNSUPPORTED, "more than %d kv heads", CK_GROUPS);
    ck_narrow_kernel<D, KIND><<<G, N::THREADS, N::LDS, stream>>>(n);
    AKV_LAUNCH_CHECK("ck_narrow_kernel");
    ck_merge_kernel<D, KIND, 1><<<dim3(G, 1), 256, 0, stream>>>(n, cut);
    AKV_LAUNCH_CHECK("ck_merge_kernel");
  }
  if (!few) {
    static akv_device_once once;
    if (const int rc = once(dev, [&]() -> int { return ck_lds((const void*)ck_wide_kernel<D, KIND>, W::LDS); })) return rc;
    ck_wide_kernel<D, KIND><<<most_groups, W::THREADS, W::LDS, stream>>>(m);
    AKV_LAUNCH_CHECK("ck_wide_kernel");
    ck_merge_kernel<D, KIND, W::WAVES><<<dim3(most_groups, W::WAVES), 256, 0, stream>>>(m, cut);
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
  if (num_blocks > 0x7fffffff) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: more than 2^31 blocks", name);
  if (T > 0x3fffffff || S > 0x3fffffff || T * (int64_t)QH > 0x7fffffff) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: more than 2^31 rows", name);
  return AKV_OK;
}
