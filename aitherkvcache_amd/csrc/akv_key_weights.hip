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
  uint16_t* turned; float* turned_by;   // packed: queries of the slab [KVH][rows][2][D], and what undoes their scale (times that of the scores)
  float2* part;                         // [parts][KVH][rows] maximum and sum
  float2* stat;                         // [KVH][rows] maximum and inverse sum
  float* out; int64_t os_seq, os_head;
  int64_t length;                       // floats of a row of the result
  int KVH, QH, G, t0, t1, add;
  uint32_t g_recip;
  int parts, splits;
  float* sums;                          // [splits][S][KVH][length], where there are several
  float* scores; int64_t stride;        // few rows: [token - t0][QH][stride]
  float2* few_part; int few_parts;      // [token - t0][QH][few_parts]
  int runs;
  bool by_token;                        // few rows: workgroups are numbered by the slab's tokens, not by the sequences
  float scale2;
};

template <int D, int KIND> struct kw_plan {
  static constexpr bool PACKED = KIND >= 2;
  static constexpr int DT = KIND == KW_BF16 ? AKV_BF16 : AKV_F16, KS = D / 16, TERMS = PACKED ? 2 : 1;
  static constexpr int KT = !PACKED && D <= 128 ? 2 : 1, N = 4 * 32 * KT;      // tiles of 32 keys a wavefront; keys of a part
  static constexpr int CHUNKS = TERMS * D / 8, BYTES = 16 * CHUNKS;         // of a row of queries
  static constexpr int ROW = BYTES + 16;                                    // in LDS: sixteen rows begin four banks apart each, and places are constants
  static constexpr int RT = 2, ROWS = 32 * RT;                              // many rows over plain keys: tiles and rows of a step
  static constexpr int LDS = 2 * ROWS * ROW;
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
__device__ __forceinline__ uint32_t kw_div(const kw_args& a, uint32_t row) {      // row / G
  uint32_t rest;
  return akv_div32(row, (uint32_t)a.G, a.g_recip, rest);
}
// token and head of row r
__device__ __forceinline__ void kw_row(const kw_args& a, const kw_rows& R, int kvh, int row, int& token, int& head) {
  uint32_t g;
  token = R.first + (int)akv_div32((uint32_t)row, (uint32_t)a.G, a.g_recip, g);
  head = kvh * a.G + (int)g;
}
// position of row r (the same in all lanes)
__device__ __forceinline__ int kw_pos(const kw_args& a, const kw_rows& R, int row) { return R.pos0 + (int)kw_div(a, (uint32_t)row); }
// where row `row` of a kv head lies in the arrays of the slab
__device__ __forceinline__ int64_t kw_slab_row(const kw_args& a, const kw_rows& R, int kvh, int row) {
  return (int64_t)kvh * ((int64_t)(a.t1 - a.t0) * a.G) + (int64_t)(R.first - a.t0) * a.G + row;
}
// ROWS rows into registers and from there to LDS; rows past the last are zero.
template <int D, int KIND, int ROWS> struct kw_stage {
  typedef kw_plan<D, KIND> P;
  static constexpr int LOADS = ROWS * P::CHUNKS / 256, AT_ONCE = 256 / P::CHUNKS;      // rows of a load
  ab_u4 v[LOADS];
  const uint8_t* p;                     // where the thread's first piece of row r0 lies
  int64_t load, step;                   // bytes from load to load, and from step to step (0: rows of a load are not whole tokens)
  __device__ __forceinline__ const uint8_t* at(const kw_args& a, const kw_rows& R, int kvh, int row) const {
    const int c = 16 * ((int)threadIdx.x % P::CHUNKS);
    if constexpr (P::PACKED) return (const uint8_t*)a.turned + kw_slab_row(a, R, kvh, row) * P::BYTES + c;
    int token, head;
    kw_row(a, R, kvh, row, token, head);
    return (const uint8_t*)a.q + 2 * ((int64_t)token * a.qs_tok + (int64_t)head * a.qs_head) + c;
  }
  // rows r0 .., and after that every `rows` behind
  __device__ __forceinline__ kw_stage(const kw_args& a, const kw_rows& R, int r0, int kvh, int rows) {
    p = at(a, R, kvh, r0 + (int)threadIdx.x / P::CHUNKS);
    if constexpr (P::PACKED) {
      load = AT_ONCE * P::BYTES;
      step = (int64_t)rows * P::BYTES;
    } else {
      const bool whole = AT_ONCE % a.G == 0 && rows % a.G == 0;
      load = whole ? 2 * (int64_t)(AT_ONCE / a.G) * a.qs_tok : 0;
      step = whole ? 2 * (int64_t)(rows / a.G) * a.qs_tok : 0;
    }
  }
  __device__ __forceinline__ void request(const kw_args& a, const kw_rows& R, int r0, int kvh) {
    if (r0 + ROWS <= R.rows && step != 0) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) v[i] = *(const ab_u4*)(p + i * load);
    } else {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int row = r0 + AT_ONCE * i + (int)threadIdx.x / P::CHUNKS;
        v[i] = (ab_u4){0u, 0u, 0u, 0u};
        if (row < R.rows) v[i] = *(const ab_u4*)at(a, R, kvh, row);
      }
    }
    p += step;
  }
  __device__ __forceinline__ void put(unsigned char* lds) const {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) *(ab_u4*)(lds + (AT_ONCE * i + (int)threadIdx.x / P::CHUNKS) * P::ROW + 16 * ((int)threadIdx.x % P::CHUNKS)) = v[i];
  }
};

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
  static constexpr int W = P::PACKED ? D * (P::PACKED ? KIND : 4) / 64 : 1;      // packed: words of half a row
  ab_u4 hi[P::KT][P::KS], lo[P::PACKED ? P::KT : 1][P::PACKED ? P::KS : 1];
  uint32_t raw[P::PACKED ? P::KT : 1][W];
  float norm[P::KT], raw_norm[P::KT];   // packed: of the lane's key
  // keys base .. base + 32 KT - 1 of a sequence of ctx > base tokens (those past the last: the last); packed: as they lie in memory
  __device__ __forceinline__ void request(const kw_args& a, int seq, int kvh, int base, int ctx) {
    const int lane = threadIdx.x & 63, h = lane >> 5, col = lane & 31;
    ab_entry e[P::KT];
    uint32_t place[P::KT];
#pragma unroll
    for (int t = 0; t < P::KT; ++t) {
      const int key = min(base + 32 * t + col, ctx - 1);
      e[t] = ab_look(a.b, seq, akv_div32((uint32_t)key, (uint32_t)a.b.block_size, a.b.bs_recip, place[t]));
    }
#pragma unroll
    for (int t = 0; t < P::KT; ++t) {
      const int64_t blk = ab_block(a.b, e[t]);
      const uint8_t* p = a.k + blk * a.k_blk + (int64_t)place[t] * a.k_pos + (int64_t)kvh * a.k_head;
      if constexpr (!P::PACKED) {
#pragma unroll
        for (int ks = 0; ks < P::KS; ++ks) hi[t][ks] = *(const ab_u4*)(p + 32 * ks + 16 * h);
      } else {
        struct __attribute__((packed, aligned(4))) words { uint32_t v[W]; };      // (rows lie at multiples of four bytes)
        const words x = *(const words*)(p + 4 * W * h);
#pragma unroll
        for (int i = 0; i < W; ++i) raw[t][i] = x.v[i];
        raw_norm[t] = a.kn[blk * a.kn_blk + (int64_t)place[t] * a.kn_pos + (int64_t)kvh * a.kn_head];
      }
    }
  }
  // packed: codes to levels
  __device__ __forceinline__ void decode(const uint32_t* levels, float unit) {
    if constexpr (P::PACKED) {
#pragma unroll
      for (int t = 0; t < P::KT; ++t) {
        norm[t] = raw_norm[t] * unit;
#pragma unroll
        for (int ks = 0; ks < P::KS; ++ks)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t x = levels[kw_code<KIND>(raw[t], ks, 2 * i)], y = levels[kw_code<KIND>(raw[t], ks, 2 * i + 1)];
            hi[t][ks][i] = __builtin_amdgcn_perm(y, x, 0x05040100u);
            lo[t][ks][i] = __builtin_amdgcn_perm(y, x, 0x07060302u);
          }
      }
    }
  }
  // products of the tiles with the 32 rows in LDS; KEYS_FIRST: a key's are in the registers, a row's in a lane.  Rows come out of LDS in runs, one of
  // them on its way while the one before is multiplied (left to itself the compiler asks for one operand at a time and waits for it).
  template <bool KEYS_FIRST> __device__ __forceinline__ void products(const unsigned char* rows, ab_f16 (&s)[P::KT]) const {
    typedef ab_math<P::DT> M;
    constexpr int STEPS = P::PACKED ? D == 256 ? 1 : 2 : 4, RUNS = P::KS / STEPS;
    const int lane = threadIdx.x & 63, h = lane >> 5, col = lane & 31;
    const unsigned char* r = rows + col * P::ROW + 16 * (P::PACKED ? P::KS * h : h);
    ab_u4 q[2][STEPS][P::TERMS];
    auto read = [&](int run) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        // (packed: a lane has the half row h, plain: half of every sixteen coordinates)
        const int ks = run * STEPS + i;
#pragma unroll
        for (int e = 0; e < P::TERMS; ++e) q[run & 1][i][e] = *(const ab_u4*)(r + 16 * (e * (D / 8) + (P::PACKED ? ks : 2 * ks)));
      }
    };
#pragma unroll
    for (int t = 0; t < P::KT; ++t) s[t] = (ab_f16)(0.f);
    read(0);
#pragma unroll
    for (int run = 0; run < RUNS; ++run) {
      __builtin_amdgcn_sched_barrier(0);
      if (run + 1 < RUNS) read(run + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int ks = run * STEPS + i;
#pragma unroll
        for (int t = 0; t < P::KT; ++t) {
          const ab_u4(&x)[P::TERMS] = q[run & 1][i];
          if constexpr (P::PACKED) {
            s[t] = KEYS_FIRST ? M::mfma32(lo[t][ks], x[0], s[t]) : M::mfma32(x[0], lo[t][ks], s[t]);
            s[t] = KEYS_FIRST ? M::mfma32(hi[t][ks], x[1], s[t]) : M::mfma32(x[1], hi[t][ks], s[t]);
          }
          s[t] = KEYS_FIRST ? M::mfma32(hi[t][ks], x[0], s[t]) : M::mfma32(x[0], hi[t][ks], s[t]);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
};

// ---- queries of packed rows: turned, scaled and as two terms.  32 rows a tile and 32 coordinates a wavefront: queries are 16-bit numbers as they are, an entry of the
// rotation three of their type, so that products and sums are float32 like those of one number after the other.  A workgroup's part of the rotation
// stays in registers for all of its tiles, queries go through LDS, the next tile's on their way.  4096 rows of 128 take 6.4 us and 47000 15, where a row of the
// rotation after the other, for eight rows a workgroup, took 9 and 43; queries in the operand's order straight from memory 7 and 18.  213000 rows of 256 take
// 117: one workgroup a CU, whose registers hold the rotation's part, multiplies and writes in turn.
template <int D, int DT> __global__ __launch_bounds__(2 * D) void kw_turn_kernel(kw_args a) {
  typedef ab_math<DT> M;
  constexpr int KS = D / 16, LANES = D / 16;         // LANES: threads of a row, in the end
  __shared__ __align__(16) float x[32][D + 4];
  __shared__ __align__(16) uint16_t in[32][D + 8];   // queries: rows arrive in the order in which they lie
  const uint32_t rows = (uint32_t)(a.t1 - a.t0) * (uint32_t)a.QH, QH = (uint32_t)a.QH;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, col = lane & 31;
  // an entry times 2^12 in float16 (a rotation's are 1 at most), so that its third term is a normal number
  constexpr float UP = DT == AKV_F16 ? 4096.f : 1.f;
  ab_u4 pi[3][KS];
  const float* const turn = a.turn + 32 * wave + col;
#pragma unroll
  for (int k = 0; k < KS; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float u = turn[(16 * k + 8 * h + 2 * e) * D] * UP, v = turn[(16 * k + 8 * h + 2 * e + 1) * D] * UP;
#pragma unroll
      for (int part = 0; part < 3; ++part) {
        const uint32_t two = M::pair(u, v);
        pi[part][k][e] = two;
        u -= M::low(two);
        v -= M::high(two);
      }
    }
  ab_u4 next[2];
  auto request = [&](uint32_t r0) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t p = tid + j * 2 * D, r = min(r0 + p / (D / 8), rows - 1), token = r / QH;
      next[j] = *(const ab_u4*)((const uint16_t*)a.q + (int64_t)(token + (uint32_t)a.t0) * a.qs_tok + (int64_t)(r - token * QH) * a.qs_head + 8 * (p % (D / 8)));
    }
  };
  request(32 * blockIdx.x);
  for (uint32_t r0 = 32 * blockIdx.x; r0 < rows; r0 += 32 * gridDim.x) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t p = tid + j * 2 * D;
      *(ab_u4*)&in[p / (D / 8)][8 * (p % (D / 8))] = next[j];
    }
    __syncthreads();
    if (r0 + 32 * gridDim.x < rows) request(r0 + 32 * gridDim.x);
    ab_f16 s[3];
#pragma unroll
    for (int part = 0; part < 3; ++part)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[part][i] = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const ab_u4 y = *(const ab_u4*)&in[col][16 * k + 8 * h];
#pragma unroll
      for (int part = 0; part < 3; ++part) s[part] = M::mfma32(y, pi[part][k], s[part]);
    }
    __syncthreads();                   // (the tile before has been read)
#pragma unroll
    for (int i = 0; i < 16; ++i) x[8 * (i / 4) + 4 * h + i % 4][32 * wave + col] = (s[0][i] + (s[1][i] + s[2][i])) * (1.f / UP);
    __syncthreads();
    // sixteen numbers of a row a thread: scaled so that the largest lies in [2^13, 2^14), and as two terms
    const uint32_t i = tid / LANES, part = tid % LANES;
    ab_f4 v[4];
    float t = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = *(const ab_f4*)&x[i][4 * (part + LANES * j)];
      t = fmaxf(fmaxf(fmaxf(t, fabsf(v[j][0])), fmaxf(fabsf(v[j][1]), fabsf(v[j][2]))), fabsf(v[j][3]));
    }
    t = fmaxf(t, akv_lane_xor<1>(t));
    t = fmaxf(t, akv_lane_xor<2>(t));
    if constexpr (LANES > 4) t = fmaxf(t, akv_lane_xor<4>(t));
    if constexpr (LANES > 8) t = fmaxf(t, akv_lane_xor<8>(t));
    if (r0 + i < rows) {
      // (no exponent below 14: the scale of a row of zeros, or next to it, is a number, 2^126 at most)
      const uint32_t exponent = max(akv_row_exponent(t), 14u), token = (r0 + i) / QH, head = r0 + i - token * QH, kvh = kw_div(a, head);
      const int64_t to = (int64_t)kvh * (a.t1 - a.t0) * a.G + (int64_t)token * a.G + (head - kvh * a.G);
      const float scale = akv_row_scale(exponent) * 8192.f;
      typedef _Float16 four __attribute__((ext_vector_type(4)));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        four hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float u = v[j][e] * scale;
          hi[e] = (_Float16)u;
          lo[e] = (_Float16)(u - (float)hi[e]);
        }
        *(four*)(a.turned + to * (2 * D) + 4 * (part + LANES * j)) = hi;
        *(four*)(a.turned + to * (2 * D) + D + 4 * (part + LANES * j)) = lo;
      }
      // (above zero, whatever the scale of the scores: what is masked is -infinity times it.  A score of such a row is below 2^-96 of the key's norm)
      if (part == 0) a.turned_by[to] = fmaxf(akv_row_unscale(exponent) * (1.f / 8192.f) * a.scale2, 0x1p-126f);
    }
  }
}

// maximum and sum of a lane's row over the wavefront's keys; c: what makes scores of the products
template <int KT> __device__ __forceinline__ void kw_row_stats(const ab_f16 (&s)[KT], float c, float& m, float& l) {
  float a = s[0][0], b = s[0][1];
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int i = t == 0 ? 2 : 0; i < 16; i += 2) {
      a = fmaxf(a, s[t][i]);
      b = fmaxf(b, s[t][i + 1]);
    }
  a = fmaxf(a, b);
  m = fmaxf(a, akv_lane_xor<32>(a)) * c;
  const float ref = m == -INFINITY || m != m ? 0.f : m;
  float l0 = 0.f, l1 = 0.f;
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      l0 += __builtin_amdgcn_exp2f(fmaf(s[t][i], c, -ref));
      l1 += __builtin_amdgcn_exp2f(fmaf(s[t][i + 1], c, -ref));
    }
  l = l0 + l1;
  l += akv_lane_xor<32>(l);
  if (m != m || m == -INFINITY) m = -INFINITY, l = 0.f;      // (-inf times 0: a row that is none)
}

// what is left of a row over a part: maximum and sum for kw_join, or, of the only part, what kw_join would make of them
__device__ __forceinline__ float2 kw_stat(const kw_args& a, float top, float sum) {
  return a.parts > 1 ? make_float2(top, sum) : sum > 0.f ? make_float2(top, 1.f / sum) : make_float2(0.f, 0.f);
}
// ---- many rows over plain keys: maxima and sums of the rows over a part of the keys, 32 KT of them a wavefront.  Rows are requested a step of ROWS ahead, and a step
// has one barrier.  Workgroups of `splits` take steps in turn.
// 1024 tokens after 7000, 16 heads on 4, heads of 256: 79 us, and 80 for kw_sum below, 790 TFLOP/s each (matrix cores 37 % of clocks, LDS 37 %, vector unit
// 29 %): a step's operands come from LDS, its maxima are taken, and the next step waits for both.
template <int D, int KIND> __global__ __launch_bounds__(256, 2) void kw_stats_kernel(kw_args a) {
  typedef kw_plan<D, KIND> P;
  constexpr int ROWS = P::ROWS, RT = P::RT;
  extern __shared__ __align__(16) unsigned char rows[];          // [2][ROWS][ROW]
  __shared__ float2 ml[2][4][ROWS];
  const int part = blockIdx.x / a.splits, split = blockIdx.x % a.splits, kvh = blockIdx.y, seq = blockIdx.z;
  const int ctx = ab_ctx(a.b, seq), from = part * P::N;
  if (from >= ctx) return;
  const kw_rows R = kw_rows_of(a, seq, ctx);
  if (R.rows == 0 || R.pos0 + (R.rows - 1) / a.G < from) return;
  const int first = (max(0, from - R.pos0) * a.G / ROWS + split) * ROWS, step = ROWS * a.splits;      // rows before see nothing of the part
  if (first >= R.rows) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, col = lane & 31;
  const int base = from + 32 * P::KT * wave;
  kw_stage<D, KIND, ROWS> next(a, R, first, kvh, step);
  next.request(a, R, first, kvh);
  kw_keys<D, KIND> K;
  const bool any = base < ctx;
  if (any) K.request(a, seq, kvh, base, ctx);
  const int64_t slab = kw_slab_row(a, R, kvh, 0);
  float2* to = (a.parts == 1 ? a.stat : a.part + (int64_t)part * a.KVH * ((int64_t)(a.t1 - a.t0) * a.G)) + slab;
  // what the wavefronts have of a step's rows, together: four lanes a row, every wavefront a quarter
  auto join = [&](int r0, int buf) {
    const int r = ROWS / 4 * wave + (lane >> 2);
    if (lane < ROWS) {
      const float2 e = ml[buf][lane & 3][r];
      float top = fmaxf(e.x, akv_lane_xor<1>(e.x));
      top = fmaxf(top, akv_lane_xor<2>(top));
      float sum = e.x == -INFINITY ? 0.f : e.y * __builtin_amdgcn_exp2f(e.x - top);
      sum += akv_lane_xor<1>(sum);
      sum += akv_lane_xor<2>(sum);
      if ((lane & 3) == 0 && r0 + r < R.rows) to[r0 + r] = kw_stat(a, top, sum);
    }
  };
  next.put(rows);
  int buf = 0, r0 = first;
  for (;; r0 += step, buf ^= 1) {
    __syncthreads();
    const bool more = r0 + step < R.rows;
    if (more) next.request(a, R, r0 + step, kvh);
    if (r0 > first) join(r0 - step, buf ^ 1);
    if (any) {
#pragma unroll 1
      for (int i = 0; i < RT; ++i) {
        const int row = r0 + 32 * i + col;
        float m, l;
        ab_f16 s[P::KT];
        K.template products<true>(rows + (ROWS * buf + 32 * i) * P::ROW, s);
        if (base + 32 * P::KT - 1 > kw_pos(a, R, min(r0 + 32 * i, R.rows - 1))) {
          const int pos = row < R.rows ? kw_pos(a, R, row) : -1;
#pragma unroll
          for (int t = 0; t < P::KT; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) s[t][e] = base + 32 * t + 8 * (e >> 2) + 4 * h + (e & 3) <= pos ? s[t][e] : -INFINITY;
        }
        kw_row_stats<P::KT>(s, a.scale2, m, l);
        if (h == 0) ml[buf][wave][32 * i + col] = make_float2(m, l);
      }
    } else if (h == 0) {
#pragma unroll
      for (int i = 0; i < RT; ++i) ml[buf][wave][32 * i + col] = make_float2(-INFINITY, 0.f);
    }
    if (!more) break;
    next.put(rows + ROWS * (buf ^ 1) * P::ROW);
  }
  __syncthreads();
  join(r0, buf);
}

// ---- the parts of a row together: a lane a row, as they lie in memory, and every wavefront a quarter of the parts.  16384 rows of 59 parts take 5 us (9.4 with
// a wavefront a row, whose lanes read a line each).
__global__ __launch_bounds__(256) void kw_join_kernel(kw_args a, int keys) {
  __shared__ float2 quarter[4][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kvh = blockIdx.y;
  const int64_t all = (int64_t)(a.t1 - a.t0) * a.G, row = (int64_t)blockIdx.x * 64 + lane;
  const int token = a.t0 + (int)kw_div(a, (uint32_t)min(row, all - 1)), last = __builtin_amdgcn_readlane(token, 63);
  // positions of the rows; sequence by sequence
  int pos = -1;
  for (int at = __builtin_amdgcn_readfirstlane(token); at <= last;) {
    const int seq = ab_last(a.b.S, at, [&](int i) { return (int64_t)ab_start(a.b, i); });
    const int s1 = ab_start(a.b, seq + 1);           // (seq = -1: rows before the first)
    if (s1 <= at) break;
    if (seq >= 0 && token >= at && token < s1) pos = ab_ctx(a.b, seq) - (s1 - token);
    at = s1;
  }
  const int count = pos < 0 ? 0 : pos / keys + 1;
  float m = -INFINITY, l = 0.f;
  for (int p0 = wave; __ballot(p0 < count); p0 += 32) {
    float2 e[8];                        // (on their way together)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      e[i] = make_float2(-INFINITY, 0.f);
      if (p0 + 4 * i < count) e[i] = a.part[((int64_t)(p0 + 4 * i) * a.KVH + kvh) * all + row];
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, e[i].x);
    if (top == -INFINITY) continue;
    l *= __builtin_amdgcn_exp2f(m - top);
#pragma unroll
    for (int i = 0; i < 8; ++i) l = fmaf(e[i].y, __builtin_amdgcn_exp2f(e[i].x - top), l);
    m = top;
  }
  quarter[wave][lane] = make_float2(m, l);
  __syncthreads();
  if (wave > 0 || row >= all) return;
  float top = m;
#pragma unroll
  for (int w = 1; w < 4; ++w) top = fmaxf(top, quarter[w][lane].x);
  float sum = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) sum += quarter[w][lane].x == -INFINITY ? 0.f : quarter[w][lane].y * __builtin_amdgcn_exp2f(quarter[w][lane].x - top);
  a.stat[kvh * all + row] = sum > 0.f ? make_float2(top, 1.f / sum) : make_float2(0.f, 0.f);
}

// Weights of 32 rows from row0 on, added up for the lane's keys base + 32 t + lane % 32: reference, inverse sum and (packed) scale of each row, from the
// lane's first one; norms of the keys.
template <int D, int KIND>
__device__ __forceinline__ void kw_weights(const kw_args& a, const kw_rows& R, ab_f16 (&s)[kw_plan<D, KIND>::KT], const float* ref, const float* inv, const float* by,
                                           const float* norm, int row0, int base, float (&w)[kw_plan<D, KIND>::KT]) {
  typedef kw_plan<D, KIND> P;
  const int h = (threadIdx.x & 63) >> 5, col = threadIdx.x & 31;
  if constexpr (P::PACKED) {
#pragma unroll
    for (int t = 0; t < P::KT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[t][i] *= norm[t];
  }
  if (base + 32 * P::KT - 1 > kw_pos(a, R, min(row0, R.rows - 1))) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int row = row0 + 8 * (i >> 2) + 4 * h + (i & 3), pos = row < R.rows ? kw_pos(a, R, row) : 0x7fffffff;      // (rows past the last weigh nothing, and have no scale)
#pragma unroll
      for (int t = 0; t < P::KT; ++t) s[t][i] = base + 32 * t + col <= pos ? s[t][i] : -INFINITY;
    }
  }
  float sum[P::KT][4] = {};
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const float4 m4 = *(const float4*)(ref + 8 * b), i4 = *(const float4*)(inv + 8 * b);
    float c[4] = {a.scale2, a.scale2, a.scale2, a.scale2};
    if constexpr (P::PACKED) {
      const float4 x = *(const float4*)(by + 8 * b);
      c[0] = x.x; c[1] = x.y; c[2] = x.z; c[3] = x.w;
    }
    const float m[4] = {m4.x, m4.y, m4.z, m4.w}, iv[4] = {i4.x, i4.y, i4.z, i4.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int t = 0; t < P::KT; ++t) sum[t][j] = fmaf(__builtin_amdgcn_exp2f(fmaf(s[t][4 * b + j], c[j], -m[j])), iv[j], sum[t][j]);
  }
#pragma unroll
  for (int t = 0; t < P::KT; ++t) w[t] += (sum[t][0] + sum[t][1]) + (sum[t][2] + sum[t][3]);
}

// ---- weights of a part's keys, summed over the rows; steps as above.  Workgroups that share a part leave their sums to kw_add_kernel.
template <int D, int KIND> __global__ __launch_bounds__(256, 2) void kw_sum_kernel(kw_args a) {
  typedef kw_plan<D, KIND> P;
  constexpr int ROWS = P::ROWS, RT = P::RT;
  extern __shared__ __align__(16) unsigned char rows[];          // [2][ROWS][ROW]
  __shared__ __align__(16) float ref[2][ROWS], inv[2][ROWS];
  const int part = blockIdx.x / a.splits, split = blockIdx.x % a.splits, kvh = blockIdx.y, seq = blockIdx.z;
  const int ctx = ab_ctx(a.b, seq);
  const int64_t from = (int64_t)part * P::N;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, col = lane & 31;
  const bool add = a.add && a.splits == 1;
  float* to = a.splits == 1 ? a.out + (int64_t)seq * a.os_seq + (int64_t)kvh * a.os_head : a.sums + (((int64_t)split * a.b.S + seq) * a.KVH + kvh) * a.length;
  const kw_rows R = kw_rows_of(a, seq, ctx);
  const int first = from < ctx ? (max(0, (int)from - R.pos0) * a.G / ROWS + split) * ROWS : R.rows, step = ROWS * a.splits;
  if (first >= R.rows || R.pos0 + (R.rows - 1) / a.G < from) {
    if (!add)
      for (int64_t i = from + tid; i < from + P::N && i < a.length; i += 256) to[i] = 0.f;
    return;
  }
  const int base = (int)from + 32 * P::KT * wave;
  const int64_t slab = kw_slab_row(a, R, kvh, 0);
  kw_stage<D, KIND, ROWS> next(a, R, first, kvh, step);
  float2 e = make_float2(0.f, 0.f);
  auto request = [&](int r0) {
    next.request(a, R, r0, kvh);
    if (tid < ROWS) {
      e = r0 + tid < R.rows ? a.stat[slab + r0 + tid] : make_float2(0.f, 0.f);
    }
  };
  auto put = [&](int buf) {
    next.put(rows + ROWS * buf * P::ROW);
    if (tid < ROWS) {
      ref[buf][tid] = e.x;
      inv[buf][tid] = e.y;
    }
  };
  request(first);
  kw_keys<D, KIND> K;
  const bool any = base < ctx;
  if (any) K.request(a, seq, kvh, base, ctx);
  float w[P::KT] = {};
  put(0);
  int buf = 0;
  for (int r0 = first;; r0 += step, buf ^= 1) {
    __syncthreads();
    const bool more = r0 + step < R.rows;
    if (more) request(r0 + step);
    if (any) {
#pragma unroll 1
      for (int i = 0; i < RT; ++i) {
        const int row0 = r0 + 32 * i;
        ab_f16 s[P::KT];
        K.template products<false>(rows + (ROWS * buf + 32 * i) * P::ROW, s);
        const float* rf = ref[buf] + 32 * i + 4 * h;
        const float* iv = inv[buf] + 32 * i + 4 * h;
        kw_weights<D, KIND>(a, R, s, rf, iv, nullptr, nullptr, row0, base, w);
      }
    }
    if (!more) break;
    put(buf ^ 1);
  }
#pragma unroll
  for (int t = 0; t < P::KT; ++t) {
    const float sum = w[t] + akv_lane_xor<32>(w[t]);
    const int64_t key = (int64_t)base + 32 * t + col;
    if (h == 0 && key < a.length) {
      if (key < ctx) to[key] = add ? to[key] + sum : sum;
      else if (!add) to[key] = 0.f;
    }
  }
}
// the sums of the workgroups that share a part, in their order
__global__ __launch_bounds__(256) void kw_add_kernel(kw_args a) {
  const int64_t key = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int kvh = blockIdx.y, seq = blockIdx.z;
  if (key >= a.length) return;
  float sum = 0.f;
  for (int s = 0; s < a.splits; ++s) sum += a.sums[(((int64_t)s * a.b.S + seq) * a.KVH + kvh) * a.length + key];
  float* to = a.out + (int64_t)seq * a.os_seq + (int64_t)kvh * a.os_head + key;
  if (!a.add) *to = sum;
  else if (key < ab_ctx(a.b, seq)) *to += sum;
}

// ---- many rows over packed keys: a block of rows stays in LDS while the wavefronts walk through `runs` x N keys, each by itself, the next codes on their
// way: codes are a quarter of the keys' bytes and cost more to turn into levels than to read again for the next block of rows.  Workgroups of
// `splits` take blocks in turn.
// The last 32 tokens of four prompts of up to 16352 keys, 32 heads on 8, 4 bits: 42 us, and 40 for the sum below (vector unit 36 % of clocks, matrix cores 29 %, LDS
// 25 %): three products a score, and codes turned into levels twice.
template <int D> struct kw_block { static constexpr int ROWS = D == 256 ? 64 : 128; };
// rows r0 .. into LDS, those past the last as zeros
template <int D, int KIND> __device__ __forceinline__ void kw_put_block(const kw_args& a, const kw_rows& R, int r0, int kvh, unsigned char* rows) {
  typedef kw_plan<D, KIND> P;
  constexpr int ROWS = kw_block<D>::ROWS, LOADS = ROWS * P::CHUNKS / 256, AT_ONCE = 256 / P::CHUNKS;
  const int r = (int)threadIdx.x / P::CHUNKS, c = 16 * ((int)threadIdx.x % P::CHUNKS);
  const uint8_t* p = (const uint8_t*)a.turned + kw_slab_row(a, R, kvh, r0 + r) * P::BYTES + c;
#pragma unroll
  for (int i0 = 0; i0 < LOADS; i0 += 8) {
    ab_u4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = r0 + AT_ONCE * (i0 + i) + r < R.rows ? *(const ab_u4*)(p + (int64_t)(AT_ONCE * (i0 + i)) * P::BYTES) : (ab_u4){0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) *(ab_u4*)(rows + (AT_ONCE * (i0 + i) + r) * P::ROW + c) = v[i];
  }
}
template <int D, int KIND> __global__ __launch_bounds__(256, 2) void kw_packed_stats_kernel(kw_args a) {
  typedef kw_plan<D, KIND> P;
  constexpr int ROWS = kw_block<D>::ROWS;
  constexpr bool AHEAD = D < 256;       // (the next codes have registers)
  extern __shared__ __align__(16) unsigned char rows[];          // [ROWS][ROW]
  __shared__ float2 ml[4][ROWS];
  __shared__ float by[ROWS];
  __shared__ __align__(16) float norms[P::N];
  __shared__ kw_levels<KIND> levels;
  const int part = blockIdx.x / a.splits, split = blockIdx.x % a.splits, kvh = blockIdx.y, seq = blockIdx.z;
  const int ctx = ab_ctx(a.b, seq);
  const int64_t from64 = (int64_t)part * P::N * a.runs;
  if (from64 >= ctx) return;
  const int from = (int)from64;
  const kw_rows R = kw_rows_of(a, seq, ctx);
  if (R.rows == 0 || kw_pos(a, R, R.rows - 1) < from) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, col = lane & 31;
  const float unit = kw_fill(levels, a.centroids);
  const int64_t slab = kw_slab_row(a, R, kvh, 0);
  float2* to = (a.parts == 1 ? a.stat : a.part + (int64_t)part * a.KVH * ((int64_t)(a.t1 - a.t0) * a.G)) + slab;
  for (int r0 = ROWS * split; r0 < R.rows; r0 += ROWS * a.splits) {
    const int count = min(ROWS, R.rows - r0), last = kw_pos(a, R, r0 + count - 1), end = min(from + P::N * a.runs, last + 1);
    if (last < from) continue;
    kw_keys<D, KIND> K;
    int base = from + 32 * P::KT * wave;
    if (AHEAD && base < end) K.request(a, seq, kvh, base, ctx);
    __syncthreads();                   // (the block before has been read)
    kw_put_block<D, KIND>(a, R, r0, kvh, rows);
    if (tid < ROWS) by[tid] = tid < count ? a.turned_by[slab + r0 + tid] : 0.f;
    for (int i = lane; i < ROWS; i += 64) ml[wave][i] = make_float2(-INFINITY, 0.f);
    __syncthreads();
    for (; base < end; base += P::N) {
      if (!AHEAD) K.request(a, seq, kvh, base, ctx);
      K.decode(levels.level, unit);
      akv_wave_sync();
      if (h == 0)
#pragma unroll
        for (int t = 0; t < P::KT; ++t) norms[32 * (P::KT * wave + t) + col] = K.norm[t];
      akv_wave_sync();
      if (AHEAD && base + P::N < end) K.request(a, seq, kvh, base + P::N, ctx);
#pragma unroll 1
      for (int i = 0; i < count; i += 32) {
        if (kw_pos(a, R, min(r0 + i + 31, R.rows - 1)) < base) continue;
        ab_f16 s[P::KT];
        K.template products<true>(rows + i * P::ROW, s);
#pragma unroll
        for (int t = 0; t < P::KT; ++t)
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const float4 n = *(const float4*)(norms + 32 * (P::KT * wave + t) + 8 * b + 4 * h);
            s[t][4 * b] *= n.x; s[t][4 * b + 1] *= n.y; s[t][4 * b + 2] *= n.z; s[t][4 * b + 3] *= n.w;
          }
        if (base + 32 * P::KT - 1 > kw_pos(a, R, r0 + i)) {
          const int pos = i + col < count ? kw_pos(a, R, r0 + i + col) : -1;
#pragma unroll
          for (int t = 0; t < P::KT; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) s[t][e] = base + 32 * t + 8 * (e >> 2) + 4 * h + (e & 3) <= pos ? s[t][e] : -INFINITY;
        }
        float m, l;
        kw_row_stats<P::KT>(s, by[i + col], m, l);
        const float2 old = ml[wave][i + col];
        const float top = fmaxf(old.x, m), ref = top == -INFINITY ? 0.f : top;
        l = old.y * __builtin_amdgcn_exp2f(old.x - ref) + l * __builtin_amdgcn_exp2f(m - ref);
        if (h == 0) ml[wave][i + col] = make_float2(top, l);
      }
    }
    __syncthreads();
    if (tid < count) {
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, ml[w][tid].x);
#pragma unroll
      for (int w = 0; w < 4; ++w) sum += ml[w][tid].x == -INFINITY ? 0.f : ml[w][tid].y * __builtin_amdgcn_exp2f(ml[w][tid].x - top);
      to[r0 + tid] = kw_stat(a, top, sum);
    }
  }
}
template <int D, int KIND> __global__ __launch_bounds__(256, 2) void kw_packed_sum_kernel(kw_args a) {
  typedef kw_plan<D, KIND> P;
  constexpr int ROWS = kw_block<D>::ROWS;
  constexpr bool AHEAD = D < 256;       // (the next codes have registers)
  extern __shared__ __align__(16) unsigned char rows[];          // [ROWS][ROW]
  __shared__ __align__(16) float ref[ROWS], inv[ROWS], by[ROWS];
  __shared__ kw_levels<KIND> levels;
  const int part = blockIdx.x / a.splits, split = blockIdx.x % a.splits, kvh = blockIdx.y, seq = blockIdx.z;
  const int ctx = ab_ctx(a.b, seq);
  const int64_t from = (int64_t)part * P::N * a.runs;
  const kw_rows R = kw_rows_of(a, seq, ctx);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, col = lane & 31;
  float* to = a.splits == 1 ? a.out + (int64_t)seq * a.os_seq + (int64_t)kvh * a.os_head : a.sums + (((int64_t)split * a.b.S + seq) * a.KVH + kvh) * a.length;
  bool add = a.add && a.splits == 1;    // (the first block that sees something of the keys writes, the others add)
  auto zeros = [&]() {
    for (int64_t i = from + tid; i < from + P::N * a.runs && i < a.length; i += 256) to[i] = 0.f;
  };
  if (from >= ctx || R.rows == 0 || kw_pos(a, R, R.rows - 1) < from) {
    if (!add) zeros();
    return;
  }
  const float unit = kw_fill(levels, a.centroids);
  const int64_t slab = kw_slab_row(a, R, kvh, 0);
  for (int r0 = ROWS * split; r0 < R.rows; r0 += ROWS * a.splits) {
    const int count = min(ROWS, R.rows - r0), last = kw_pos(a, R, r0 + count - 1);
    if (last < from) continue;
    kw_keys<D, KIND> K;
    int base = (int)from + 32 * P::KT * wave;
    const int64_t behind = min(from + P::N * a.runs, a.length);
    if (AHEAD && base <= last) K.request(a, seq, kvh, base, ctx);
    __syncthreads();                   // (the block before has been read)
    kw_put_block<D, KIND>(a, R, r0, kvh, rows);
    if (tid < ROWS) {
      const float2 e = tid < count ? a.stat[slab + r0 + tid] : make_float2(0.f, 0.f);
      ref[tid] = e.x;
      inv[tid] = e.y;
      by[tid] = tid < count ? a.turned_by[slab + r0 + tid] : 0.f;
    }
    __syncthreads();
    for (; base < behind; base += P::N) {
      float w[P::KT] = {};
      if (base <= last) {
        if (!AHEAD) K.request(a, seq, kvh, base, ctx);
        K.decode(levels.level, unit);
        if (AHEAD && base + P::N <= last && base + P::N < behind) K.request(a, seq, kvh, base + P::N, ctx);
#pragma unroll 1
        for (int i = 0; i < count; i += 32) {
          if (kw_pos(a, R, min(r0 + i + 31, R.rows - 1)) < base) continue;
          ab_f16 s[P::KT];
          K.template products<false>(rows + i * P::ROW, s);
          const int at = i + 4 * h;
          kw_weights<D, KIND>(a, R, s, ref + at, inv + at, by + at, K.norm, r0 + i, base, w);
        }
      }
#pragma unroll
      for (int t = 0; t < P::KT; ++t) {
        const float sum = w[t] + akv_lane_xor<32>(w[t]);
        const int64_t key = (int64_t)base + 32 * t + col;
        if (h == 0 && key < a.length) {
          if (!add) to[key] = key < ctx ? sum : 0.f;
          else if (key <= last) to[key] += sum;
        }
      }
    }
    add = true;
  }
  if (!add) zeros();                    // (none of the workgroup's blocks does)
}

// ---- few rows a sequence: keys are read once, as long as a sequence and kv head has no more rows than a tile; scores are kept, four bytes a row and
// key, and read back by kw_few_sum with the statistics of the rows.  A workgroup of four wavefronts takes `runs` x N keys, the next ones on
// their way while the ones before are multiplied.
// One token of 16 sequences, 1024 to 41000 keys each, 8 heads of 128: 120 us, 4.3 TB/s of what is read; kw_few_sum 15.
#define KW_FEW 32
// The sequence of a workgroup, or -1.  Where a slab has half as many tokens as there are sequences, or fewer, workgroups are numbered by its tokens: the first one that a
// sequence has in the slab stands for the sequence.
__device__ __forceinline__ int kw_few_seq(const kw_args& a) {
  if (!a.by_token) return blockIdx.z;
  const int token = a.t0 + (int)blockIdx.z, seq = ab_last(a.b.S, token, [&](int i) { return (int64_t)ab_start(a.b, i); });
  return seq >= 0 && token == max(ab_start(a.b, seq), a.t0) && token < ab_start(a.b, seq + 1) ? seq : -1;
}
template <int D, int KIND> __global__ __launch_bounds__(256, 2) void kw_few_kernel(kw_args a) {
  typedef kw_plan<D, KIND> P;
  __shared__ __align__(16) unsigned char rows[32 * P::ROW];
  __shared__ float2 ml[4][32];
  __shared__ __align__(16) float norms[P::PACKED ? P::N : 4];
  __shared__ kw_levels<P::PACKED ? KIND : 4> levels;
  const int part = blockIdx.x, kvh = blockIdx.y, seq = kw_few_seq(a);
  if (seq < 0) return;
  const int ctx = ab_ctx(a.b, seq);
  const int64_t from64 = (int64_t)part * P::N * a.runs;
  if (from64 >= ctx) return;
  const int from = (int)from64;
  const kw_rows R = kw_rows_of(a, seq, ctx);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, col = lane & 31;
  float unit = 1.f;
  if constexpr (P::PACKED) unit = kw_fill(levels, a.centroids);
  for (int r0 = 0; r0 < R.rows; r0 += 32) {
    const int last = R.pos0 + (min(r0 + 32, R.rows) - 1) / a.G;  // position of the tile's last row
    if (last < from) continue;
    kw_stage<D, KIND, 32> q(a, R, r0, kvh, 32);
    q.request(a, R, r0, kvh);
    __syncthreads();                   // (the tile before has been read)
    q.put(rows);
    __syncthreads();
    const bool valid = r0 + col < R.rows;
    int token, head;
    kw_row(a, R, kvh, min(r0 + col, R.rows - 1), token, head);
    const int pos = valid ? R.pos0 + token - R.first : -1;
    float c = a.scale2;
    if constexpr (P::PACKED) c = a.turned_by[kw_slab_row(a, R, kvh, min(r0 + col, R.rows - 1))];
    float* scores = a.scores + ((int64_t)(token - a.t0) * a.QH + head) * a.stride;
    float m = -INFINITY, l = 0.f;
    kw_keys<D, KIND> K;
    const int end = min(from + P::N * a.runs, last + 1);         // keys that some row sees
    int base = from + 32 * P::KT * wave;
    if (base < end) K.request(a, seq, kvh, base, ctx);
    for (; base < end; base += P::N) {
      if constexpr (P::PACKED) {
        K.decode(levels.level, unit);
        akv_wave_sync();
        if (h == 0)
#pragma unroll
          for (int t = 0; t < P::KT; ++t) norms[32 * (P::KT * wave + t) + col] = K.norm[t];
        akv_wave_sync();
      }
      ab_f16 s[P::KT];
      K.template products<true>(rows, s);
      if (base + P::N < end) K.request(a, seq, kvh, base + P::N, ctx);
      const bool edge = __ballot(base + 32 * P::KT - 1 > pos && valid) != 0;
#pragma unroll
      for (int t = 0; t < P::KT; ++t) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          float4 n = make_float4(1.f, 1.f, 1.f, 1.f);
          if constexpr (P::PACKED) n = *(const float4*)(norms + 32 * (P::KT * wave + t) + 8 * b + 4 * h);
          s[t][4 * b] *= n.x * c; s[t][4 * b + 1] *= n.y * c; s[t][4 * b + 2] *= n.z * c; s[t][4 * b + 3] *= n.w * c;
        }
        if (edge) {
#pragma unroll
          for (int i = 0; i < 16; ++i) s[t][i] = base + 32 * t + 8 * (i >> 2) + 4 * h + (i & 3) <= pos ? s[t][i] : -INFINITY;
        }
        if (valid) {
#pragma unroll
          for (int b = 0; b < 4; ++b) *(float4*)(scores + base + 32 * t + 8 * b + 4 * h) = make_float4(s[t][4 * b], s[t][4 * b + 1], s[t][4 * b + 2], s[t][4 * b + 3]);
        }
      }
      float top, sum;
      kw_row_stats<P::KT>(s, 1.f, top, sum);
      const float to = fmaxf(m, top);
      if (to > -INFINITY) {
        l = l * __builtin_amdgcn_exp2f(m - to) + sum * __builtin_amdgcn_exp2f(top - to);
        m = to;
      }
    }
    if (h == 0) ml[wave][col] = make_float2(m, l);
    __syncthreads();
    if (tid < 32 && valid) {
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, ml[w][tid].x);
#pragma unroll
      for (int w = 0; w < 4; ++w) sum += ml[w][tid].x == -INFINITY ? 0.f : ml[w][tid].y * __builtin_amdgcn_exp2f(ml[w][tid].x - top);
      a.few_part[((int64_t)(token - a.t0) * a.QH + head) * a.few_parts + part] = make_float2(top, sum);
    }
  }
}
// Weights of KW_FEW_KEYS keys from the scores that were kept; `keys` of a part of kw_few_kernel.
#define KW_FEW_KEYS 1024
__global__ __launch_bounds__(256) void kw_few_sum_kernel(kw_args a, int keys) {
  __shared__ float2 stat[KW_FEW];
  const int kvh = blockIdx.y, seq = kw_few_seq(a), tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (seq < 0) return;
  const int ctx = ab_ctx(a.b, seq);
  const int64_t key0 = (int64_t)blockIdx.x * KW_FEW_KEYS, key = key0 + 4 * tid;
  const kw_rows R = kw_rows_of(a, seq, ctx);
  float* to = a.out + (int64_t)seq * a.os_seq + (int64_t)kvh * a.os_head;
  float w[4] = {};
  for (int r0 = 0; r0 < R.rows; r0 += KW_FEW) {
    const int count = min(KW_FEW, R.rows - r0), last = R.pos0 + (r0 + count - 1) / a.G;
    if (key0 > last) continue;
    __syncthreads();                   // (the statistics before have been read)
    for (int r = wave; r < count; r += 4) {
      int token, head;
      kw_row(a, R, kvh, r0 + r, token, head);
      const float2* e = a.few_part + ((int64_t)(token - a.t0) * a.QH + head) * a.few_parts;
      float m = -INFINITY, l = 0.f;
      for (int p = lane; p <= last / keys; p += 64) {
        const float2 x = e[p];
        const float top = fmaxf(m, x.x);
        if (top == -INFINITY) continue;
        l = l * __builtin_amdgcn_exp2f(m - top) + x.y * __builtin_amdgcn_exp2f(x.x - top);
        m = top;
      }
      const float top = akv_wave_max(m);
      l = akv_wave_sum(m == -INFINITY ? 0.f : l * __builtin_amdgcn_exp2f(m - top));
      if (lane == 0) stat[r] = l > 0.f ? make_float2(top, 1.f / l) : make_float2(0.f, 0.f);
    }
    __syncthreads();
    if (key > last) continue;          // (scores are kept up to there, those behind a row's own position as -infinity)
    for (int r = 0; r < count; ++r) {
      int token, head;
      kw_row(a, R, kvh, r0 + r, token, head);
      const float4 s = *(const float4*)(a.scores + ((int64_t)(token - a.t0) * a.QH + head) * a.stride + key);
      const float m = stat[r].x, iv = stat[r].y, x[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (key + i <= last) w[i] = fmaf(__builtin_amdgcn_exp2f(x[i] - m), iv, w[i]);
    }
  }
  const int end = R.rows > 0 ? R.pos0 + (R.rows - 1) / a.G : -1;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (key + i >= a.length) continue;
    if (!a.add) to[key + i] = w[i];
    else if (key + i <= end) to[key + i] += w[i];
  }
}

// ---- launches
#define KW_SCRATCH (256ll << 20)
struct kw_scratch { int64_t tokens; size_t stat, part, turned, by, scores, few_part, sums, bytes; int parts, few_parts, runs, splits; int64_t stride; bool few; };
// Scratch of a call, its tokens in slabs of what KW_SCRATCH holds, or of one where it does not hold that (and the sums of workgroups that share a part besides, 2 MB at
// most).  Scores are kept where the batch has no more than a tile of rows a sequence and kv head on average: a key of 128 coordinates that is read again
// costs 256 bytes, the scores of 4 rows written and read 32.  (One token of 16 sequences of up to 41000 keys 135 us against 229, four tokens 197 against 243.)
// Kept scores take four bytes for every query head and place of the tables, whatever the contexts are, and every slab reads and adds anew: with fewer than KW_FEW_LEAST
// tokens a slab they are made twice.  Tables of 131072, us kept and made twice: 16 sequences of up to 40000 keys, 32 heads on 8, fifteen tokens a slab, 297 and 384 (4
// bits 232 and 395); 64 of up to 8000 870 and 644 (608 and 904); 64 heads, seven tokens a slab, 1092 and 638 (742 and 908).  In tables of 2^18 four tokens of 32
// sequences, seven a slab, 1379 and 490 (1188 and 576).
#define KW_FEW_LEAST 8
static inline kw_scratch kw_layout(int64_t T, int S, int QH, int KVH, int D, bool packed, int keys, int64_t length, bool few) {
  kw_scratch w = {};
  w.few = few;
  w.stride = (length + keys * 4 - 1) / (keys * 4) * (keys * 4);
  // runs of keys a workgroup: as many as leave forty workgroups a CU (48 sequences 509 us against 517 with one run; two sequences 25 with one against 31 with
  // four); over packed keys, whose rows have to come to LDS first, four (the last 32 tokens of four prompts 105 us then against 110, 128 tokens 342 against 353)
  w.runs = 4;
  while (w.runs > 1 && w.stride / (keys * w.runs) * S * KVH < (w.few ? 40 : 4) * ab_cus()) w.runs /= 2;
  w.few_parts = w.few ? (int)(w.stride / (keys * w.runs)) : 0;
  w.parts = w.few ? 0 : packed ? (int)((length + keys * w.runs - 1) / (keys * w.runs)) : (int)((length + keys - 1) / keys);
  // workgroups that share the rows of a part: as many as give every CU two (1024 tokens after 7000, heads of 256, 172 us against 229; after 1000, 62 against 228;
  // 4 bits, 1469 tokens of 8 heads on 2 after 3884, 184 against 616), and no more than an average sequence has steps (blocks) of rows: 30 prompts of 10 to 21
  // tokens, 64 heads on 8, 4 bits, 44 us against 61 with four
  w.splits = 1;
  const int64_t step = packed && D < 256 ? 128 : 64;
  while (!w.few && w.splits < 8 && T * (QH / KVH) > step * w.splits * S && (int64_t)w.parts * S * KVH * w.splits < 2 * ab_cus()) w.splits *= 2;
  const int64_t per = (int64_t)QH * (8 + 8 * (int64_t)w.parts + (packed ? 4 * D + 4 : 0) + (w.few ? 4 * w.stride + 8 * w.few_parts : 0));
  w.tokens = KW_SCRATCH / per;
  if (few && w.tokens < (T < KW_FEW_LEAST ? T : KW_FEW_LEAST)) return kw_layout(T, S, QH, KVH, D, packed, keys, length, false);
  if (w.tokens > 32) w.tokens = w.tokens / 32 * 32;
  if (w.tokens < 1) w.tokens = 1;
  if (w.tokens > T) w.tokens = T;
  const size_t rows = (size_t)(w.tokens * QH);
  w.stat = 0;
  w.part = akv_align256(rows * 8);
  w.turned = w.part + akv_align256(rows * 8 * w.parts);
  w.by = w.turned + (packed ? akv_align256(rows * 4 * D) : 0);
  w.scores = w.by + (packed ? akv_align256(rows * 4) : 0);
  w.few_part = w.scores + (w.few ? akv_align256(rows * 4 * w.stride) : 0);
  w.sums = w.few_part + (w.few ? akv_align256(rows * 8 * w.few_parts) : 0);
  w.bytes = w.sums + (w.splits > 1 ? akv_align256((size_t)w.splits * S * KVH * length * 4) : 0);
  return w;
}
static inline int kw_part(int D, bool packed) { return !packed && D <= 128 ? 256 : 128; }
static inline size_t kw_bytes(int64_t T, int S, int QH, int KVH, int D, bool packed, int64_t length) {
  return T <= 0 || S <= 0 || QH <= 0 || KVH <= 0 || length <= 0 || !ab_head_size(D) ? 0 : kw_layout(T, S, QH, KVH, D, packed, kw_part(D, packed), length, T * (QH / KVH) <= (int64_t)KW_FEW * S).bytes;
}
extern "C" size_t akv_key_weights_workspace_bytes(int64_t num_tokens, int num_seqs, int num_q_heads, int num_kv_heads, int d, int64_t length) { return kw_bytes(num_tokens, num_seqs, num_q_heads, num_kv_heads, d, false, length); }
extern "C" size_t akv_packed_key_weights_workspace_bytes(int64_t num_tokens, int num_seqs, int num_q_heads, int num_kv_heads, int d, int64_t length) { return kw_bytes(num_tokens, num_seqs, num_q_heads, num_kv_heads, d, true, length); }

template <int D, int KIND> static int kw_launch(kw_args a, int64_t T, void* scratch, hipStream_t stream) {
  typedef kw_plan<D, KIND> P;
  static_assert(P::N == (!P::PACKED && D <= 128 ? 256 : 128), "kw_part");
  const kw_scratch w = kw_layout(T, a.b.S, a.QH, a.KVH, D, P::PACKED, P::N, a.length, T * (a.QH / a.KVH) <= (int64_t)KW_FEW * a.b.S);
  char* const at = (char*)scratch;
  a.stat = (float2*)(at + w.stat);
  a.part = (float2*)(at + w.part);
  a.turned = (uint16_t*)(at + w.turned);
  a.turned_by = (float*)(at + w.by);
  a.scores = (float*)(at + w.scores);
  a.few_part = (float2*)(at + w.few_part);
  a.sums = (float*)(at + w.sums);
  a.splits = w.splits;
  a.parts = w.parts; a.few_parts = w.few_parts; a.stride = w.stride; a.runs = w.runs;
  a.g_recip = (uint32_t)(0xffffffffull / (uint32_t)a.G);
  int dev = 0;
  AKV_HIP(hipGetDevice(&dev));
  static akv_device_once once;
  constexpr int LDS = P::PACKED ? kw_block<D>::ROWS * P::ROW : P::LDS;
  if (const int rc = once(dev, [&]() -> int {
        const void *one, *two;
        if constexpr (P::PACKED) one = (const void*)kw_packed_stats_kernel<D, KIND>, two = (const void*)kw_packed_sum_kernel<D, KIND>;
        else one = (const void*)kw_stats_kernel<D, KIND>, two = (const void*)kw_sum_kernel<D, KIND>;
        const int rc1 = ab_lds(one, LDS);
        return rc1 ? rc1 : ab_lds(two, LDS);
      }))
    return rc;
  const int add = a.add;
  const int keys = P::PACKED ? P::N * w.runs : P::N;      // of a part
  const dim3 grid((uint32_t)((a.length + keys - 1) / keys * w.splits), (uint32_t)a.KVH, (uint32_t)a.b.S);
  int64_t t = 0;
  do {                                  // (without a token: zeros)
    a.t0 = (int)t;
    a.t1 = (int)(t + w.tokens < T ? t + w.tokens : T);
    a.add = add || t > 0;
    const int64_t rows = (int64_t)(a.t1 - a.t0) * a.QH;
    if (rows > 0) {
      if constexpr (P::PACKED) {
        const int64_t tiles = (rows + 31) / 32, most = 8 * 32 / D * ab_cus();
        const uint32_t groups = (uint32_t)(tiles < most ? tiles : most);
        if (a.dtype == AKV_F16) kw_turn_kernel<D, AKV_F16><<<groups, 2 * D, 0, stream>>>(a);
        else kw_turn_kernel<D, AKV_BF16><<<groups, 2 * D, 0, stream>>>(a);
        AKV_LAUNCH_CHECK("kw_turn_kernel");
      }
      if (w.few) {
        a.by_token = w.tokens < T && 2 * w.tokens <= a.b.S;
        kw_few_kernel<D, KIND><<<dim3((uint32_t)w.few_parts, (uint32_t)a.KVH, (uint32_t)(a.by_token ? a.t1 - a.t0 : a.b.S)), 256, 0, stream>>>(a);
        AKV_LAUNCH_CHECK("kw_few_kernel");
      } else {
        if constexpr (P::PACKED) kw_packed_stats_kernel<D, KIND><<<grid, 256, LDS, stream>>>(a);
        else kw_stats_kernel<D, KIND><<<grid, 256, LDS, stream>>>(a);
        AKV_LAUNCH_CHECK("kw_stats_kernel");
        if (w.parts > 1) {
          kw_join_kernel<<<dim3((uint32_t)(((int64_t)(a.t1 - a.t0) * a.G + 63) / 64), (uint32_t)a.KVH), 256, 0, stream>>>(a, keys);
          AKV_LAUNCH_CHECK("kw_join_kernel");
        }
      }
    }
    if (w.few) {
      a.by_token = a.by_token && a.add;          // (what is not added to is written for every sequence)
      kw_few_sum_kernel<<<dim3((uint32_t)((a.length + KW_FEW_KEYS - 1) / KW_FEW_KEYS), (uint32_t)a.KVH, (uint32_t)(a.by_token ? a.t1 - a.t0 : a.b.S)), 256, 0, stream>>>(a, P::N * w.runs);
      AKV_LAUNCH_CHECK("kw_few_sum_kernel");
    } else {
      if constexpr (P::PACKED) kw_packed_sum_kernel<D, KIND><<<grid, 256, LDS, stream>>>(a);
      else kw_sum_kernel<D, KIND><<<grid, 256, LDS, stream>>>(a);
      AKV_LAUNCH_CHECK("kw_sum_kernel");
      if (w.splits > 1) {
        kw_add_kernel<<<dim3((uint32_t)((a.length + 255) / 256), (uint32_t)a.KVH, (uint32_t)a.b.S), 256, 0, stream>>>(a);
        AKV_LAUNCH_CHECK("kw_add_kernel");
      }
    }
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
  const size_t need = kw_bytes(T, a.b.S, a.QH, a.KVH, d, packed, a.length);
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
