// Attention of a chunk of new tokens over a paged cache: arguments, and how the work of a call is cut.
//
// Sequence i brings n_i query tokens, the newest of its ctx_i tokens: token j of them stands at position ctx_i - n_i + j and sees
// the keys at its own position and before.  The query heads of a kv head meet the same keys, so the rows of a tile are (token,
// query head) pairs of one kv head, token-major, as many whole tokens as fit; their keys reach from `lo` (0, or what the window of
// the tile's first token leaves) to the position of the tile's last token.
//
// The tiles of a sequence, of all sequences, once for every kv head, lie end to end on one axis, each as long as its units (runs of
// keys) and START more, what a tile costs besides: rows, first keys, results.  Workgroup g of G takes what lies in [g F / G, (g + 1) F / G)
// of that axis.  So every workgroup has as much to do, however the lengths are spread and whatever the causal edge leaves of a tile, and
// few rows over many keys are split by themselves.  A tile that lies in one range is finished there; the pieces of one that does not go
// to memory and are joined by ck_merge_kernel in the order of the axis.  All of it is derived on the device: no call waits for a length.
#pragma once
#include "akv_attn_common.h"

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

// Sequences whose starts and lengths are held in LDS.  More are read from memory, by every workgroup's search (256 of 1 to 3 tokens after 500
// packed keys 177 us, 257 201, 1024 699).
#define CK_SEQS 256
// A sequence of at most so many rows a kv head goes to the narrow kernel.  Measured with all on it | all on the wide one, 4 rows a token, us.
// 4 bits, 32 sequences after 4000 keys: heads of 128, 24 rows 82 | 194, 64 rows 145 | 197, 68 rows 203 | 196, 128 rows 275 | 201; of 256
// 205 | 663, 384 | 681, 555 | 714, 739 | 758; of 64 49 | 94, 85 | 106, 118 | 112, 155 | 125.  One sequence after 20000: narrow at any of these.
// Plain rows, one sequence of 24 to 64 rows after 20000 keys: heads of 64 39 | 44 to 61, of 128 50 | 38 and 54 | 43, of 256 87 | 70 and
// 115 | 84; 32 sequences after 4000, where memory counts: 64 91 | 70 and 113 | 75, 128 139 | 119 and 171 | 122, 256 323 | 251 and 628 | 271:
// plain rows would gain by a lower number.
#define CK_NARROW_ROWS 64

struct ck_record {                // what a workgroup leaves of the tile that begins in its range and ends in another
  int64_t end;                    // one past the tile on the axis
  int64_t total;                  // length of the axis
  int32_t valid, head, token, tokens;      // valid: CK_LEFT_ of the kernel, 0: none
  int32_t base, count;            // the workgroups that share the axis
};
#define CK_LEFT_NARROW 1
#define CK_LEFT_WIDE 2

struct ck_args {
  const void* q; int64_t qs_tok, qs_head;        // queries, strides in elements
  const uint4 *turn_in, *turn_out;               // packed: the rotation's tables, and their scale
  const akv_prep_scale* turn_scale;
  int dtype;                                     // packed: type of queries and outputs
  const uint8_t* k; int64_t k_blk, k_pos, k_head;          // bytes
  const uint8_t* v; int64_t v_blk, v_pos, v_head;
  const float* kn; int64_t kn_blk, kn_pos, kn_head;        // packed: norms, elements
  const float* vn; int64_t vn_blk, vn_pos, vn_head;
  const float* centroids;
  const void* tables; int64_t bt_stride;
  const void* lens;
  const void* starts;
  int tables_it, lens_it, starts_it;
  void* out; int64_t os_tok, os_head;
  int kv_alike;                                  // keys and values lie alike, and so do their norms
  float* part; float2* part_ml; ck_record* rec;
  int S, T, QH, KVH, G, HS, GC;                  // G query heads a kv head, in HS groups of GC
  int block_size; uint32_t bs_recip;
  int64_t max_blocks, num_blocks;
  int window;                                    // 0: none; at most 2^30, as far as a position may lie below 0: their difference has 32 bits
  int kind;                                      // sequences of this launch: 0 all, 1 those of few rows, 2 the others
  int tail;                                      // rows of no sequence, behind the last or before the first, are zeroed
  float scale2;                                  // score scale x log2 e
};

struct ck_seq { int q0, n, ctx; };               // first query row, query tokens, tokens

template <int THREADS> struct ck_lengths {       // starts and lengths of the batch
  alignas(8) int start[CK_SEQS + 1];
  int ctx[CK_SEQS];
  int64_t sum[THREADS / 64];
  int64_t total;
  int found[2];
};

__device__ __forceinline__ int ck_clamp(int64_t v, int64_t hi) { return (int)(v < 0 ? 0 : v > hi ? hi : v); }
__device__ __forceinline__ int ck_start_of(const ck_args& a, int i) { return ck_clamp(akv_load_index(a.starts, a.starts_it, i), a.T); }
__device__ __forceinline__ int ck_ctx_of(const ck_args& a, int i) {
  const int64_t cap = a.max_blocks * a.block_size;
  return ck_clamp(akv_load_index(a.lens, a.lens_it, i), cap < 0x7fff0000 ? cap : 0x7fff0000);
}

template <int THREADS> __device__ __forceinline__ void ck_load_lengths(const ck_args& a, ck_lengths<THREADS>& L) {
  if (a.S <= CK_SEQS) {
    for (int i = threadIdx.x; i <= a.S; i += THREADS) L.start[i] = ck_start_of(a, i);
    for (int i = threadIdx.x; i < a.S; i += THREADS) L.ctx[i] = ck_ctx_of(a, i);
  }
  __syncthreads();
}

// Sequence i; i == S: the rows behind the last one, which see nothing.
template <int THREADS> __device__ __forceinline__ ck_seq ck_sequence(const ck_args& a, const ck_lengths<THREADS>& L, int i) {
  const bool held = a.S <= CK_SEQS;
  ck_seq s;
  s.q0 = held ? L.start[i] : ck_start_of(a, i);
  if (i == a.S) {
    s.n = a.tail && a.kind != 2 ? a.T - s.q0 : 0;
    s.ctx = 0;
    return s;
  }
  const int q1 = held ? L.start[i + 1] : ck_start_of(a, i + 1);
  s.n = q1 > s.q0 ? q1 - s.q0 : 0;
  s.ctx = held ? L.ctx[i] : ck_ctx_of(a, i);
  if (a.kind != 0 && ((int64_t)s.n * a.G <= CK_NARROW_ROWS) != (a.kind == 1)) s.n = 0;
  return s;
}

// keys [lo, hi) that rows of tile j see, TM tokens a tile; a tile has at least one unit of N keys
struct ck_range { int first, units, lo, hi; };
template <int N> __device__ __forceinline__ ck_range ck_keys(const ck_args& a, const ck_seq& s, int j, int TM) {
  const int t0 = j * TM, t1 = t0 + TM < s.n ? t0 + TM : s.n;
  ck_range r;
  r.hi = s.ctx - s.n + t1;
  if (r.hi < 0) r.hi = 0;
  r.lo = 0;
  if (a.window > 0) {
    r.lo = s.ctx - s.n + t0 - a.window + 1;
    if (r.lo < 0) r.lo = 0;
  }
  r.first = r.lo / N;
  r.units = (r.hi + N - 1) / N - r.first;
  if (r.units < 1) r.units = 1;
  return r;
}

// Tiles are numbered with gaps: tile j of sequence i is floor(start_i / TM) + i + j, which no two tiles share.  (Where starts go back some do,
// and the axis has a part of the tiles: whatever a workgroup finds there is a tile of a sequence, and its way from one to the next ends
// with the last sequence.)
__device__ __forceinline__ int ck_tile_numbers(const ck_args& a, int TM) { return a.T / TM + a.S + 1; }
template <int THREADS, int N, int START>
__device__ __forceinline__ int ck_units_of(const ck_args& a, const ck_lengths<THREADS>& L, int x, int TM, int& seq, int& tile) {
  int lo = 0, hi = a.S + 1;                 // the last i with floor(start_i / TM) + i <= x
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    const int s = a.S <= CK_SEQS ? L.start[mid] : ck_start_of(a, mid);
    if (s / TM + mid <= x) lo = mid; else hi = mid;
  }
  const ck_seq s = ck_sequence(a, L, lo);
  seq = lo;
  tile = x - (s.q0 / TM + lo);
  if (tile < 0 || (int64_t)tile * TM >= s.n) return 0;
  return ck_keys<N>(a, s, tile, TM).units + START;
}

// The axis may pass 2^31 (a chunk of a million tokens, few of them a tile, is a million tiles over up to a million tokens): places on it
// have 64 bits.  A tile is at most (2^31 - 2^16) / 32 units long, so that those of a wavefront fit 32 bits together.
__device__ __forceinline__ uint32_t ck_wave_scan(int v) { return (uint32_t)akv_wave_inclusive_scan(v); }
__device__ __forceinline__ int64_t ck_readfirst(int64_t v) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

// length of one kv head's part of the axis, in every thread
template <int THREADS, int N, int START> __device__ __forceinline__ int64_t ck_total(const ck_args& a, ck_lengths<THREADS>& L, int TM) {
  static_assert(N >= 32 && 64ll * (0x7fff0000ll / N + 1 + START) <= 0xffffffffll, "the tiles of a wavefront fit 32 bits");
  int64_t sum = 0;
  int seq, tile;
  const int numbers = ck_tile_numbers(a, TM);
  for (int x0 = 0; x0 < numbers; x0 += THREADS) {
    const int x = x0 + (int)threadIdx.x, u = x < numbers ? ck_units_of<THREADS, N, START>(a, L, x, TM, seq, tile) : 0;
    sum += (uint32_t)akv_wave_sum(u);
  }
  if ((threadIdx.x & 63) == 0) L.sum[threadIdx.x >> 6] = sum;
  __syncthreads();
  int64_t all = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) all += L.sum[w];
  __syncthreads();
  return all;
}

// the tile that holds `at` (< total): its sequence, number and place on the axis
template <int THREADS, int N, int START>
__device__ __forceinline__ void ck_find(const ck_args& a, ck_lengths<THREADS>& L, int TM, int64_t at, int& seq, int& tile, int64_t& first) {
  const int numbers = ck_tile_numbers(a, TM);
  int64_t base = 0;
  for (int x0 = 0;; x0 += THREADS) {
    const int x = x0 + (int)threadIdx.x;
    int sq = 0, tl = 0;
    const int u = x < numbers ? ck_units_of<THREADS, N, START>(a, L, x, TM, sq, tl) : 0;
    const uint32_t inc = ck_wave_scan(u);
    if ((threadIdx.x & 63) == 63) L.sum[threadIdx.x >> 6] = inc;
    __syncthreads();
    int64_t before = base, all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
      const int64_t s = L.sum[w];
      if (w < (int)(threadIdx.x >> 6)) before += s;
      all += s;
    }
    const int64_t b = before + inc - u;
    if (u > 0 && at >= b && at < b + u) {
      L.found[0] = sq;
      L.found[1] = tl;
      L.total = b;
    }
    __syncthreads();
    base += all;
    if (at < base || x0 + THREADS >= numbers) break;      // (the second never before the first: at < total)
  }
  seq = __builtin_amdgcn_readfirstlane(L.found[0]);
  tile = __builtin_amdgcn_readfirstlane(L.found[1]);
  first = ck_readfirst(L.total);
}

// Rows before the first sequence, by all workgroups: zeros.  (Those behind the last one are a sequence of no keys; these are as many as a caller
// who takes a part of a batch leaves.)
template <int THREADS> __device__ __forceinline__ void ck_clear_front(const ck_args& a, const ck_lengths<THREADS>& L, int D) {
  const int rows = !a.tail ? 0 : a.S <= CK_SEQS ? L.start[0] : ck_start_of(a, 0);
  if (rows == 0) return;
  const int per = a.QH * (D / 4);
  for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < (int64_t)rows * per; i += (int64_t)gridDim.x * THREADS) {
    const int64_t token = i / per;
    const int rest = (int)(i - token * per), head = rest / (D / 4);
    *(ck_u2*)((uint16_t*)a.out + token * a.os_tok + (int64_t)head * a.os_head + 4 * (rest - head * (D / 4))) = (ck_u2){0u, 0u};
  }
}

// where workgroup g's range begins: floor(total g / G), G at most 2^15
struct ck_share { int64_t whole; uint32_t rest; };
__device__ __forceinline__ ck_share ck_share_of(int64_t total, int G) {
  if (total <= 0xffffffffll) {
    const uint32_t w = (uint32_t)total / (uint32_t)G;
    return {(int64_t)w, (uint32_t)total - w * (uint32_t)G};
  }
  const int64_t w = total / G;
  return {w, (uint32_t)(total - w * G)};
}
__device__ __forceinline__ int64_t ck_begin(const ck_share& s, int g, int G) { return s.whole * g + s.rest * (uint32_t)g / (uint32_t)G; }
