// A batch of sequences over a paged cache, as the kernels read and write a part of a long context see it (akv_block_index.hip,
// akv_sparse_attn.hip, akv_key_weights.hip, akv_evict.hip).
//
// Sequence i owns query rows [start_i, start_{i+1}), the newest n_i of its ctx_i tokens: token j of them stands at position ctx_i - n_i + j.
// Everything is read on the device, and clamped: starts into [0, T], lengths to what the tables hold, table entries into the cache.
#pragma once
#include "akv_attn_common.h"

typedef _Float16 ab_half8 __attribute__((ext_vector_type(8)));
typedef __bf16 ab_bf8 __attribute__((ext_vector_type(8)));
typedef float ab_f4 __attribute__((ext_vector_type(4)));
typedef float ab_f16 __attribute__((ext_vector_type(16)));
typedef uint32_t ab_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t ab_u2 __attribute__((ext_vector_type(2)));
typedef int ab_i4 __attribute__((ext_vector_type(4)));

struct ab_batch {
  const void *tables, *lens, *starts;
  int tables_it, lens_it, starts_it;
  int64_t bt_stride;
  int S, T, block_size;
  uint32_t bs_recip;
  int64_t max_blocks, num_blocks;
};

#define AB_MOST_TOKENS 0x7fff0000ll
__device__ __forceinline__ int ab_clamp(int64_t v, int64_t hi) { return (int)(v < 0 ? 0 : v > hi ? hi : v); }
__device__ __forceinline__ int ab_start(const ab_batch& b, int i) { return ab_clamp(akv_load_index(b.starts, b.starts_it, i), b.T); }
__device__ __forceinline__ int ab_ctx(const ab_batch& b, int i) {
  const int64_t cap = b.max_blocks * b.block_size;
  return ab_clamp(akv_load_index(b.lens, b.lens_it, i), cap < AB_MOST_TOKENS ? cap : AB_MOST_TOKENS);
}
// A table entry as it is requested (both words of a 64-bit one), and the cache block from it.  (Taken apart, and without a branch, so that
// several are on their way together.)
struct ab_entry { uint32_t lo, hi; };
__device__ __forceinline__ ab_entry ab_look(const ab_batch& b, int seq, int64_t col) {
  const int wide = b.tables_it == AKV_I64;
  const uint32_t* p = (const uint32_t*)b.tables + (((int64_t)seq * b.bt_stride + col) << wide);
  return {p[0], p[wide]};
}
__device__ __forceinline__ int64_t ab_block(const ab_batch& b, ab_entry e) {
  const int64_t id = b.tables_it == AKV_I64 ? (int64_t)((uint64_t)e.hi << 32 | e.lo) : (int64_t)(int32_t)e.lo;
  return akv_clamp_block(id, b.num_blocks);
}
// cache block of table column `col` (below max_blocks) of sequence `seq`
__device__ __forceinline__ int64_t ab_block(const ab_batch& b, int seq, int64_t col) { return ab_block(b, ab_look(b, seq, col)); }
// the last i in [0, S) with number(i) <= x, for numbers that do not decrease; the same in all lanes (-1: none)
template <class Number> __device__ __forceinline__ int ab_last(int S, int64_t x, Number number) {
  const int lane = threadIdx.x & 63;
  int found = 0;
  for (int i = 0; i < S; i += 64) {
    const uint64_t there = __ballot(i + lane < S && number(i + lane) <= x);
    found += __popcll(there);
    if (there != ~0ull) break;
  }
  return found - 1;
}

template <int DT> struct ab_math {
  static __device__ __forceinline__ ab_f16 mfma32(ab_u4 a, ab_u4 b, ab_f16 c) {
    if constexpr (DT == AKV_BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(ab_bf8, a), __builtin_bit_cast(ab_bf8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(ab_half8, a), __builtin_bit_cast(ab_half8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ ab_f4 mfma16(ab_u4 a, ab_u4 b, ab_f4 c) {
    if constexpr (DT == AKV_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(ab_bf8, a), __builtin_bit_cast(ab_bf8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ab_half8, a), __builtin_bit_cast(ab_half8, b), c, 0, 0, 0);
  }
  // two numbers rounded to the type, to nearest
  static __device__ __forceinline__ uint32_t pair(float x, float y) {
    if constexpr (DT == AKV_BF16) {
      typedef __bf16 b2 __attribute__((ext_vector_type(2)));
      b2 r = {(__bf16)x, (__bf16)y};
      return __builtin_bit_cast(uint32_t, r);
    } else {
      typedef _Float16 h2 __attribute__((ext_vector_type(2)));
      h2 r = {(_Float16)x, (_Float16)y};
      return __builtin_bit_cast(uint32_t, r);
    }
  }
  static __device__ __forceinline__ float low(uint32_t v) {
    if constexpr (DT == AKV_BF16) return __uint_as_float(v << 16);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)v);
  }
  static __device__ __forceinline__ float high(uint32_t v) {
    if constexpr (DT == AKV_BF16) return __uint_as_float(v & 0xffff0000u);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)(v >> 16));
  }
};

// ---- host ---------------------------------------------------------------------------------------------------------------------------
static inline bool ab_aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
static inline ab_batch ab_make(const void* tables, int tables_it, int64_t bt_stride, const void* lens, int lens_it, const void* starts, int starts_it, int S, int64_t T,
                               int block_size, int64_t num_blocks, int64_t max_blocks) {
  ab_batch b = {};
  b.tables = tables; b.tables_it = tables_it; b.bt_stride = bt_stride;
  b.lens = lens; b.lens_it = lens_it; b.starts = starts; b.starts_it = starts_it;
  b.S = S; b.T = (int)T; b.block_size = block_size;
  b.bs_recip = (uint32_t)(0xffffffffull / (uint32_t)block_size);
  b.max_blocks = num_blocks > 0 ? max_blocks : 0; b.num_blocks = num_blocks;
  return b;
}
// what every entry point asks of its batch
static inline int ab_check(const char* name, const void* tables, int tables_it, const void* lens, int lens_it, const void* starts, int starts_it, int S, int64_t T, int heads,
                           int block_size, int64_t num_blocks, int64_t max_blocks) {
  AKV_REQUIRE(akv_valid_itype(tables_it) && akv_valid_itype(lens_it) && akv_valid_itype(starts_it), "%s: bad index type", name);
  AKV_REQUIRE(S >= 0 && T >= 0 && heads > 0, "%s: %d sequences, %lld tokens, %d kv heads", name, S, (long long)T, heads);
  AKV_REQUIRE(block_size > 0 && num_blocks >= 0 && max_blocks >= 0, "%s: bad block_size %d, num_blocks %lld or max_blocks_per_seq %lld", name, block_size, (long long)num_blocks, (long long)max_blocks);
  AKV_REQUIRE(S == 0 || lens, "%s: null pointer", name);
  AKV_REQUIRE(S == 0 || max_blocks == 0 || num_blocks == 0 || tables, "%s: null pointer", name);
  if (num_blocks > 0x7fffffff || max_blocks > 0x7fffffff) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: more than 2^31 blocks", name);
  if (T > 0x3fffffff || S > 0x3fffff) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: more than 2^30 tokens or 2^22 sequences", name);
  return AKV_OK;
}
static inline bool ab_head_size(int d) { return d == 64 || d == 128 || d == 256; }
static inline int ab_cus() {
  const int cus = akv_cached_cu_count();
  return cus > 0 ? cus : 256;
}
static inline int ab_lds(const void* kernel, int bytes) {
  AKV_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  return AKV_OK;
}
