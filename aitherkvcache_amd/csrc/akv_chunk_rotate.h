// Rotations of a chunk's rows inside the kernels that attend: queries on the way in, results on the way out.
//
//   Y^T[n, row] = sum_k M[n, k] X[row, k]            v_mfma_f32_32x32x16_f16, A = 32 rows of the matrix, B = 32 rows of X
//
// The matrix (Pi for queries, Pi^T for results) is prepared as two float16 terms of its entries times 1024 (22 bits), in the order of
// the operand: [hi, lo][n / 32][k / 16][64 lanes] sixteen bytes.  float16 queries are operands as they are; bfloat16 ones are scaled by
// a power of two a row, which keeps what lies within 2^14 of the largest exact.  Results are scaled alike and split into two terms.
// Per tile of 32 rows a rotation takes 2 (3 for results) x 32 products at head_dim 128, some 1 (1.5) us of a wavefront; kernels of their own
// before and after took 6 + 6 us for small calls and 39 + 51 us for 65,000 rows, and the float32 rows between them.
#pragma once
#include "akv_chunk.h"

#define CK_TURN 1024.f
// k of element j of a lane of half h in a step of sixteen: queries 8 h + j; results in the order in which the second product of attention
// leaves them, 4 h + j and 8 + 4 h + j - 4
__host__ __device__ constexpr int ck_result_k(int h, int j) { return 4 * h + (j & 3) + 8 * (j >> 2); }
// (a pointer the compiler knows nothing of: it would keep the whole table in registers from one tile for the next; but one to device memory: reads
// of LDS would wait for a generic one)
typedef const __attribute__((address_space(1))) ck_u4* ck_table;
__device__ __forceinline__ ck_table ck_turn_table(const uint4* table) {
  ck_table t = (ck_table)(uintptr_t)table;
  asm volatile("" : "+s"(t));
  return t;
}
__device__ __forceinline__ ck_u4 ck_turn_at(ck_table table, int D, int term, int dt, int ks) {
  return table[(((size_t)term * (D / 32) + dt) * (D / 16) + ks) * 64 + (threadIdx.x & 63)];
}
// Rows dt of M times rows held as operands: one term (queries) ...  Four steps of the table are requested together, no more (registers) and no
// less: left to the scheduler one to three requests were on their way, as it counted registers (3 bits, heads of 256, 8 drafts of four tokens
// after 3000 to 9000: 95 to 112 us from build to build, 85 now; 16 drafts at heads of 128 162 and 152 us).
template <int D> __device__ __forceinline__ ck_f16v ck_turn(const uint4* __restrict__ all, int dt, const ck_u4 (&x)[D / 16]) {
  const ck_table table = ck_turn_table(all);
  ck_f16v y = (ck_f16v)(0.f);
#pragma unroll
  for (int k0 = 0; k0 < D / 16; k0 += 4) {
    ck_u4 lo[4], hi[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { lo[i] = ck_turn_at(table, D, 1, dt, k0 + i); hi[i] = ck_turn_at(table, D, 0, dt, k0 + i); }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y = ck_math<CK_F16>::mfma(lo[i], x[k0 + i], y);
      y = ck_math<CK_F16>::mfma(hi[i], x[k0 + i], y);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  return y;
}
// ... or two (results)
template <int D> __device__ __forceinline__ ck_f16v ck_turn(const uint4* __restrict__ all, int dt, const ck_u4 (&x)[D / 16], const ck_u4 (&xl)[D / 16]) {
  const ck_table table = ck_turn_table(all);
  ck_f16v y = (ck_f16v)(0.f);
#pragma unroll
  for (int k0 = 0; k0 < D / 16; k0 += 4) {
    ck_u4 lo[4], hi[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { lo[i] = ck_turn_at(table, D, 1, dt, k0 + i); hi[i] = ck_turn_at(table, D, 0, dt, k0 + i); }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y = ck_math<CK_F16>::mfma(lo[i], x[k0 + i], y);
      y = ck_math<CK_F16>::mfma(hi[i], xl[k0 + i], y);
      y = ck_math<CK_F16>::mfma(hi[i], x[k0 + i], y);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  return y;
}
// Rows dt of the matrix for results: read where they are multiplied, or (HELD: D at most 128, a workgroup of four wavefronts with one dt each)
// requested before the results are there.
template <int D, bool HELD> struct ck_turn_rows {
  const uint4* all;
  ck_u4 x[HELD ? 2 * (D / 16) : 1];
  __device__ __forceinline__ ck_turn_rows(const uint4* table, int dt) : all(table) {
    if constexpr (HELD) {
      if (dt < D / 32) {
#pragma unroll
        for (int i = 0; i < 2 * (D / 16); ++i) x[i] = ck_turn_at((ck_table)(uintptr_t)table, D, i & 1, dt, i >> 1);
      }
    }
  }
  __device__ __forceinline__ ck_f16v turn(int dt, const ck_u4 (&hi)[D / 16], const ck_u4 (&lo)[D / 16]) const {
    if constexpr (!HELD) return ck_turn<D>(all, dt, hi, lo);
    ck_f16v y = (ck_f16v)(0.f);
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const ck_u4 m_hi = x[HELD ? 2 * ks : 0], m_lo = x[HELD ? 2 * ks + 1 : 0];
      y = ck_math<CK_F16>::mfma(m_lo, hi[ks], y);
      y = ck_math<CK_F16>::mfma(m_hi, lo[ks], y);
      y = ck_math<CK_F16>::mfma(m_hi, hi[ks], y);
    }
    return y;
  }
};
// A row of queries (this lane's half of every sixteen coordinates) as operand; returns what undoes its scale.
template <int D> __device__ __forceinline__ float ck_query_operand(ck_u4 (&x)[D / 16], int dtype) {
  if (dtype == AKV_F16) return 1.f;
  uint32_t m = 0u;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, max((x[ks][i] << 16) & 0x7fff0000u, x[ks][i] & 0x7fff0000u));
  m = max(m, akv_lane_xor_u32<32>(m));
  const uint32_t e = akv_row_exponent(__uint_as_float(m));
  const float sc = akv_row_scale(e);
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
    for (int i = 0; i < 4; ++i) x[ks][i] = ck_math<CK_F16>::pair(__uint_as_float(x[ks][i] << 16) * sc, __uint_as_float(x[ks][i] & 0xffff0000u) * sc);
  return akv_row_unscale(e);
}
// Scale of turned queries, by the row's largest: the usual sizes go as they are, times `f`, and need no factor later; others are brought to
// [1, 2), and `later` is what their scores are multiplied with.
__device__ __forceinline__ float ck_query_scale(float largest, float f, float& later) {
  const float m = largest * f;
  if (m >= 0x1p-8f && m <= 0x1p12f) {
    later = 1.f;
    return f;
  }
  const uint32_t e = akv_row_exponent(largest);
  later = akv_row_unscale(e) * f;
  return akv_row_scale(e);
}
// results of a row, times `f`, as two operands; returns what undoes their scale
template <int D, class Get> __device__ __forceinline__ float ck_result_operand(Get get, ck_u4 (&hi)[D / 16], ck_u4 (&lo)[D / 16]) {
  float m = 0.f;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(get(ks, j)));
  m = fmaxf(m, akv_lane_xor<32>(m));
  const uint32_t e = akv_row_exponent(m);
  const float sc = akv_row_scale(e);
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = get(ks, 2 * i) * sc, y = get(ks, 2 * i + 1) * sc;
      hi[ks][i] = ck_math<CK_F16>::pair(x, y);
      typedef _Float16 h2 __attribute__((ext_vector_type(2)));
      const h2 h = __builtin_bit_cast(h2, (uint32_t)hi[ks][i]);
      lo[ks][i] = ck_math<CK_F16>::pair(x - (float)h[0], y - (float)h[1]);
    }
  return akv_row_unscale(e);
}
