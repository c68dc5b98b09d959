// Rotations of a chunk's queries and outputs for attention over packed rows.
#pragma once
#include "akv_chunk_kernels.h"
#include "akv_attn_rows.h"

// ---- packed: rotations of queries and outputs ---------------------------------------------------------------------------------
// Rows of `in` (any strides) times the matrix, 16 rows a step; workgroup (b, slice): 64 outputs.  QUERY: to float16, times the scale of the
// scores and log2 e; `fac` is what a row has to be multiplied with still, 1 unless its largest coordinate is far from 1 (then the row
// is stored with that between 2^5 and 2^6).
template <int D, int XDT, bool QUERY, int ODT>
__global__ __launch_bounds__(256) void ck_rotate_kernel(const void* __restrict__ in, int64_t is_tok, int64_t is_head, int64_t rows, int QH,
                                                        const float* __restrict__ matrix, const akv_prep_scale* __restrict__ scale,
                                                        void* __restrict__ out, int64_t os_tok, int64_t os_head, float* __restrict__ fac, float qscale,
                                                        const void* __restrict__ starts, int starts_it, int S, int tail) {
  constexpr int TERMS = ar_terms<XDT>(), EPT = D / 16;
  __shared__ ar_rows<D, TERMS> r;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, slice = blockIdx.y, n0 = 64 * slice + 16 * wave;
  const int row = tid >> 4, part = tid & 15;
  ar_matrix<D> m;
  m.load(matrix + (size_t)n0 * D, AR_M_SCALE * scale->down);
  const float up = scale->up;
  int64_t limit = rows;                 // rows behind the last sequence are left as they were
  if (!QUERY && !tail) {
    const int64_t last = akv_load_index(starts, starts_it, S) * QH;
    limit = last < 0 ? 0 : last < rows ? last : rows;
  }
  for (int64_t tile = blockIdx.x; tile * 16 < rows; tile += gridDim.x) {
    const int64_t n = tile * 16 + row;
    float x[EPT];
    const int64_t tok = n / QH, at = tok * is_tok + (n - tok * QH) * is_head;
    float mx = 0.f;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      x[i] = n < rows ? akv_elem<XDT>::load(in, at + 64 * (i >> 2) + 4 * part + (i & 3)) : 0.f;
      mx = fmaxf(mx, fabsf(x[i]));
    }
    mx = fmaxf(mx, akv_lane_xor<1>(mx)); mx = fmaxf(mx, akv_lane_xor<2>(mx));
    mx = fmaxf(mx, akv_lane_xor<4>(mx)); mx = fmaxf(mx, akv_lane_xor<8>(mx));
    float un;
    const float sc = ar_scale(mx, un);
    un *= up;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      float v = x[i] * sc;
      const int d = 64 * (i >> 2) + 4 * part + (i & 3);
#pragma unroll
      for (int j = 0; j < TERMS; ++j) {
        const _Float16 t = (_Float16)(j == 2 ? v * AR_THIRD : v);
        r.term[j][row][d] = t;
        v -= (float)t;
      }
    }
    if (part == 0) {
      // queries: the usual sizes go as they are (the factor is in the row), the others scaled
      const bool usual = mx * qscale >= 0x1p-8f && mx * qscale <= 0x1p8f;
      r.unscale[row] = !QUERY ? un : usual ? un * qscale : 1.f / AR_M_SCALE;
      if (QUERY && slice == 0 && n < rows) fac[n] = usual ? 1.f : un * AR_M_SCALE * qscale;
    }
    __syncthreads();
    const ar_float4 y = m.times(r);
    const int rr = lane & 15, d0 = n0 + 4 * (lane >> 4);
    const int64_t no = tile * 16 + rr;
    if (no < limit) {
      if constexpr (QUERY) {
        const float f = r.unscale[rr];
        ck_u2 v;
        v[0] = ck_math<CK_F16>::pair(y[0] * f, y[1] * f);
        v[1] = ck_math<CK_F16>::pair(y[2] * f, y[3] * f);
        *(ck_u2*)((uint16_t*)out + no * D + d0) = v;
      } else {
        const float f = r.unscale[rr];
        const int64_t t = no / QH, o = t * os_tok + (no - t * QH) * os_head + d0;
#pragma unroll
        for (int e = 0; e < 4; ++e) akv_elem<ODT>::store(out, o + e, y[e] * f);
      }
    }
    __syncthreads();
  }
}
