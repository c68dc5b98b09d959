// Rotations of a chunk's queries and outputs for attention over packed rows.
#pragma once
#include "akv_chunk_kernels.h"
#include "akv_attn_rows.h"

// ---- packed: rotations of queries and outputs ---------------------------------------------------------------------------------
// Rows of `in` (any strides) times the matrix, 16 rows a step; workgroup (b, slice): 64 outputs.  IN_PLACES: the row's coordinates lie in
// the order of the packed groups.
template <int D, int XDT, int BITS, bool QUERY, int ODT>
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
      int d = 64 * (i >> 2) + 4 * part + (i & 3);
      if constexpr (!QUERY) d = (d & ~7) + ck_coord<BITS>(d & 7);
#pragma unroll
      for (int j = 0; j < TERMS; ++j) {
        const _Float16 t = (_Float16)(j == 2 ? v * AR_THIRD : v);
        r.term[j][row][d] = t;
        v -= (float)t;
      }
    }
    if (part == 0) {
      r.unscale[row] = un;
      if (QUERY && slice == 0 && n < rows) fac[n] = un * AR_M_SCALE * qscale;
    }
    __syncthreads();
    const ar_float4 y = m.times(r);
    const int rr = lane & 15, d0 = n0 + 4 * (lane >> 4);
    const int64_t no = tile * 16 + rr;
    if (no < limit) {
      if constexpr (QUERY) {
        uint16_t* dst = (uint16_t*)out + no * D + (d0 & ~7);
#pragma unroll
        for (int e = 0; e < 4; ++e) dst[ck_place<BITS>((d0 & 7) + e)] = __builtin_bit_cast(unsigned short, (_Float16)(y[e] * (1.f / AR_M_SCALE)));
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
