// akv_rope_append: queries and keys turned by their positions, keys and values appended to a paged cache of plain rows.
//
//   y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin        for the pairs p < R / 2 of a row's first R coordinates
//
// Partners are p and p + R / 2, or 2 p and 2 p + 1; cos and sin of pair p stand in row positions[axis(p)][token] of a table, axes taking
// runs of pairs.  Every value is read once and written once, and 32-bit arithmetic ends in one rounding to the type it is stored
// in, so memory bounds it: a thread takes a unit of sixteen coordinates of a row, eight pairs or sixteen that do not turn, in
// pieces of eight (16 bytes); units of the token's other rows find the table's row in the first-level cache.  Where the axes take whole units a
// unit has one position and reads the table in wide loads (with a position looked up for every pair 4097 tokens of three axes took 40 us).
// 8192 tokens of 48 rows of 128 in bfloat16, 206 MB: 43.0 us, 4.8 TB/s, where the inputs come from memory (a large copy reaches 5.2), 33.8 where
// the last-level cache holds them from the call before; one token 4.7 us, the host's time.
#include "akv_common.h"

#define RP_AXES 4

struct rp_rows { const void* x; int64_t s_tok, s_head; };
struct rp_args {
  rp_rows q, k, v;
  void* q_out; int64_t qo_tok, qo_head;
  void* kc; int64_t kc_blk, kc_pos, kc_head;
  void* vc; int64_t vc_blk, vc_pos, vc_head;
  const void* positions; int64_t pos_axis; int pos_it;
  const float* table; int64_t table_rows;
  const void* slots; int slots_it;
  int64_t slots_end;                  // block_size x blocks: slots beyond are skipped
  int64_t units;                      // tokens x rows x D / 16
  uint32_t per_token, per_row;        // units of a token, of a row
  int QH, KVH, R, block_size, axes, interleaved;
  int whole;                          // every axis takes whole units
  int ends[RP_AXES];                  // one past the last pair of each axis
};

// eight elements as floats, from memory and to it; VEC: 16-byte accesses
template <int DT, bool VEC> __device__ __forceinline__ void rp_load(const void* __restrict__ p, int64_t i, float (&x)[8]) {
  if constexpr (VEC && DT == AKV_F32) {
    const float4* q = (const float4*)((const float*)p + i);
    const float4 a = q[0], b = q[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else if constexpr (VEC) {
    const uint4 a = *(const uint4*)((const uint16_t*)p + i);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint16_t b = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
      x[e] = DT == AKV_BF16 ? akv_bf16_bits_to_float(b) : __half2float(__ushort_as_half(b));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = akv_elem<DT>::load(p, i + e);
  }
}
typedef uint32_t rp_u4 __attribute__((ext_vector_type(4)));
typedef float rp_f4 __attribute__((ext_vector_type(4)));
// sixteen bytes; PAST: past the caches
template <bool PAST, class T> __device__ __forceinline__ void rp_put(void* p, T v) {
  if constexpr (PAST) __builtin_nontemporal_store(v, (T*)p);
  else *(T*)p = v;
}
template <int DT> __device__ __forceinline__ uint16_t rp_bits(float v) {
  if constexpr (DT == AKV_BF16) return __builtin_bit_cast(unsigned short, (__bf16)v);
  else return __half_as_ushort(__float2half_rn(v));
}
template <int DT, bool VEC, bool PAST> __device__ __forceinline__ void rp_store(void* __restrict__ p, int64_t i, const float (&x)[8]) {
  if constexpr (VEC && DT == AKV_F32) {
    rp_put<PAST>((float*)p + i, (rp_f4){x[0], x[1], x[2], x[3]});
    rp_put<PAST>((float*)p + i + 4, (rp_f4){x[4], x[5], x[6], x[7]});
  } else if constexpr (VEC) {
    rp_u4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = (uint32_t)rp_bits<DT>(x[2 * e]) | (uint32_t)rp_bits<DT>(x[2 * e + 1]) << 16;
    rp_put<PAST>((uint16_t*)p + i, w);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) akv_elem<DT>::store(p, i + e, x[e]);
  }
}

template <int XDT, int CDT, bool VEC, bool PAST>
__global__ __launch_bounds__(256) void rp_kernel(rp_args a) {
  for (int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x; n < a.units; n += (int64_t)gridDim.x * 256) {
    int64_t tok;
    uint32_t rest;
    if (a.units <= 0xffffffffll) {
      tok = (uint32_t)n / a.per_token;
      rest = (uint32_t)n - (uint32_t)tok * a.per_token;
    } else {
      tok = n / a.per_token;
      rest = (uint32_t)(n - tok * a.per_token);
    }
    const int row = (int)(rest / a.per_row), unit = (int)(rest - (uint32_t)row * a.per_row);
    const bool is_q = row < a.QH, is_k = !is_q && row < a.QH + a.KVH;
    const rp_rows src = is_q ? a.q : is_k ? a.k : a.v;
    const int head = is_q ? row : is_k ? row - a.QH : row - a.QH - a.KVH;
    const int half = a.R / 2, p0 = 8 * unit;
    const bool turns = (is_q || is_k) && p0 < half;
    const int d0 = turns && !a.interleaved ? p0 : 16 * unit, d1 = turns && !a.interleaved ? half + p0 : 16 * unit + 8;
    // the destination first: a token without one is not read
    int64_t dst;
    if (is_q) {
      dst = tok * a.qo_tok + head * a.qo_head;
    } else {
      const int64_t slot = akv_load_index(a.slots, a.slots_it, tok);
      if (slot < 0 || slot >= a.slots_end) continue;
      int64_t blk, pos;
      if (slot <= 0x7fffffff) {
        const uint32_t b = (uint32_t)slot / (uint32_t)a.block_size;
        blk = b;
        pos = (uint32_t)slot - b * (uint32_t)a.block_size;
      } else {
        blk = slot / a.block_size;
        pos = slot - blk * a.block_size;
      }
      dst = is_k ? blk * a.kc_blk + pos * a.kc_pos + head * a.kc_head : blk * a.vc_blk + pos * a.vc_pos + head * a.vc_head;
    }
    const int64_t at = tok * src.s_tok + head * src.s_head;
    float x[8], y[8];
    rp_load<XDT, VEC>(src.x, at + d0, x);
    rp_load<XDT, VEC>(src.x, at + d1, y);
    if (turns) {
      float c[8], s[8];
      if (a.whole) {
        int ax = 0;
#pragma unroll
        for (int i = 0; i + 1 < RP_AXES; ++i) ax += i + 1 < a.axes && p0 >= a.ends[i] ? 1 : 0;
        int64_t pos = akv_load_index(a.positions, a.pos_it, ax * a.pos_axis + tok);
        pos = pos < 0 ? 0 : pos >= a.table_rows ? a.table_rows - 1 : pos;
        const float* t = a.table + pos * a.R + p0;
        rp_load<AKV_F32, true>(t, 0, c);
        rp_load<AKV_F32, true>(t, half, s);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          int ax = 0;
#pragma unroll
          for (int i = 0; i + 1 < RP_AXES; ++i) ax += i + 1 < a.axes && p0 + e >= a.ends[i] ? 1 : 0;
          int64_t pos = akv_load_index(a.positions, a.pos_it, ax * a.pos_axis + tok);
          pos = pos < 0 ? 0 : pos >= a.table_rows ? a.table_rows - 1 : pos;
          c[e] = a.table[pos * a.R + p0 + e];
          s[e] = a.table[pos * a.R + half + p0 + e];
        }
      }
      if (a.interleaved) {
        float u[8], w[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          u[2 * e] = x[2 * e] * c[e] - x[2 * e + 1] * s[e];
          u[2 * e + 1] = x[2 * e + 1] * c[e] + x[2 * e] * s[e];
          w[2 * e] = y[2 * e] * c[4 + e] - y[2 * e + 1] * s[4 + e];
          w[2 * e + 1] = y[2 * e + 1] * c[4 + e] + y[2 * e] * s[4 + e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) { x[e] = u[e]; y[e] = w[e]; }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float u = x[e] * c[e] - y[e] * s[e];
          y[e] = y[e] * c[e] + x[e] * s[e];
          x[e] = u;
        }
      }
    }
    if (is_q) {
      rp_store<XDT, VEC, PAST>(a.q_out, dst + d0, x);
      rp_store<XDT, VEC, PAST>(a.q_out, dst + d1, y);
    } else {
      void* to = is_k ? a.kc : a.vc;
      rp_store<CDT, VEC, PAST>(to, dst + d0, x);
      rp_store<CDT, VEC, PAST>(to, dst + d1, y);
    }
  }
}

template <int XDT, int CDT, bool VEC, bool PAST> static int rp_launch(const rp_args& a, hipStream_t s) {
  const int cus = akv_cached_cu_count();
  const int64_t blocks = (a.units + 255) / 256, most = (int64_t)(cus > 0 ? cus : 256) * 64;
  rp_kernel<XDT, CDT, VEC, PAST><<<(int)(blocks < most ? blocks : most), 256, 0, s>>>(a);
  AKV_LAUNCH_CHECK("rp_kernel");
  return AKV_OK;
}
template <int XDT, int CDT> static int rp_launch(const rp_args& a, bool vec, hipStream_t s) {
  // What no cache could keep anyway is stored past it: 4097 tokens of 48 rows of 128 with three axes 19.8 us (otherwise 23.0), 8192 of one
  // axis 43.0 (47.6).  Up to the 32 MB of the second-level caches the attention that follows finds the rows there.
  const bool past = a.units * 32 * (XDT == AKV_F32 ? 2 : 1) > (32 << 20);
  return !vec ? rp_launch<XDT, CDT, false, false>(a, s) : past ? rp_launch<XDT, CDT, true, true>(a, s) : rp_launch<XDT, CDT, true, false>(a, s);
}
template <int XDT> static int rp_launch(const rp_args& a, int cdt, bool vec, hipStream_t s) {
  return cdt == AKV_F16 ? rp_launch<XDT, AKV_F16>(a, vec, s) : cdt == AKV_BF16 ? rp_launch<XDT, AKV_BF16>(a, vec, s) : rp_launch<XDT, AKV_F32>(a, vec, s);
}

extern "C" int akv_rope_append(const void* query, int64_t qs_tok, int64_t qs_head, void* query_out, int64_t qo_tok, int64_t qo_head,
                               const void* key, int64_t ks_tok, int64_t ks_head, const void* value, int64_t vs_tok, int64_t vs_head, int x_dtype,
                               const void* positions, int pos_itype, int64_t pos_axis_stride, const float* cos_sin, int64_t cos_sin_rows, int rotary_dim,
                               const int* sections, int num_axes, int interleaved, const void* slot_mapping, int slot_itype,
                               void* key_cache, int64_t kc_blk, int64_t kc_pos, int64_t kc_head, void* value_cache, int64_t vc_blk, int64_t vc_pos, int64_t vc_head, int cache_dtype,
                               int64_t num_tokens, int num_q_heads, int num_kv_heads, int d, int block_size, int64_t num_blocks, void* stream) {
  const char* name = "akv_rope_append";
  AKV_REQUIRE(akv_valid_dtype(x_dtype) && akv_valid_dtype(cache_dtype), "%s: bad dtype", name);
  AKV_REQUIRE(akv_valid_itype(slot_itype) && akv_valid_itype(pos_itype), "%s: bad index type", name);
  AKV_REQUIRE(num_tokens >= 0 && num_q_heads >= 0 && num_kv_heads >= 0 && d > 0 && block_size > 0 && num_blocks >= 0, "%s: bad sizes", name);
  AKV_REQUIRE(rotary_dim >= 0 && rotary_dim <= d, "%s: rotary_dim %d of %d coordinates", name, rotary_dim, d);
  AKV_REQUIRE(num_axes >= 1 && num_axes <= RP_AXES, "%s: %d position axes; 1 to %d are supported", name, num_axes, RP_AXES);
  if (num_tokens == 0 || num_q_heads + num_kv_heads == 0) return AKV_OK;
  AKV_REQUIRE(num_q_heads == 0 || (query && query_out), "%s: null pointer", name);
  AKV_REQUIRE(num_kv_heads == 0 || (key && value && slot_mapping), "%s: null pointer", name);
  AKV_REQUIRE(num_kv_heads == 0 || num_blocks == 0 || (key_cache && value_cache), "%s: null pointer", name);
  AKV_REQUIRE(rotary_dim == 0 || (positions && cos_sin && cos_sin_rows > 0), "%s: positions and a table are needed to rotate", name);
  AKV_REQUIRE(num_axes == 1 || sections, "%s: sections are needed for several axes", name);
  if (d % 16 != 0 || rotary_dim % 16 != 0) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: head_dim %d and rotary_dim %d must be multiples of 16", name, d, rotary_dim);
  if (((uintptr_t)cos_sin & 15) != 0) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: the table must lie at a multiple of 16 bytes", name);
  rp_args a = {};
  a.q = {query, qs_tok, qs_head}; a.k = {key, ks_tok, ks_head}; a.v = {value, vs_tok, vs_head};
  a.q_out = query_out; a.qo_tok = qo_tok; a.qo_head = qo_head;
  a.kc = key_cache; a.kc_blk = kc_blk; a.kc_pos = kc_pos; a.kc_head = kc_head;
  a.vc = value_cache; a.vc_blk = vc_blk; a.vc_pos = vc_pos; a.vc_head = vc_head;
  a.positions = positions; a.pos_axis = pos_axis_stride; a.pos_it = pos_itype;
  a.table = cos_sin; a.table_rows = cos_sin_rows; a.slots = slot_mapping; a.slots_it = slot_itype;
  a.slots_end = num_blocks * block_size;
  a.QH = num_q_heads; a.KVH = num_kv_heads; a.R = rotary_dim; a.block_size = block_size; a.axes = num_axes; a.interleaved = interleaved;
  bool whole = true;
  if (num_axes > 1) {
    int end = 0;
    for (int i = 0; i < num_axes; ++i) {
      AKV_REQUIRE(sections[i] >= 0 && sections[i] <= rotary_dim / 2, "%s: bad section %d", name, sections[i]);
      end += sections[i];
      a.ends[i] = end;
      whole = whole && end % 8 == 0;
    }
    AKV_REQUIRE(end == rotary_dim / 2, "%s: sections of %d pairs, but %d pairs turn", name, end, rotary_dim / 2);
  }
  const int64_t rows = (int64_t)num_q_heads + 2 * (int64_t)num_kv_heads;
  AKV_REQUIRE(rows * (d / 16) <= 0x7fffffff, "%s: too many heads", name);
  a.per_row = (uint32_t)(d / 16);
  a.per_token = (uint32_t)(rows * (d / 16));
  a.units = num_tokens * (int64_t)a.per_token;
  a.whole = whole;
  // 16-byte accesses where every row begins at a multiple of 16 bytes
  const int64_t xs = qs_tok | qs_head | qo_tok | qo_head | ks_tok | ks_head | vs_tok | vs_head, cs = kc_blk | kc_pos | kc_head | vc_blk | vc_pos | vc_head;
  const uintptr_t xp = (uintptr_t)query | (uintptr_t)query_out | (uintptr_t)key | (uintptr_t)value, cp = (uintptr_t)key_cache | (uintptr_t)value_cache;
  const bool vec = ((xp | cp) & 15) == 0 && (xs & (x_dtype == AKV_F32 ? 3 : 7)) == 0 && (cs & (cache_dtype == AKV_F32 ? 3 : 7)) == 0;
  const hipStream_t s = (hipStream_t)stream;
  return x_dtype == AKV_F16 ? rp_launch<AKV_F16>(a, cache_dtype, vec, s) : x_dtype == AKV_BF16 ? rp_launch<AKV_BF16>(a, cache_dtype, vec, s) : rp_launch<AKV_F32>(a, cache_dtype, vec, s);
}
