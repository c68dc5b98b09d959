// akv_sparse_attn: causal attention of new tokens over the blocks of a paged cache of plain rows that each token and kv head has selected.
//
//   S^T[key, row] = K[key, :] . Q[row, :]          v_mfma_f32_16x16x32, A = 16 keys, B = 16 rows
//   O^T[d, row] = sum_key V[key, d] P^T[key, row]  A = 16 coordinates, B = 16 rows
//
// The rows of a tile are (token, query head) pairs of one kv head, as many tokens of a sequence as fit sixteen rows.  Neighbouring tokens
// select much the same blocks, so the tile reads the union of what its tokens selected, each block once, and a bit a token says whose it is.
// A lane holds one row and, of sixteen keys, four: the softmax is taken in the lane with an exchange between the four rows of lanes, and
// the weights of two groups of sixteen keys are the operand of the second product, whose k axis takes keys in the order in which lanes hold
// them.  V^T comes out of LDS by transposing reads (four keys of a coordinate a lane).
#include "akv_batch.h"
#include "akv_device_once.h"

struct sa_args {
  ab_batch b;
  const void* q; int64_t qs_tok, qs_head;
  const uint8_t* k; int64_t k_blk, k_pos, k_head;    // bytes
  const uint8_t* v; int64_t v_blk, v_pos, v_head;
  const int32_t* selected; int64_t ss_tok, ss_head;
  void* out; int64_t os_tok, os_head;
  int KVH, QH, G, HS, GC, TG;           // G query heads a kv head in HS groups of GC; TG tokens a tile
  int k_sel, words;                     // entries of a list of selected blocks; words of a bitmap of table columns
  int parts; uint32_t parts_recip;      // groups of sixteen keys a block
  int tail;
  float scale2;
};

#define SA_FRAME 8.f
template <int DT> constexpr float SA_LIFT = DT == AKV_BF16 ? 0.f : 5.f;

template <int D> struct sa_lds {        // behind bitmaps (or in their place) and lists
  static constexpr int WAVES = 4, V_BYTES = 32 * 2 * D, STAGE = WAVES * V_BYTES;
  static __device__ __forceinline__ int f(int r) { return D == 64 ? 2 * ((r >> 1) & 3) : 2 * (r & 7); }
};

template <int D, int DT> __global__ __launch_bounds__(256, 2) void sa_kernel(sa_args a) {
  typedef sa_lds<D> P;
  typedef ab_math<DT> M;
  constexpr int KS = D / 32, OT = D / 16, LPR = D / 8, RPI = 64 / LPR, VI = 32 / RPI, W = P::WAVES;
  extern __shared__ __align__(1024) unsigned char lds[];
  __shared__ int wave_sum[W];
  __shared__ float2 ml[W][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, hq = lane >> 4;
  const int heads = a.KVH * a.HS, bs = a.b.block_size;
  const int head = blockIdx.x % heads;
  const int64_t x = blockIdx.x / heads;
  const int kvh = head / a.HS, g0 = (head % a.HS) * a.GC;

  // rows before the first sequence, by all workgroups
  const int front = a.tail ? ab_start(a.b, 0) : 0;
  if (front > 0) {
    const int64_t per = (int64_t)a.QH * (D / 4);
    for (int64_t i = (int64_t)blockIdx.x * 256 + tid; i < front * per; i += (int64_t)gridDim.x * 256) {
      const int64_t token = i / per, rest = i - token * per, hd = rest / (D / 4);
      *(ab_u2*)((uint16_t*)a.out + token * a.os_tok + hd * a.os_head + 4 * (rest - hd * (D / 4))) = (ab_u2){0u, 0u};
    }
  }
  // Tiles are numbered with gaps: tile j of sequence i is floor(start_i / TG) + i + j; sequence S is the rows behind the last.
  const int seq = ab_last(a.b.S + 1, x, [&](int i) { return (int64_t)ab_start(a.b, i) / a.TG + i; });
  if (seq < 0) return;
  const int s0 = ab_start(a.b, seq), s1 = seq < a.b.S ? ab_start(a.b, seq + 1) : a.tail ? a.b.T : s0;
  const int64_t first64 = s0 + (x - ((int64_t)s0 / a.TG + seq)) * a.TG;
  if (first64 >= s1) return;
  const int first = (int)first64, tokens = min(a.TG, s1 - first);
  const int pos0 = seq < a.b.S ? ab_ctx(a.b, seq) - (s1 - first) : -tokens;      // position of the first token
  const int last = pos0 + tokens - 1;
  const int t_row = col / a.GC, g_row = g0 + col - t_row * a.GC;
  const bool valid = t_row < tokens && g_row < a.G;
  const int pos = valid ? pos0 + t_row : -1;
  const int64_t q_row = valid ? (int64_t)(first + t_row) * a.qs_tok + (int64_t)(kvh * a.G + g_row) * a.qs_head : 0;

  ab_u4 q[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    q[ks] = (ab_u4){0u, 0u, 0u, 0u};
    if (valid) q[ks] = *(const ab_u4*)((const uint16_t*)a.q + q_row + 32 * ks + 8 * hq);
  }

  // ---- the union of what the tokens selected
  unsigned char* const stage = lds;
  uint32_t* const bits = (uint32_t*)lds;             // [TG][words], before the values
  const int cap = min(a.TG * a.k_sel, a.words * 32);
  const int area = max(P::STAGE, (a.TG * a.words * 4 + 15) & ~15);
  int* const cols = (int*)(lds + area);
  int* const blks = cols + cap;
  uint16_t* const masks = (uint16_t*)(blks + cap);
  const int words = last >= 0 ? last / bs / 32 + 1 : 0;
  for (int i = tid; i < tokens * words; i += 256) bits[i] = 0u;
  __syncthreads();
  if (words > 0) {
    for (int i = tid; i < tokens * a.k_sel; i += 256) {
      const int t = i / a.k_sel;
      const int c = a.selected[(int64_t)(first + t) * a.ss_tok + (int64_t)kvh * a.ss_head + (i - t * a.k_sel)];
      if (pos0 + t >= 0 && c >= 0 && c <= (pos0 + t) / bs) atomicOr(bits + t * words + (c >> 5), 1u << (c & 31));
    }
  }
  __syncthreads();
  int count = 0;
  for (int w0 = 0; w0 < words; w0 += 256) {
    uint32_t u = 0u;
    if (w0 + tid < words)
      for (int t = 0; t < tokens; ++t) u |= bits[t * words + w0 + tid];
    const int mine = __popc(u), inc = akv_wave_inclusive_scan(mine);
    if (lane == 63) wave_sum[wave] = inc;
    __syncthreads();
    int at = count + inc - mine;
    for (int w = 0; w < W; ++w) {
      const int s = wave_sum[w];
      if (w < wave) at += s;
      count += s;
    }
    for (; u; u &= u - 1) cols[at++] = 32 * (w0 + tid) + __ffs(u) - 1;
    __syncthreads();
  }
  for (int i = tid; i < count; i += 256) {
    const int c = cols[i];
    uint32_t m = 0u;
    for (int t = 0; t < tokens; ++t) m |= ((bits[t * words + (c >> 5)] >> (c & 31)) & 1u) << t;
    blks[i] = (int)ab_block(a.b, seq, c);
    masks[i] = (uint16_t)m;
  }
  __syncthreads();           // (the bitmaps have been read)

  // ---- the wavefront's groups of 2 x 16 keys
  const int groups = count * a.parts;
  unsigned char* const vl = stage + wave * P::V_BYTES;
  uint32_t v_at[OT];
#pragma unroll
  for (int dt = 0; dt < OT; ++dt) {
    const int r = 4 * hq + (lane & 15) / 4, c = 2 * dt + ((lane & 3) >> 1);
    v_at[dt] = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)vl + r * 2 * D + 16 * (c ^ P::f(r)) + 8 * (lane & 1);
  }
  struct keys {
    ab_u4 k[2][KS], v[VI];
    int base[2], end[2];               // of sixteen keys: position of the first, one past the last of the block (0: none)
    uint32_t mask[2];
  };
  auto request = [&](int p, keys& w) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int st = __builtin_amdgcn_readfirstlane(min(2 * p + s, groups - 1));
      uint32_t part;
      const int e = (int)akv_div32((uint32_t)st, (uint32_t)a.parts, a.parts_recip, part);
      const int64_t blk = __builtin_amdgcn_readfirstlane(blks[e]);
      const int c = __builtin_amdgcn_readfirstlane(cols[e]), place = 16 * (int)part;
      w.base[s] = c * bs + place;
      w.end[s] = 2 * p + s < groups ? c * bs + bs : 0;
      w.mask[s] = __builtin_amdgcn_readfirstlane(masks[e]);
      const uint8_t* kp = a.k + blk * a.k_blk + (int64_t)kvh * a.k_head + (int64_t)min(place + col, bs - 1) * a.k_pos + 16 * hq;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) w.k[s][ks] = *(const ab_u4*)(kp + 64 * ks);
      const uint8_t* vp = a.v + blk * a.v_blk + (int64_t)kvh * a.v_head + 16 * (lane % LPR);
#pragma unroll
      for (int i = 0; i < VI / 2; ++i) {
        // (a value that no token of the tile may see is zero, whatever lies there)
        const int r = RPI * i + lane / LPR, key = w.base[s] + r;
        w.v[s * (VI / 2) + i] = *(const ab_u4*)(vp + (int64_t)min(place + r, bs - 1) * a.v_pos);
        if (key > last || key >= w.end[s]) w.v[s * (VI / 2) + i] = (ab_u4){0u, 0u, 0u, 0u};
      }
    }
  };
  ab_f4 o[OT];
#pragma unroll
  for (int i = 0; i < OT; ++i) o[i] = (ab_f4){0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  for (int p = wave; 2 * p < groups; p += W) {
    keys w;
    request(p, w);
    akv_wave_sync();                   // (the values before have been read)
#pragma unroll
    for (int i = 0; i < VI; ++i) {
      const int r = RPI * i + lane / LPR;
      *(ab_u4*)(vl + r * 2 * D + 16 * ((lane % LPR) ^ P::f(r))) = w.v[i];
    }
    ab_f4 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = (ab_f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s[t] = M::mfma16(w.k[t][ks], q[ks], s[t]);
    }
    float top = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int limit = ((w.mask[t] >> t_row) & 1u) ? min(w.end[t] - 1, pos) : -1;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[t][i] = w.base[t] + 4 * hq + i <= limit ? s[t][i] * a.scale2 : -INFINITY;
        top = fmaxf(top, s[t][i]);
      }
    }
    top = akv_rows_max(top);
    const bool grown = top - m > SA_LIFT<DT> + SA_FRAME;
    if (__ballot(grown)) {
      const float to = grown ? top - SA_LIFT<DT> : m, alpha = grown ? __builtin_amdgcn_exp2f(m - to) : 1.f;
      m = to;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < OT; ++i) o[i] *= alpha;
    }
    const float ref = m == -INFINITY ? 0.f : m;
    ab_u4 pw;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[t][i] = __builtin_amdgcn_exp2f(s[t][i] - ref);
        l += s[t][i];
      }
      pw[2 * t] = M::pair(s[t][0], s[t][1]);
      pw[2 * t + 1] = M::pair(s[t][2], s[t][3]);
    }
    akv_wave_sync();
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4 lds_s4;
#pragma unroll
    for (int dt = 0; dt < OT; ++dt) {
      const ab_u2 lo = __builtin_bit_cast(ab_u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)v_at[dt]));
      const ab_u2 hi = __builtin_bit_cast(ab_u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)(v_at[dt] + 16 * 2 * D)));
      o[dt] = M::mfma16((ab_u4){lo[0], lo[1], hi[0], hi[1]}, pw, o[dt]);
    }
  }

  // ---- the wavefronts' sums together
  l = akv_rows_sum(l);
  if (hq == 0) ml[wave][col] = make_float2(m, l);
  __syncthreads();           // (the values have been read)
  float4* const part = (float4*)stage;
#pragma unroll
  for (int dt = 0; dt < OT; ++dt) part[(wave * OT + dt) * 64 + lane] = make_float4(o[dt][0], o[dt][1], o[dt][2], o[dt][3]);
  __syncthreads();
  float top = -INFINITY, sum = 0.f, f[W];
#pragma unroll
  for (int w = 0; w < W; ++w) top = fmaxf(top, ml[w][col].x);
#pragma unroll
  for (int w = 0; w < W; ++w) {
    f[w] = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[w][col].x - top);
    sum = fmaf(ml[w][col].y, f[w], sum);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (valid) {
    uint16_t* to = (uint16_t*)a.out + (int64_t)(first + t_row) * a.os_tok + (int64_t)(kvh * a.G + g_row) * a.os_head + 4 * hq;
    for (int dt = wave; dt < OT; dt += W) {
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float4 z = part[(w * OT + dt) * 64 + lane];
        y.x = fmaf(z.x, f[w], y.x); y.y = fmaf(z.y, f[w], y.y); y.z = fmaf(z.z, f[w], y.z); y.w = fmaf(z.w, f[w], y.w);
      }
      *(ab_u2*)(to + 16 * dt) = (ab_u2){M::pair(y.x * inv, y.y * inv), M::pair(y.z * inv, y.w * inv)};
    }
  }
}

#define SA_LDS (150 << 10)
#define SA_MOST_SELECTED 4096
template <int D, int DT> static int sa_launch(sa_args a, hipStream_t stream) {
  a.HS = (a.G + 15) / 16;
  a.GC = (a.G + a.HS - 1) / a.HS;
  a.parts = (a.b.block_size + 15) / 16;
  a.parts_recip = (uint32_t)(0xffffffffull / (uint32_t)a.parts);
  a.words = (int)((a.b.max_blocks + 31) / 32);
  if (a.words < 1) a.words = 1;
  int64_t bytes = 0;
  for (a.TG = 16 / a.GC;; a.TG = (a.TG + 1) / 2) {
    const int64_t bits = ((int64_t)a.TG * a.words * 4 + 15) & ~15ll, all = (int64_t)a.words * 32;
    const int64_t cap = (int64_t)a.TG * a.k_sel < all ? (int64_t)a.TG * a.k_sel : all;
    bytes = (bits > sa_lds<D>::STAGE ? bits : sa_lds<D>::STAGE) + 10 * cap;
    if (bytes <= SA_LDS || a.TG == 1) break;
  }
  if (bytes > SA_LDS) return akv_fail(AKV_ERR_UNSUPPORTED, "akv_sparse_attn: block tables of %lld columns", (long long)a.b.max_blocks);
  const int64_t tiles = (int64_t)a.b.T / a.TG + a.b.S + 1, units = tiles * a.KVH * a.HS;
  if (units > 0x7fffffff) return akv_fail(AKV_ERR_UNSUPPORTED, "akv_sparse_attn: more than 2^31 rows");
  int dev = 0;
  AKV_HIP(hipGetDevice(&dev));
  static akv_device_once once;
  if (const int rc = once(dev, [&]() -> int { return ab_lds((const void*)sa_kernel<D, DT>, SA_LDS); })) return rc;
  sa_kernel<D, DT><<<(uint32_t)units, 256, bytes, stream>>>(a);
  AKV_LAUNCH_CHECK("sa_kernel");
  return AKV_OK;
}

extern "C" int akv_sparse_attn(const void* query, int dtype, int64_t qs_tok, int64_t qs_head, const void* key_cache, int64_t ks_blk, int64_t ks_pos, int64_t ks_head, const void* value_cache,
                               int64_t vs_blk, int64_t vs_pos, int64_t vs_head, const void* block_tables, int bt_itype, int64_t bt_stride, const void* context_lens, int cl_itype,
                               const void* query_starts, int qs_itype, const int32_t* selected, int64_t ss_tok, int64_t ss_head, int num_selected, void* out, int64_t os_tok, int64_t os_head,
                               int zero_tail, int num_seqs, int64_t num_tokens, int num_q_heads, int num_kv_heads, int d, int block_size, int64_t num_blocks, int64_t max_blocks_per_seq,
                               float scale, void* stream) {
  const char* name = "akv_sparse_attn";
  AKV_REQUIRE(akv_valid_dtype(dtype), "%s: bad dtype %d", name, dtype);
  const int rc = ab_check(name, block_tables, bt_itype, context_lens, cl_itype, query_starts, qs_itype, num_seqs, num_tokens, num_kv_heads, block_size, num_blocks, max_blocks_per_seq);
  if (rc) return rc;
  AKV_REQUIRE(num_q_heads > 0 && num_q_heads % num_kv_heads == 0, "%s: %d query heads on %d kv heads", name, num_q_heads, num_kv_heads);
  AKV_REQUIRE(num_selected >= 0, "%s: %d selected blocks", name, num_selected);
  AKV_REQUIRE(scale > 0.f && scale < INFINITY, "%s: scale must be positive and finite", name);
  if (dtype == AKV_F32) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: float32 queries are not supported; use float16 or bfloat16", name);
  if (!ab_head_size(d)) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: head_dim %d; kernels are built for 64, 128 and 256", name, d);
  if (num_tokens == 0) return AKV_OK;
  AKV_REQUIRE(query && out && query_starts && (selected || num_selected == 0), "%s: null pointer", name);
  AKV_REQUIRE(num_blocks == 0 || (key_cache && value_cache), "%s: null pointer", name);
  if (block_size > 4096) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: blocks of %d tokens", name, block_size);
  if (num_selected > SA_MOST_SELECTED) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: more than %d selected blocks", name, SA_MOST_SELECTED);
  if (!ab_aligned(query, 16) || !ab_aligned(key_cache, 16) || !ab_aligned(value_cache, 16) || !ab_aligned(out, 8) || ((qs_tok | qs_head | ks_blk | ks_pos | ks_head | vs_blk | vs_pos | vs_head) & 7) || ((os_tok | os_head) & 3))
    return akv_fail(AKV_ERR_UNSUPPORTED, "%s: rows must lie at multiples of 16 bytes (outputs of 8)", name);
  sa_args a = {};
  a.b = ab_make(block_tables, bt_itype, bt_stride, context_lens, cl_itype, query_starts, qs_itype, num_seqs, num_tokens, block_size, num_blocks, max_blocks_per_seq);
  a.q = query; a.qs_tok = qs_tok; a.qs_head = qs_head;
  a.k = (const uint8_t*)key_cache; a.k_blk = 2 * ks_blk; a.k_pos = 2 * ks_pos; a.k_head = 2 * ks_head;
  a.v = (const uint8_t*)value_cache; a.v_blk = 2 * vs_blk; a.v_pos = 2 * vs_pos; a.v_head = 2 * vs_head;
  a.selected = selected; a.ss_tok = ss_tok; a.ss_head = ss_head; a.k_sel = num_selected;
  a.out = out; a.os_tok = os_tok; a.os_head = os_head;
  a.KVH = num_kv_heads; a.QH = num_q_heads; a.G = num_q_heads / num_kv_heads;
  a.tail = zero_tail; a.scale2 = scale * 1.44269504088896341f;
  const hipStream_t s = (hipStream_t)stream;
#define SA_CASE(DIM) if (d == DIM) return dtype == AKV_F16 ? sa_launch<DIM, AKV_F16>(a, s) : sa_launch<DIM, AKV_BF16>(a, s);
  SA_CASE(64) SA_CASE(128) SA_CASE(256)
#undef SA_CASE
  return AKV_ERR_UNSUPPORTED;
}
