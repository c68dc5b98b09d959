// akv_sparse_attn: causal attention of new tokens over the blocks of a paged cache of plain rows that each token and kv head has selected.
//
//   S^T[key, row] = K[key, :] . Q[row, :]          v_mfma_f32_32x32x16, A = 32 keys, B = 32 rows
//   O^T[d, row] = sum_key V[key, d] P^T[key, row]  A = 32 coordinates, B = 32 rows
//
// The rows of a tile are (token, query head) pairs of one kv head, as many tokens of a sequence as fit 32 rows.  Neighbouring tokens select much
// the same blocks, so the tile reads the union of what its tokens selected, each block once, and a bit a token says whose it is.  A lane holds one
// row and half of 32 keys: the softmax is taken in the lane with one exchange between the halves of the wavefront, and the weights are the operand of
// the second product, whose k axis takes keys in the order in which lanes hold them.  V^T comes out of LDS by transposing reads (four keys of a
// coordinate a lane).
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
  int splits;                           // workgroups that share a tile's keys
  float* part; float2* part_ml;         // of splits > 1, [T][QH][splits]: sums of D coordinates; largest score, sum of weights
};

#define SA_FRAME 8.f
template <int DT> constexpr float SA_LIFT = DT == AKV_BF16 ? 0.f : 5.f;

// Of a wavefront in LDS, behind bitmaps (or in their place) and before lists: 32 keys, then in their place 32 values, then 64 coordinates of its sums.
// Rows lie apart so that the operands' reads meet no bank twice: sixteen bytes more for keys, 32 for transposing reads of values.
template <int D> struct sa_lds {
  static constexpr int W = 4;           // wavefronts
  static constexpr int K_ROW = 2 * D + 16, V_ROW = 2 * D + 32, WAVE = 32 * V_ROW, AREA = W * (WAVE > 8192 ? WAVE : 8192) + 32 * K_ROW;
};

// What a CU takes in bounds long prompts: 2048 tokens, 64 blocks of some 1900 each, 8 heads of 128, read 3.1 GB in tiles (of eight tokens some 190 blocks a
// head; 84 % found in the second cache) and take 197 us, 16 TB/s or 26 bytes a clock and CU; LDS is busy for 51 % of clocks, the vector unit 41 %, the
// matrix cores 24 %.  Keys in the operand's order straight from memory, a row a lane, took 337 us (the address unit takes a line a clock); tiles of
// sixteen rows 277, 32 rows 217, with queries in LDS and keys or values on their way, not both, so that three workgroups fit a CU, 201, without comparisons where
// no key lies ahead 195.  Four groups of sixteen rows that share steps of keys in LDS halve what is read, and took 257: each wavefront multiplies half of a
// step, and all wait at its ends.
template <int D, int DT> __global__ __launch_bounds__(256, D == 256 ? 1 : D == 128 ? 3 : 4) void sa_kernel(sa_args a) {
  typedef sa_lds<D> P;
  typedef ab_math<DT> M;
  constexpr int KS = D / 16, OT = D / 32, LPR = D / 8, RPI = 64 / LPR, VI = 32 / RPI, W = P::W, THREADS = 64 * W;
  extern __shared__ __align__(1024) unsigned char lds[];
  __shared__ int wave_sum[W];
  __shared__ float2 ml[W][32];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), row = lane & 31, half = lane >> 5;
  const int heads = a.KVH * a.HS, bs = a.b.block_size;
  const int head = blockIdx.x % heads;
  const int64_t x = blockIdx.x / heads;
  const int kvh = head / a.HS, g0 = (head % a.HS) * a.GC;

  // rows before the first sequence, by all workgroups
  const int front = a.tail ? ab_start(a.b, 0) : 0;
  if (front > 0 && blockIdx.y == 0) {
    const int64_t per = (int64_t)a.QH * (D / 4);
    for (int64_t i = (int64_t)blockIdx.x * THREADS + tid; i < front * per; i += (int64_t)gridDim.x * THREADS) {
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
  const int t_row = row / a.GC, g_row = g0 + row - t_row * a.GC;
  const bool valid = t_row < tokens && g_row < a.G;
  const int pos = valid ? pos0 + t_row : -1;

  // ---- the union of what the tokens selected
  uint32_t* const bits = (uint32_t*)lds;             // [TG][words], before the values
  const int cap = min(a.TG * a.k_sel, a.words * 32);
  const int area = max(P::AREA, (a.TG * a.words * 4 + 15) & ~15);
  int* const cols = (int*)(lds + area);
  int* const blks = cols + cap;
  uint32_t* const masks = (uint32_t*)(blks + cap);
  const int words = last >= 0 ? last / bs / 32 + 1 : 0;
  for (int i = tid; i < tokens * words; i += THREADS) bits[i] = 0u;
  __syncthreads();
  if (words > 0) {
    for (int i = tid; i < tokens * a.k_sel; i += THREADS) {
      const int t = i / a.k_sel;
      const int c = a.selected[(int64_t)(first + t) * a.ss_tok + (int64_t)kvh * a.ss_head + (i - t * a.k_sel)];
      if (pos0 + t >= 0 && c >= 0 && c <= (pos0 + t) / bs) atomicOr(bits + t * words + (c >> 5), 1u << (c & 31));
    }
  }
  __syncthreads();
  int count = 0;
  for (int w0 = 0; w0 < words; w0 += THREADS) {
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
  for (int i = tid; i < count; i += THREADS) {
    const int c = cols[i];
    uint32_t m = 0u;
    for (int t = 0; t < tokens; ++t) m |= ((bits[t * words + (c >> 5)] >> (c & 31)) & 1u) << t;
    blks[i] = (int)ab_block(a.b, seq, c);
    masks[i] = m;
  }
  __syncthreads();           // (the bitmaps have been read)

  // rows of queries for the operand's reads, the same for all wavefronts
  const uint32_t q_lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds + P::AREA - 32 * P::K_ROW, q_at = q_lds + row * P::K_ROW + 16 * half;
  for (int i = tid; i < 32 * LPR; i += THREADS) {
    const int r = i / LPR, t = r / a.GC, g = g0 + r - t * a.GC;
    ab_u4 x = {0u, 0u, 0u, 0u};
    if (t < tokens && t < a.TG && g < a.G) x = *(const ab_u4*)((const uint16_t*)a.q + (int64_t)(first + t) * a.qs_tok + (int64_t)(kvh * a.G + g) * a.qs_head + 8 * (i % LPR));
    *(__attribute__((address_space(3))) ab_u4*)(uintptr_t)(q_lds + r * P::K_ROW + 16 * (i % LPR)) = x;
  }

  // ---- the wavefront's units of 2 x 16 keys: rows arrive in the order in which they lie, and go through LDS into that of the operands
  const int sixteens = count * a.parts, units = (sixteens + 1) / 2;
  const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds + wave * P::WAVE;
  const uint32_t k_at = at + row * P::K_ROW + 16 * half, v_at = at + (4 * half + (lane & 15) / 4) * P::V_ROW + 32 * (lane >> 4 & 1) + 8 * (lane & 3);
  typedef __attribute__((address_space(3))) ab_u4 lds_u4;
  typedef short s4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s4 lds_s4;
  const uint8_t* const kp = a.k + (int64_t)kvh * a.k_head;
  const uint8_t* const vp = a.v + (int64_t)kvh * a.v_head;
  const uint32_t k_pos = (uint32_t)a.k_pos, v_pos = (uint32_t)a.v_pos;
  uint32_t k_off[VI / 2], v_off[VI / 2];             // a thread's pieces of a sixteen
#pragma unroll
  for (int i = 0; i < VI / 2; ++i) {
    k_off[i] = (RPI * i + lane / LPR) * k_pos + 16 * (lane % LPR);
    v_off[i] = (RPI * i + lane / LPR) * v_pos + 16 * (lane % LPR);
  }
  // An entry of the lists for each sixteen of a unit, in two lanes in turn (looked up a unit ahead, so that nothing waits for it), and what is made of it.
  struct entry { int blk, col, mask, place; };
  struct unit { const uint8_t *k[2], *v[2]; int left[2], base[2], mask[2]; };        // keys of the block from there on, position of the first, whose they are
  auto look = [&](int p) {
    const int st = 2 * p + (lane & 1);
    uint32_t part;
    const int e = (int)akv_div32((uint32_t)max(0, min(st, sixteens - 1)), (uint32_t)a.parts, a.parts_recip, part);
    return entry{blks[e], cols[e], st < sixteens ? (int)masks[e] : 0, 16 * (int)part};
  };
  auto find = [&](const entry& x) {
    unit u;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int64_t blk = __builtin_amdgcn_readlane(x.blk, s);
      const int place = __builtin_amdgcn_readlane(x.place, s);
      u.k[s] = kp + blk * a.k_blk + place * a.k_pos;
      u.v[s] = vp + blk * a.v_blk + place * a.v_pos;
      u.left[s] = min(16, bs - place);
      u.base[s] = __builtin_amdgcn_readlane(x.col, s) * bs + place;
      u.mask[s] = __builtin_amdgcn_readlane(x.mask, s);
    }
    return u;
  };
  auto request = [&](ab_u4* to, const uint8_t* const* from, const int* left, const uint32_t* off, uint32_t pos) {
#pragma unroll
    for (int i = 0; i < VI; ++i) to[i] = *(const ab_u4*)(from[2 * i / VI] + min(off[i % (VI / 2)], (left[2 * i / VI] - 1) * pos + 16 * (lane % LPR)));
  };
  // (A weight of zero times a value that is not finite is no zero.  What no token of the tile may see is a zero in LDS, whatever lies in the cache; where a token
  // would meet such a value of another, the tile is done again a token at a time.)
  __syncthreads();
  for (int only = -1;;) {
    const int seen = only < 0 ? last : pos0 + only;  // position of the last key that is seen
    const uint32_t mine = only < 0 ? 0xffffffffu : 1u << only;
    ab_f16 o[OT];
#pragma unroll
    for (int i = 0; i < OT; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) o[i][j] = 0.f;
    float m = -INFINITY, l = 0.f;
    ab_u4 x[VI];             // keys or values on their way
    unit now = {};
    entry ahead = {};
    const int mine0 = (int)blockIdx.y * W + wave, stride = a.splits * W;
    if (mine0 < units) {
      now = find(look(mine0));
      ahead = look(mine0 + stride);
      request(x, now.k, now.left, k_off, k_pos);
    }
    for (int p = mine0; p < units; p += stride) {
      const bool more = p + stride < units;
      const unit next = find(ahead);
      ahead = look(p + 2 * stride);
      akv_wave_sync();                   // (the values before have been read)
#pragma unroll
      for (int i = 0; i < VI; ++i) *(lds_u4*)(uintptr_t)(at + (RPI * i + lane / LPR) * P::K_ROW + 16 * (lane % LPR)) = x[i];
      request(x, now.v, now.left, v_off, v_pos);
      akv_wave_sync();
      ab_f16 s;
#pragma unroll
      for (int j = 0; j < 16; ++j) s[j] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s = M::mfma32(*(const lds_u4*)(uintptr_t)(k_at + 32 * ks), *(const lds_u4*)(uintptr_t)(q_at + 32 * ks), s);
      // Where every token stands behind all 32 keys, a row is selected or not: what is added to its scores says so.  (A score that is no finite number makes
      // the sum none, and the tile is done again.)
      const bool plain = only < 0 && min(now.left[0], now.left[1]) >= 16 && max(now.base[0], now.base[1]) + 15 <= pos0;
      float off[2], most_of[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const bool his = (now.mask[t] & mine) >> t_row & 1;
        if (!plain) {
          const int limit = (his ? min(now.left[t] - 1, pos - now.base[t]) : -1) - 4 * half;
#pragma unroll
          for (int i = 0; i < 8; ++i) s[8 * t + i] = 8 * (i / 4) + i % 4 <= limit ? s[8 * t + i] : -INFINITY;
        }
        most_of[t] = s[8 * t];
#pragma unroll
        for (int i = 1; i < 8; ++i) most_of[t] = fmaxf(most_of[t], s[8 * t + i]);
        off[t] = his ? 0.f : -INFINITY;
      }
      float top = fmaxf(off[0] < 0.f ? -INFINITY : most_of[0], off[1] < 0.f ? -INFINITY : most_of[1]);
      auto other = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
      top = fmaxf(__uint_as_float(other[0]), __uint_as_float(other[1])) * a.scale2;
      const bool grown = top - m > SA_LIFT<DT> + SA_FRAME;
      if (__ballot(grown)) {
        const float to = grown ? top - SA_LIFT<DT> : m, alpha = grown ? __builtin_amdgcn_exp2f(m - to) : 1.f;
        m = to;
        l *= alpha;
#pragma unroll
        for (int i = 0; i < OT; ++i) o[i] *= alpha;
      }
      const float ref = m == -INFINITY ? 0.f : m;
      off[0] = plain ? off[0] - ref : -ref;
      off[1] = plain ? off[1] - ref : -ref;
      ab_u4 pw[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], a.scale2, off[i / 8]));
        l += s[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) pw[i / 4][i % 4] = M::pair(s[2 * i], s[2 * i + 1]);
      int held[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) held[t] = now.mask[t] & mine ? min(now.left[t], seen + 1 - now.base[t]) : 0;
      if (min(held[0], held[1]) < 16) {
#pragma unroll
        for (int i = 0; i < VI; ++i)
          if (RPI * (i % (VI / 2)) + lane / LPR >= held[2 * i / VI]) x[i] = (ab_u4){0u, 0u, 0u, 0u};
      }
#pragma unroll
      for (int i = 0; i < VI; ++i) *(lds_u4*)(uintptr_t)(at + (RPI * i + lane / LPR) * P::V_ROW + 16 * (lane % LPR)) = x[i];
      if (more) request(x, next.k, next.left, k_off, k_pos);
      akv_wave_sync();
#pragma unroll
      for (int dt = 0; dt < OT; ++dt)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const ab_u2 lo = __builtin_bit_cast(ab_u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)(v_at + 64 * dt + 16 * t * P::V_ROW)));
          const ab_u2 hi = __builtin_bit_cast(ab_u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)(v_at + 64 * dt + (16 * t + 8) * P::V_ROW)));
          o[dt] = M::mfma32((ab_u4){lo[0], lo[1], hi[0], hi[1]}, pw[t], o[dt]);
        }
      now = next;
    }

    // ---- the wavefronts' sums together
    auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(halves[0]) + __uint_as_float(halves[1]);
    if (half == 0) ml[wave][row] = make_float2(m, l);
    __syncthreads();         // (the values have been read)
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, ml[w][row].x);
#pragma unroll
    for (int w = 0; w < W; ++w) sum = fmaf(ml[w][row].y, top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[w][row].x - top), sum);
    const float inv = sum == 0.f ? 0.f : 1.f / sum, f = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    uint32_t most = 0u;      // of the sums' bits without the sign: 0x7f800000 or more where one is not finite
    uint16_t* const to = (uint16_t*)a.out + (int64_t)(first + t_row) * a.os_tok + (int64_t)(kvh * a.G + g_row) * a.os_head + 4 * half;
    float4* const part = (float4*)lds;
    const int64_t place = ((int64_t)(first + t_row) * a.QH + kvh * a.G + g_row) * a.splits + blockIdx.y;
    if (a.splits > 1 && wave == 0 && half == 0 && valid && (only < 0 || t_row == only)) a.part_ml[place] = make_float2(top, sum);
#pragma unroll
    for (int d0 = 0; d0 < OT; d0 += 2) {
      // 64 coordinates at a time; of their eight groups of 4 + 4 (a lane of each half four) a wavefront adds 8 / W
      if (d0 > 0) __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const ab_f16& x = o[d0 + i / 4];
        part[(wave * 8 + i) * 64 + lane] = make_float4(x[4 * (i % 4)] * f, x[4 * (i % 4) + 1] * f, x[4 * (i % 4) + 2] * f, x[4 * (i % 4) + 3] * f);
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8 / W; ++j) {
        const int i = wave * (8 / W) + j;
        float4 y = part[i * 64 + lane];
#pragma unroll
        for (int w = 1; w < W; ++w) {
          const float4 z = part[(w * 8 + i) * 64 + lane];
          y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
        }
        if (valid) {
          most = max(max(most, max(__float_as_uint(y.x) & 0x7fffffffu, __float_as_uint(y.y) & 0x7fffffffu)), max(__float_as_uint(y.z) & 0x7fffffffu, __float_as_uint(y.w) & 0x7fffffffu));
          if (only >= 0 && t_row != only) continue;
          if (a.splits == 1) *(ab_u2*)(to + 32 * d0 + 8 * i) = (ab_u2){M::pair(y.x * inv, y.y * inv), M::pair(y.z * inv, y.w * inv)};
          else *(float4*)(a.part + place * D + 4 * half + 32 * d0 + 8 * i) = y;
        }
      }
    }
    if (tokens == 1) break;
    const bool again = __syncthreads_or(most >= 0x7f800000u);
    if (only < 0 && !again) break;
    if (++only == tokens) break;
  }
}

// The sums of the workgroups that share a tile's keys: a wavefront a row
template <int D, int DT> __global__ __launch_bounds__(256) void sa_join_kernel(sa_args a) {
  constexpr int N = D / 64;
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), token = row / a.QH;
  if (token >= a.b.T || token < ab_start(a.b, 0) || (!a.tail && token >= ab_start(a.b, a.b.S))) return;
  const float2* const ml = a.part_ml + row * a.splits;
  const float* const from = a.part + row * a.splits * D + N * lane;
  float top = -INFINITY, sum = 0.f, y[N] = {};
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, ml[s].x);
  for (int s = 0; s < a.splits; ++s) {
    const float f = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[s].x - top);
    sum = fmaf(ml[s].y, f, sum);
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = fmaf(from[(int64_t)s * D + i], f, y[i]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint16_t* const to = (uint16_t*)a.out + token * a.os_tok + (row - token * a.QH) * a.os_head + N * lane;
  if constexpr (N == 1) *to = (uint16_t)ab_math<DT>::pair(y[0] * inv, 0.f);
  else
#pragma unroll
    for (int i = 0; i < N; i += 2) *(uint32_t*)(to + i) = ab_math<DT>::pair(y[i] * inv, y[i + 1] * inv);
}

#define SA_LDS (150 << 10)
#define SA_MOST_SELECTED 4096
#define SA_SPLITS 8
#define SA_MOST_STRIDE ((1ll << 27) - 1)          // of a block's tokens: sixteen of them within 2^32 bytes
template <int D, int DT> static int sa_launch(sa_args a, hipStream_t stream) {
  typedef sa_lds<D> P;
  a.parts = (a.b.block_size + 15) / 16;
  a.parts_recip = (uint32_t)(0xffffffffull / (uint32_t)a.parts);
  a.words = (int)((a.b.max_blocks + 31) / 32);
  if (a.words < 1) a.words = 1;
  int64_t bytes = 0;
  for (a.TG = 32 / a.GC;; a.TG = (a.TG + 1) / 2) {
    const int64_t bits = ((int64_t)a.TG * a.words * 4 + 15) & ~15ll, all = (int64_t)a.words * 32;
    const int64_t cap = (int64_t)a.TG * a.k_sel < all ? (int64_t)a.TG * a.k_sel : all;
    bytes = (bits > P::AREA ? bits : P::AREA) + 12 * cap;
    if (bytes <= SA_LDS || a.TG == 1) break;
  }
  if (bytes > SA_LDS) return akv_fail(AKV_ERR_UNSUPPORTED, "akv_sparse_attn: block tables of %lld columns", (long long)a.b.max_blocks);
  const int64_t tiles = (int64_t)a.b.T / a.TG + a.b.S + 1, units = tiles * a.KVH * a.HS;
  if (units > 0x7fffffff) return akv_fail(AKV_ERR_UNSUPPORTED, "akv_sparse_attn: more than 2^31 rows");
  int dev = 0;
  AKV_HIP(hipGetDevice(&dev));
  static akv_device_once once;
  if (const int rc = once(dev, [&]() -> int { return ab_lds((const void*)sa_kernel<D, DT>, SA_LDS); })) return rc;
  sa_kernel<D, DT><<<dim3((uint32_t)units, (uint32_t)a.splits), 64 * P::W, bytes, stream>>>(a);
  AKV_LAUNCH_CHECK("sa_kernel");
  if (a.splits > 1) {
    sa_join_kernel<D, DT><<<(uint32_t)(((int64_t)a.b.T * a.QH + 3) / 4), 256, 0, stream>>>(a);
    AKV_LAUNCH_CHECK("sa_join_kernel");
  }
  return AKV_OK;
}
// Query heads of a kv head in groups of at most 32 rows
static inline int sa_groups(int G) { return (G + 31) / 32; }
// Workgroups that share the keys of a tile: one token a sequence, and few of them, leave most CUs without a tile, and a CU takes in some 36 bytes a clock.
// Joining takes 4 us, so that it has to be for 1024 keys or more, and half of the CUs take in what memory gives.  32 heads on 8, blocks of 16, us with one
// workgroup and with 8 / units of 128: one token and 64 blocks 18.3 and 13.5, 128 blocks 28.4 and 14.7, 32 blocks 13.1 and 13.5; four tokens, 64 blocks, 18.7
// and 16.1; eight 20.8 and 19.4 (four workgroups a tile 21.0); sixteen 23.9 and, with two, 28.4.
static inline int sa_splits(int64_t T, int S, int QH, int KVH, int block_size, int k_sel) {
  if (T <= 0 || T > S || QH <= 0 || KVH <= 0 || block_size <= 0 || (int64_t)k_sel * ((block_size + 15) / 16) < 64) return 1;
  const int64_t units = T * KVH * sa_groups(QH / KVH);
  int splits = 1;
  while (splits < SA_SPLITS && 4 * splits * units <= ab_cus()) splits *= 2;
  return splits;
}
static inline size_t sa_sums(int64_t rows, int splits) { return akv_align256((size_t)rows * splits * 8); }
extern "C" size_t akv_sparse_attn_workspace_bytes(int64_t num_tokens, int num_seqs, int num_q_heads, int num_kv_heads, int d, int block_size, int num_selected) {
  const int splits = sa_splits(num_tokens, num_seqs, num_q_heads, num_kv_heads, block_size, num_selected);
  return splits == 1 || !ab_head_size(d) ? 0 : sa_sums(num_tokens * num_q_heads, splits) + (size_t)(num_tokens * num_q_heads) * splits * d * 4;
}

extern "C" int akv_sparse_attn(const void* query, int dtype, int64_t qs_tok, int64_t qs_head, const void* key_cache, int64_t ks_blk, int64_t ks_pos, int64_t ks_head, const void* value_cache,
                               int64_t vs_blk, int64_t vs_pos, int64_t vs_head, const void* block_tables, int bt_itype, int64_t bt_stride, const void* context_lens, int cl_itype,
                               const void* query_starts, int qs_itype, const int32_t* selected, int64_t ss_tok, int64_t ss_head, int num_selected, void* out, int64_t os_tok, int64_t os_head,
                               int zero_tail, int num_seqs, int64_t num_tokens, int num_q_heads, int num_kv_heads, int d, int block_size, int64_t num_blocks, int64_t max_blocks_per_seq,
                               float scale, void* workspace, size_t workspace_bytes, void* stream) {
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
  if (block_size == 1) ks_pos = vs_pos = 0;
  if (ks_pos < 0 || vs_pos < 0 || ks_pos > SA_MOST_STRIDE || vs_pos > SA_MOST_STRIDE) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: tokens of a block 2^27 elements apart", name);
  const size_t need = akv_sparse_attn_workspace_bytes(num_tokens, num_seqs, num_q_heads, num_kv_heads, d, block_size, num_selected);
  if (need && (!workspace || workspace_bytes < need || !ab_aligned(workspace, 256))) return akv_fail(AKV_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", name, need);
  sa_args a = {};
  a.b = ab_make(block_tables, bt_itype, bt_stride, context_lens, cl_itype, query_starts, qs_itype, num_seqs, num_tokens, block_size, num_blocks, max_blocks_per_seq);
  a.q = query; a.qs_tok = qs_tok; a.qs_head = qs_head;
  a.k = (const uint8_t*)key_cache; a.k_blk = 2 * ks_blk; a.k_pos = 2 * ks_pos; a.k_head = 2 * ks_head;
  a.v = (const uint8_t*)value_cache; a.v_blk = 2 * vs_blk; a.v_pos = 2 * vs_pos; a.v_head = 2 * vs_head;
  a.selected = selected; a.ss_tok = ss_tok; a.ss_head = ss_head; a.k_sel = num_selected;
  a.out = out; a.os_tok = os_tok; a.os_head = os_head;
  a.KVH = num_kv_heads; a.QH = num_q_heads; a.G = num_q_heads / num_kv_heads;
  a.HS = sa_groups(a.G);
  a.GC = (a.G + a.HS - 1) / a.HS;
  a.splits = sa_splits(num_tokens, num_seqs, num_q_heads, num_kv_heads, block_size, num_selected);
  a.part_ml = (float2*)workspace;
  a.part = (float*)((char*)workspace + sa_sums(num_tokens * num_q_heads, a.splits));
  a.tail = zero_tail; a.scale2 = scale * 1.44269504088896341f;
  const hipStream_t s = (hipStream_t)stream;
#define SA_CASE(DIM) if (d == DIM) return dtype == AKV_F16 ? sa_launch<DIM, AKV_F16>(a, s) : sa_launch<DIM, AKV_BF16>(a, s);
  SA_CASE(64) SA_CASE(128) SA_CASE(256)
#undef SA_CASE
  return AKV_ERR_UNSUPPORTED;
}
