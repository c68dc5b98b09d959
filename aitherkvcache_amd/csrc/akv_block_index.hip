// What a block of plain keys looks like from afar, and the blocks that a query reads by it.
//
//   update   per (block, kv head) the mean of the block's keys in 8 bits: m = sum k / n,  scale = max|m| (1 / 127),  code = rint(m (1 / max|m| 127)),
//            every operation on the mean rounded to float32
//   select   per (token, kv head) c_q = rint(q (1 / max|q| 127)) of the sum q of the group's queries; the score of a block is
//            (c_q . code) scale, and the best k are listed, the first and last blocks of the context before all others
//
// Which blocks are chosen hangs on the order of their scores, so these are made to come out the same however they are summed: means
// and sums of queries in 64 bits (sums of 16-bit numbers, exact unless their sizes are some 2^30 apart), products of whole numbers
// (v_mfma_i32_16x16x64_i8; below 127^2 x 256 < 2^24, a float32 number), and one float32 product with the scale.  Equal scores: the lower column.
#include "akv_batch.h"
#include "akv_device_once.h"

struct bi_args {
  ab_batch b;
  const uint8_t* k; int64_t k_blk, k_pos, k_head;    // bytes
  int8_t* codes; float* scales;                      // [blocks][KVH][D], [blocks][KVH]
  int KVH, each;
};

// ---- update -----------------------------------------------------------------------------------------------------------------------------
// A wavefront takes a block and kv head: D / 8 lanes a key, sixteen bytes each, 512 / D keys at a time, four steps on their way together.
// `each` workgroups a sequence take the table columns that its new tokens came to (without starts: all of them) in turn.
template <int D, int DT> __global__ __launch_bounds__(256) void bi_update_kernel(bi_args a) {
  constexpr int LANES = D / 8, KEYS = 64 / LANES, AHEAD = 4;
  const int lane = threadIdx.x & 63, head = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (head >= a.KVH) return;
  const int bs = a.b.block_size, seq = blockIdx.x / a.each;
  const int ctx = ab_ctx(a.b, seq);
  int64_t col = 0;
  if (a.b.starts) {
    const int n = ab_start(a.b, seq + 1) - ab_start(a.b, seq);
    if (n <= 0) return;
    col = (ctx > n ? ctx - n : 0) / bs;
  }
  const int mine = lane / LANES;
  for (col += blockIdx.x % a.each; col * bs < ctx; col += a.each) {
    const int count = (int)min((int64_t)bs, ctx - col * bs);
    const int64_t blk = ab_block(a.b, seq, col);
    const uint8_t* from = a.k + blk * a.k_blk + (int64_t)head * a.k_head + 16 * (lane % LANES);
    double sum[8] = {};
    for (int p0 = 0; p0 < count; p0 += KEYS * AHEAD) {
      ab_u4 v[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int p = p0 + KEYS * i + mine;
        v[i] = p < count ? *(const ab_u4*)(from + (int64_t)p * a.k_pos) : (ab_u4){0u, 0u, 0u, 0u};
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sum[2 * e] += (double)ab_math<DT>::low(v[i][e]);
          sum[2 * e + 1] += (double)ab_math<DT>::high(v[i][e]);
        }
    }
#pragma unroll
    for (int m = LANES; m < 64; m *= 2)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += __shfl_xor(sum[e], m, 64);
    float mean[8], top = 0.f;
    bool fine = true;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      mean[e] = (float)(sum[e] / (double)count);
      fine = fine && fabsf(mean[e]) < INFINITY;
      top = fmaxf(top, fabsf(mean[e]));
    }
#pragma unroll
    for (int m = 1; m < LANES; m *= 2) top = fmaxf(top, __shfl_xor(top, m, 64));
    // (a mean that is not finite, or nothing but zeros, or so small that its inverse is infinite: zeros)
    const float per = 1.f / top * 127.f;
    fine = __ballot(fine) == ~0ull && per < INFINITY;
    uint32_t c[2] = {0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e >> 2] |= (uint32_t)((int)(fine ? rintf(mean[e] * per) : 0.f) & 255) << (8 * (e & 3));
    const int64_t to = blk * a.KVH + head;
    if (lane < LANES) *(ab_u2*)(a.codes + to * D + 8 * lane) = (ab_u2){c[0], c[1]};
    if (lane == 0) a.scales[to] = fine ? top * (1.f / 127.f) : 0.f;
  }
}

extern "C" int akv_block_index_update(const void* key_cache, int dtype, int64_t ks_blk, int64_t ks_pos, int64_t ks_head, const void* block_tables, int bt_itype, int64_t bt_stride,
                                      const void* context_lens, int cl_itype, const void* query_starts, int qs_itype, int8_t* codes, float* scales, int num_seqs, int64_t num_tokens,
                                      int num_kv_heads, int d, int block_size, int64_t num_blocks, int64_t max_blocks_per_seq, void* stream) {
  const char* name = "akv_block_index_update";
  AKV_REQUIRE(akv_valid_dtype(dtype), "%s: bad dtype %d", name, dtype);
  const int rc = ab_check(name, block_tables, bt_itype, context_lens, cl_itype, query_starts, qs_itype, num_seqs, num_tokens, num_kv_heads, block_size, num_blocks, max_blocks_per_seq);
  if (rc) return rc;
  if (dtype == AKV_F32) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: float32 keys are not supported; use float16 or bfloat16", name);
  if (!ab_head_size(d)) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: head_dim %d; kernels are built for 64, 128 and 256", name, d);
  if (num_seqs == 0 || num_blocks == 0 || max_blocks_per_seq == 0 || (query_starts && num_tokens == 0)) return AKV_OK;
  AKV_REQUIRE(key_cache && codes && scales, "%s: null pointer", name);
  if (!ab_aligned(key_cache, 16) || ((ks_blk | ks_pos | ks_head) & 7)) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: rows must lie at multiples of 16 bytes", name);
  if (!ab_aligned(codes, 8)) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: codes must lie at multiples of 8 bytes", name);
  bi_args a = {};
  a.b = ab_make(block_tables, bt_itype, bt_stride, context_lens, cl_itype, query_starts, qs_itype, num_seqs, num_tokens, block_size, num_blocks, max_blocks_per_seq);
  a.k = (const uint8_t*)key_cache; a.k_blk = 2 * ks_blk; a.k_pos = 2 * ks_pos; a.k_head = 2 * ks_head;
  a.codes = codes; a.scales = scales; a.KVH = num_kv_heads;
  const int64_t rows = (num_kv_heads + 3) / 4;
  // (16 workgroups a CU have more than their share of the memory's latency to wait for)
  int64_t each = 16 * ab_cus() / (num_seqs * rows) + 1;
  if (each > max_blocks_per_seq) each = max_blocks_per_seq;
  if (rows > 65535 || each * num_seqs > 0x7fffffff) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: more than 2^18 kv heads", name);
  a.each = (int)each;
  const dim3 grid((uint32_t)(each * num_seqs), (uint32_t)rows);
  const hipStream_t s = (hipStream_t)stream;
#define BI_CASE(DIM)                                                              \
  if (d == DIM) {                                                                 \
    if (dtype == AKV_F16) bi_update_kernel<DIM, AKV_F16><<<grid, 256, 0, s>>>(a); \
    else bi_update_kernel<DIM, AKV_BF16><<<grid, 256, 0, s>>>(a);                 \
  }
  BI_CASE(64) BI_CASE(128) BI_CASE(256)
#undef BI_CASE
  AKV_LAUNCH_CHECK("bi_update_kernel");
  return AKV_OK;
}

// ---- select ------------------------------------------------------------------------------------------------------------------------------
struct bi_rank_args {
  ab_batch b;
  const void* q; int64_t qs_tok, qs_head;
  const int8_t* codes; const float* scales;
  float* scores;                        // [rows][columns], row (token - t0) x KVH + head
  int32_t* out;                         // [T][KVH][k]
  int KVH, G, k, sinks, recent;
  int t0, t1;                           // tokens of this launch
  int64_t columns;                      // floats of a row
  int span;                             // columns of a workgroup
};

// Sequence and position of a query token (wavefront-uniform); false: it is in no sequence, or stands before the first key.
__device__ __forceinline__ bool bi_token(const ab_batch& b, int token, int& seq, int& pos) {
  seq = ab_last(b.S, token, [&](int i) { return (int64_t)ab_start(b, i); });
  if (seq < 0) return false;
  const int s0 = ab_start(b, seq), s1 = ab_start(b, seq + 1);
  pos = ab_ctx(b, seq) - (s1 - token);
  return token >= s0 && token < s1 && pos >= 0;
}
// a group's queries in 8 bits, D / 64 coordinates of 64 lanes: coordinate D / 64 lane + i
template <int D, int DT> __device__ __forceinline__ void bi_quantize(const bi_rank_args& a, int token, int head, int8_t (&c)[D / 64]) {
  constexpr int N = D / 64;
  const int lane = threadIdx.x & 63;
  const uint16_t* q = (const uint16_t*)a.q + (int64_t)token * a.qs_tok + (int64_t)head * a.G * a.qs_head + N * lane;
  double sum[N] = {};
  for (int g = 0; g < a.G; ++g)
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] += (double)ab_math<DT>::low(q[(int64_t)g * a.qs_head + i]);
  float x[N], top = 0.f;
  bool fine = true;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] = (float)sum[i];
    fine = fine && fabsf(x[i]) < INFINITY;
    top = fmaxf(top, fabsf(x[i]));
  }
  top = akv_wave_max(top);
  const float per = 1.f / top * 127.f;
  fine = __ballot(fine) == ~0ull && per < INFINITY;
#pragma unroll
  for (int i = 0; i < N; ++i) c[i] = (int8_t)(int)(fine ? rintf(x[i] * per) : 0.f);
}
// order of scores as whole numbers, above 0 (a zero is a zero, whatever its sign)
__device__ __forceinline__ uint32_t bi_order(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// Scores of sixteen tokens of a sequence and `span` columns; tiles of tokens are numbered with gaps, floor(start_i / 16) + i + j.
template <int D, int DT> __global__ __launch_bounds__(256) void bi_scores_kernel(bi_rank_args a) {
  constexpr int KS = D / 64, ROW = D + 16;
  __shared__ __align__(16) int8_t qc[16 * ROW];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), head = blockIdx.y;
  const int64_t x = blockIdx.x;
  const int seq = ab_last(a.b.S, x, [&](int i) { return (int64_t)ab_start(a.b, i) / 16 + i; });
  if (seq < 0) return;
  const int s0 = ab_start(a.b, seq), s1 = ab_start(a.b, seq + 1);
  const int64_t j = x - (s0 / 16 + (int64_t)seq);
  const int64_t first = s0 + 16 * j;
  if (first >= s1 || first >= a.t1 || first + 16 <= a.t0) return;
  const int tokens = (int)min((int64_t)16, s1 - first), ctx = ab_ctx(a.b, seq);
  const int last = ctx - (s1 - (int)first) + tokens - 1;          // position of the last token
  if (last < 0) return;
  const int64_t c0 = (int64_t)blockIdx.z * a.span, c1 = min(c0 + a.span, (int64_t)last / a.b.block_size + 1);
  if (c0 >= c1) return;
  for (int t = wave; t < 16; t += 4) {
    int8_t c[KS] = {};
    if (t < tokens) bi_quantize<D, DT>(a, (int)first + t, head, c);
#pragma unroll
    for (int i = 0; i < KS; ++i) qc[t * ROW + KS * lane + i] = c[i];
  }
  __syncthreads();
  const int col = lane & 15, hq = lane >> 4;
  ab_i4 q[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) q[ks] = *(const ab_i4*)(qc + col * ROW + 64 * ks + 16 * hq);
  const int token = (int)first + col;
  float* to = a.scores + ((int64_t)(token - a.t0) * a.KVH + head) * a.columns;
  const bool store = col < tokens && token >= a.t0 && token < a.t1;
  for (int64_t c = c0 + 16 * wave; c < c1; c += 64) {
    const int64_t mine = min(c + col, c1 - 1);
    const int64_t at = ab_block(a.b, seq, mine) * a.KVH + head;
    const float scale = a.scales[at];
    ab_i4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const ab_i4*)(a.codes + at * D + 64 * ks + 16 * hq), q[ks], acc, 0, 0, 0);
    ab_f4 s;
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = akv_mul_rn((float)acc[i], __shfl(scale, 4 * hq + i, 64));
    if (store) *(ab_f4*)(to + c + 4 * hq) = s;         // (rows have room for whole tiles)
  }
}

// A wavefront lists the best k columns of a row: the k-th largest score by halving the range of its order, bit by bit, then the columns
// above it and the first ones that equal it, ascending.
__global__ __launch_bounds__(256) void bi_select_kernel(bi_rank_args a) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= (int64_t)(a.t1 - a.t0) * a.KVH) return;
  const int token = a.t0 + (int)(row / a.KVH);
  int32_t* out = a.out + ((int64_t)token * a.KVH + row % a.KVH) * a.k;
  int seq, pos, n = 0;
  if (bi_token(a.b, token, seq, pos)) n = pos / a.b.block_size + 1;
  const float* s = a.scores + row * a.columns;
  if (n <= a.k) {
    for (int i = lane; i < a.k; i += 64) out[i] = i < n ? i : -1;
    return;
  }
  const int recent = n - a.recent;
  auto order = [&](int i) { return i >= n ? 0u : i < a.sinks || i >= recent ? 0xffffffffu : bi_order(s[i]); };
  uint32_t t = 0u;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t c = t | 1u << bit;
    int count = 0;
    for (int i = lane; i - lane < n; i += 64) count += __popcll(__ballot(order(i) >= c));
    if (count >= a.k) t = c;
    if (count == a.k) break;
  }
  int above = 0;
  for (int i = lane; i - lane < n; i += 64) above += __popcll(__ballot(order(i) > t));
  int equal = a.k - above, at = 0;
  const uint64_t below = (1ull << lane) - 1;
  for (int i = lane; i - lane < n; i += 64) {
    const uint32_t o = order(i);
    const uint64_t tied = __ballot(o == t && i < n);
    const bool take = o > t || (o == t && i < n && __popcll(tied & below) < equal);
    const uint64_t taken = __ballot(take);
    if (take) out[at + __popcll(taken & below)] = i;
    at += __popcll(taken);
    equal -= min(equal, (int)__popcll(tied));
  }
}

// Sixteen tokens of a sequence and a kv head by one workgroup, scores and all: nothing goes to memory but the lists.
//
// A lane holds the scores of its token (lane % 16) and four columns of every sixteen, in registers as long as W x HELD tiles do, otherwise made
// anew for each of the passes.  The k-th largest score is found by a histogram over equal parts of the range of a row's scores (a
// part's number does not fall as the score rises, so whatever is rounded on the way the parts are in order), then among the scores of the one part in
// which the count passes k; where these are more than a wavefront can sort out (scores that are alike), by halving the range of all scores bit
// by bit.  Columns above it, and those that equal it, are marked in two bitmaps a token, from which the lists are written in order.
#define BI_PARTS 256
#define BI_CANDIDATES 128
struct bi_row {                         // of a token
  float lo, scale;                      // of the histogram: part = (score - lo) scale
  float threshold;
  int part, equal, candidates, found;       // the part in which the count passes k, how many of it are taken; how many scores at the threshold
};
template <int D, int DT, int W, int HELD> __global__ __launch_bounds__(64 * W) void bi_pick_kernel(bi_rank_args a) {
  constexpr int KS = D / 64, ROW = D + 16, T = 64 * W, BATCH = 2;
  __shared__ __align__(16) int8_t qc[16 * ROW];
  __shared__ int hist[16 * (BI_PARTS + 1)];
  __shared__ float cand[16 * BI_CANDIDATES];
  __shared__ float range[2][W][16];
  __shared__ bi_row rows[16];
  __shared__ int again;
  extern __shared__ uint32_t marks[];   // [16][words][2]: above, equal
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), head = blockIdx.x % a.KVH, col = lane & 15, hq = lane >> 4;
  const int64_t x = blockIdx.x / a.KVH;
  const int bs = a.b.block_size;
  // tiles of tokens are numbered with gaps, floor(start_i / 16) + i + j; sequence S: the rows behind the last
  const int seq = ab_last(a.b.S + 1, x, [&](int i) { return (int64_t)ab_start(a.b, i) / 16 + i; });
  if (x == 0) {                         // rows before the first sequence
    const int64_t front = (int64_t)ab_start(a.b, 0) * a.k;
    for (int64_t i = tid; i < front; i += T) a.out[(i / a.k * a.KVH + head) * a.k + i % a.k] = -1;
  }
  if (seq < 0) return;
  const int s0 = ab_start(a.b, seq), s1 = seq < a.b.S ? ab_start(a.b, seq + 1) : a.b.T;
  const int64_t first64 = s0 + 16 * (x - (s0 / 16 + (int64_t)seq));
  if (first64 >= s1) return;
  const int first = (int)first64, tokens = min(16, s1 - first);
  const int pos0 = seq < a.b.S ? ab_ctx(a.b, seq) - (s1 - first) : -tokens, last = pos0 + tokens - 1;
  const int columns = last < 0 ? 0 : last / bs + 1;       // up to the last token's own
  auto columns_of = [&](int t) { return pos0 + t < 0 ? 0 : (pos0 + t) / bs + 1; };
  // lists that take all there is
  const bool all = columns <= a.k;
  for (int t = wave; t < tokens; t += W) {
    const int n = columns_of(t);
    if (n > a.k) continue;
    int32_t* out = a.out + ((int64_t)(first + t) * a.KVH + head) * a.k;
    for (int i = lane; i < a.k; i += 64) out[i] = i < n ? i : -1;
  }
  if (all) return;

  for (int t = wave; t < 16; t += W) {
    int8_t c[KS] = {};
    if (t < tokens) bi_quantize<D, DT>(a, first + t, head, c);
#pragma unroll
    for (int i = 0; i < KS; ++i) qc[t * ROW + KS * lane + i] = c[i];
  }
  const int words = (columns + 31) / 32;
  for (int i = tid; i < 16 * (BI_PARTS + 1); i += T) hist[i] = 0;
  for (int i = tid; i < tokens * words * 2; i += T) marks[i] = 0u;
  if (tid == 0) again = 0;
  __syncthreads();
  ab_i4 q[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) q[ks] = *(const ab_i4*)(qc + col * ROW + 64 * ks + 16 * hq);
  // columns of the lane's token: from .. to - 1 are free to be chosen, the others of its n are listed anyway
  const int n = col < tokens ? columns_of(col) : 0;
  const int from = a.sinks, to = n > a.k ? n - a.recent : 0, need = a.k - a.sinks - a.recent;
  // scores of BATCH tiles of the wavefront, which takes tiles wave, wave + W, ...; -infinity where a column is not free
  const int tiles = (columns + 15) / 16;
  auto scores = [&](int tile0, ab_f4 (&s)[BATCH]) {
    int64_t at[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) at[i] = ab_block(a.b, seq, min(16 * (tile0 + W * i) + col, columns - 1)) * a.KVH + head;
    ab_i4 c[BATCH][KS];
    float scale[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) c[i][ks] = *(const ab_i4*)(a.codes + at[i] * D + 64 * ks + 16 * hq);
      scale[i] = a.scales[at[i]];
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      ab_i4 acc = {0, 0, 0, 0};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(c[i][ks], q[ks], acc, 0, 0, 0);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int cc = 16 * (tile0 + W * i) + 4 * hq + e;
        const float v = akv_mul_rn((float)acc[e], __shfl(scale[i], 4 * hq + e, 64));
        s[i][e] = cc >= from && cc < to ? v : -INFINITY;
      }
    }
  };
  const bool fits = tiles <= W * HELD;
  ab_f4 held[HELD];
  if (fits) {
#pragma unroll
    for (int i = 0; i < HELD; i += BATCH) {
      ab_f4 s[BATCH];
#pragma unroll
      for (int j = 0; j < BATCH; ++j) s[j] = (ab_f4)(-INFINITY);
      if (wave + W * i < tiles) scores(wave + W * i, s);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < BATCH; ++j) held[i + j] = s[j];
    }
  }
  // ---- passes over the scores.  (One loop with the pass as a variable: there is one copy of the code that makes scores anew.)
  enum { RANGE, PARTS, CANDIDATES, BITS, MARKS };
  float lo = INFINITY, hi = -INFINITY, my_lo = 0.f, my_scale = 0.f, threshold = INFINITY;
  int part = 0, count = 0, bit = 31, more = 0;
  int cq = 4 * hq;
  uint32_t order = 0u;                  // BITS: the threshold's, as far as it is known
  auto part_of = [&](float s) { return min(BI_PARTS - 1, (int)((s - my_lo) * my_scale)); };
  auto take = [&](int pass, int tile, const ab_f4& s) {
    if (pass == RANGE) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        lo = fminf(lo, s[e] == -INFINITY ? INFINITY : s[e]);
        hi = fmaxf(hi, s[e]);
      }
    } else if (pass == PARTS) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (s[e] != -INFINITY) atomicAdd(hist + col * (BI_PARTS + 1) + part_of(s[e]), 1);
    } else if (pass == CANDIDATES) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (s[e] != -INFINITY && part_of(s[e]) == part) {
          const int at = atomicAdd(&rows[col].candidates, 1);
          if (at < BI_CANDIDATES) cand[col * BI_CANDIDATES + at] = s[e];
        }
    } else if (pass == BITS) {
#pragma unroll
      for (int e = 0; e < 4; ++e) count += s[e] != -INFINITY && bi_order(s[e]) >= (order | 1u << bit);
    } else {
      uint32_t above = 0u, equal = 0u;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = 16 * tile + cq + e;
        above |= (uint32_t)(s[e] > threshold || (c < n && (c < from || c >= to))) << e;
        equal |= (uint32_t)(s[e] == threshold) << e;
      }
      const int shift = 16 * (tile & 1) + cq;
      uint32_t* m = marks + (col * words + (tile >> 1)) * 2;
      if (above) atomicOr(m, above << shift);
      if (equal) atomicOr(m + 1, equal << shift);
    }
  };
  int pass = need > 0 ? RANGE : MARKS;
#pragma unroll 1
  for (;;) {
    // (what a pass makes of a score is not made before the loop and kept: registers hold the scores)
    asm volatile("" : "+v"(cq));
#pragma unroll
    for (int i = 0; i < HELD; ++i) asm volatile("" : "+v"(held[i]));
    if (fits) {
#define BI_PASS(P)                              \
  case P:                                       \
    _Pragma("unroll") for (int i = 0; i < HELD; ++i) \
        if (wave + W * i < tiles) take(P, wave + W * i, held[i]); \
    break;
      switch (pass) { BI_PASS(RANGE) BI_PASS(PARTS) BI_PASS(CANDIDATES) BI_PASS(BITS) BI_PASS(MARKS) }
#undef BI_PASS
    } else {
#pragma unroll 1
      for (int tile = wave; tile < tiles; tile += W * BATCH) {
        ab_f4 s[BATCH];
        scores(tile, s);
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
          if (tile + W * i < tiles) take(pass, tile + W * i, s[i]);
      }
    }
    if (pass == MARKS) break;
    if (pass == RANGE) {
      lo = -akv_rows_max(-lo);
      hi = akv_rows_max(hi);
      if (hq == 0) {
        range[0][wave][col] = lo;
        range[1][wave][col] = hi;
      }
      __syncthreads();
      if (tid < 16) {
        float l = INFINITY, h = -INFINITY;
        for (int w = 0; w < W; ++w) {
          l = fminf(l, range[0][w][tid]);
          h = fmaxf(h, range[1][w][tid]);
        }
        const float scale = BI_PARTS / (h - l);
        rows[tid].lo = l;
        rows[tid].scale = scale < INFINITY ? scale : 0.f;      // (scores that are all alike, or nearly: one part; and none where h < l)
        rows[tid].candidates = 0;
      }
      __syncthreads();
      my_lo = rows[col].lo;
      my_scale = rows[col].scale;
      pass = PARTS;
    } else if (pass == PARTS) {
      __syncthreads();
      for (int t = wave; t < tokens; t += W) {
        // a lane four parts, the first lane the uppermost
        const int* h = hist + t * (BI_PARTS + 1) + BI_PARTS - 4 - 4 * lane;
        const int c[4] = {h[3], h[2], h[1], h[0]}, sum = c[0] + c[1] + c[2] + c[3], inc = akv_wave_inclusive_scan(sum);
        int before = inc - sum;
        if (before < need && need <= inc) {
          int i = 0;
#pragma unroll
          for (int j = 0; j < 3; ++j)
            if (i == j && before + c[j] < need) before += c[j], ++i;
          rows[t].part = BI_PARTS - 1 - 4 * lane - i;
          rows[t].equal = need - before;          // of that part
        }
      }
      __syncthreads();
      part = rows[col].part;
      pass = CANDIDATES;
    } else if (pass == CANDIDATES) {
      __syncthreads();
      for (int t = wave; t < tokens; t += W) {
        const int have = rows[t].candidates, want = rows[t].equal;
        if (columns_of(t) <= a.k) continue;
        if (have > BI_CANDIDATES) {
          if (lane == 0) again = 1;
          continue;
        }
        const float* c = cand + t * BI_CANDIDATES;
        for (int i0 = 0; i0 < have; i0 += 64) {
          const float mine = c[min(i0 + lane, have - 1)];
          int above = 0, same = 0;
          for (int i = 0; i < have; ++i) {
            above += c[i] > mine;
            same += c[i] == mine;
          }
          if (above < want && want <= above + same) {       // (lanes of one value write the same)
            rows[t].threshold = mine;
            rows[t].found = want - above;
          }
        }
      }
      __syncthreads();
      pass = again ? BITS : MARKS;
    } else {
      count += akv_lane_xor<16>(count);
      count += akv_lane_xor<32>(count);
      int* sums = hist + (bit & 1) * W * 16;
      __syncthreads();
      if (hq == 0) sums[wave * 16 + col] = count;
      __syncthreads();
      int total = 0;
      for (int w = 0; w < W; ++w) total += sums[w * 16 + col];
      if (total >= need) order |= 1u << bit;
      else more = total;                // above the threshold, in the end
      count = 0;
      if (--bit < 0) {
        if (n > a.k && rows[col].candidates > BI_CANDIDATES && wave == 0 && hq == 0) {
          rows[col].threshold = __uint_as_float(order ^ ((order >> 31) ? 0x80000000u : 0xffffffffu));
          rows[col].found = need - more;
        }
        __syncthreads();
        pass = MARKS;
      }
    }
    if (pass == MARKS && n > a.k) threshold = rows[col].threshold;
  }
  __syncthreads();
  for (int t = wave; t < tokens; t += W) {
    if (columns_of(t) <= a.k) continue;
    int32_t* out = a.out + ((int64_t)(first + t) * a.KVH + head) * a.k;
    int tied = need > 0 ? rows[t].found : 0, at = 0;
    for (int w0 = 0; w0 < words; w0 += 64) {
      const int w = w0 + lane;
      uint32_t take = w < words ? marks[(t * words + w) * 2] : 0u, same = w < words ? marks[(t * words + w) * 2 + 1] : 0u;
      const int s = __popc(same), s_inc = akv_wave_inclusive_scan(s);
      for (int left = min(s, tied - (s_inc - s)); left > 0; --left) {
        take |= same & -same;
        same &= same - 1;
      }
      const int c = __popc(take), c_inc = akv_wave_inclusive_scan(c);
      int to_at = at + c_inc - c;
      for (; take; take &= take - 1) out[to_at++] = 32 * w + __ffs(take) - 1;
      tied -= __builtin_amdgcn_readlane(s_inc, 63);
      at += __builtin_amdgcn_readlane(c_inc, 63);
    }
  }
}

// Wider tables go the long way over scores in memory.
#define BI_WIDE 16384
template <int D, int DT> static int bi_pick(const bi_rank_args& a, int64_t max_blocks, hipStream_t stream) {
  const int64_t units = ((int64_t)a.b.T / 16 + a.b.S + 1) * a.KVH;
  const int bytes = (int)(16 * ((max_blocks + 31) / 32) * 8);
  if (units > 0x7fffffff) return akv_fail(AKV_ERR_UNSUPPORTED, "akv_block_index_select: more than 2^31 rows");
  int dev = 0;
  AKV_HIP(hipGetDevice(&dev));
  static akv_device_once once;
  if (const int rc = once(dev, [&]() -> int {
        const int rc8 = ab_lds((const void*)bi_pick_kernel<D, DT, 16, 8>, 16 * BI_WIDE / 4);
        return rc8 ? rc8 : ab_lds((const void*)bi_pick_kernel<D, DT, 16, 14>, 16 * BI_WIDE / 4);
      }))
    return rc;
  if (max_blocks <= 16 * 16 * 8) bi_pick_kernel<D, DT, 16, 8><<<(uint32_t)units, 1024, bytes, stream>>>(a);
  else bi_pick_kernel<D, DT, 16, 14><<<(uint32_t)units, 1024, bytes, stream>>>(a);
  AKV_LAUNCH_CHECK("bi_pick_kernel");
  return AKV_OK;
}

// scores of so many bytes at most are held at a time
#define BI_SCRATCH (256ll << 20)
static inline int64_t bi_columns(int64_t max_blocks) { return (max_blocks + 15) / 16 * 16; }
static inline int64_t bi_tokens_at_once(int64_t T, int KVH, int64_t max_blocks) {
  const int64_t most = BI_SCRATCH / (4 * bi_columns(max_blocks) * KVH);
  return most >= T ? T : most > 16 ? most : 16;
}
extern "C" size_t akv_block_index_select_workspace_bytes(int64_t num_tokens, int num_kv_heads, int64_t max_blocks_per_seq) {
  if (num_tokens <= 0 || num_kv_heads <= 0 || max_blocks_per_seq <= BI_WIDE || max_blocks_per_seq > 0x7fffffff) return 0;
  return (size_t)(4 * bi_columns(max_blocks_per_seq) * num_kv_heads * bi_tokens_at_once(num_tokens, num_kv_heads, max_blocks_per_seq));
}

extern "C" int akv_block_index_select(const void* query, int dtype, int64_t qs_tok, int64_t qs_head, const int8_t* codes, const float* scales, const void* block_tables, int bt_itype,
                                      int64_t bt_stride, const void* context_lens, int cl_itype, const void* query_starts, int qs_itype, int32_t* selected, int num_seqs,
                                      int64_t num_tokens, int num_q_heads, int num_kv_heads, int d, int block_size, int64_t num_blocks, int64_t max_blocks_per_seq, int num_selected,
                                      int num_sink_blocks, int num_recent_blocks, void* workspace, size_t workspace_bytes, void* stream) {
  const char* name = "akv_block_index_select";
  AKV_REQUIRE(akv_valid_dtype(dtype), "%s: bad dtype %d", name, dtype);
  const int rc = ab_check(name, block_tables, bt_itype, context_lens, cl_itype, query_starts, qs_itype, num_seqs, num_tokens, num_kv_heads, block_size, num_blocks, max_blocks_per_seq);
  if (rc) return rc;
  AKV_REQUIRE(num_q_heads > 0 && num_q_heads % num_kv_heads == 0, "%s: %d query heads on %d kv heads", name, num_q_heads, num_kv_heads);
  AKV_REQUIRE(num_selected > 0 && num_sink_blocks >= 0 && num_recent_blocks >= 1 && num_sink_blocks <= num_selected - num_recent_blocks,
              "%s: %d blocks cannot hold the first %d and last %d (at least 1)", name, num_selected, num_sink_blocks, num_recent_blocks);
  if (dtype == AKV_F32) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: float32 queries are not supported; use float16 or bfloat16", name);
  if (!ab_head_size(d)) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: head_dim %d; kernels are built for 64, 128 and 256", name, d);
  if (num_tokens == 0) return AKV_OK;
  AKV_REQUIRE(query && query_starts && selected, "%s: null pointer", name);
  AKV_REQUIRE(num_blocks == 0 || (codes && scales), "%s: null pointer", name);
  if (num_kv_heads > 65535) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: more than 65535 kv heads", name);
  if (!ab_aligned(query, 16) || ((qs_tok | qs_head) & 7)) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: queries must lie at multiples of 16 bytes", name);
  if (!ab_aligned(codes, 16)) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: codes must lie at multiples of 16 bytes", name);
  const size_t need = akv_block_index_select_workspace_bytes(num_tokens, num_kv_heads, max_blocks_per_seq);
  if (need && (!workspace || workspace_bytes < need || !ab_aligned(workspace, 256))) return akv_fail(AKV_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", name, need);
  bi_rank_args a = {};
  a.b = ab_make(block_tables, bt_itype, bt_stride, context_lens, cl_itype, query_starts, qs_itype, num_seqs, num_tokens, block_size, num_blocks, max_blocks_per_seq);
  a.q = query; a.qs_tok = qs_tok; a.qs_head = qs_head;
  a.codes = codes; a.scales = scales; a.scores = (float*)workspace; a.out = selected;
  a.KVH = num_kv_heads; a.G = num_q_heads / num_kv_heads; a.k = num_selected; a.sinks = num_sink_blocks; a.recent = num_recent_blocks;
  a.columns = bi_columns(max_blocks_per_seq);
  const hipStream_t s = (hipStream_t)stream;
  if (max_blocks_per_seq <= BI_WIDE) {
#define BI_CASE(DIM) if (d == DIM) return dtype == AKV_F16 ? bi_pick<DIM, AKV_F16>(a, max_blocks_per_seq, s) : bi_pick<DIM, AKV_BF16>(a, max_blocks_per_seq, s);
    BI_CASE(64) BI_CASE(128) BI_CASE(256)
#undef BI_CASE
  }
  const int64_t at_once = max_blocks_per_seq > 0 ? bi_tokens_at_once(num_tokens, num_kv_heads, max_blocks_per_seq) : num_tokens;
  const int64_t tiles = num_tokens / 16 + num_seqs;
  // columns of a workgroup: at least 64, and no more workgroups than some rounds of the chip
  int64_t spans = 8 * ab_cus() / (tiles * num_kv_heads > 0 ? tiles * num_kv_heads : 1);
  spans = spans < 1 ? 1 : spans > a.columns / 64 + 1 ? a.columns / 64 + 1 : spans;
  a.span = (int)(((a.columns + spans - 1) / spans + 63) / 64 * 64);
  if (a.span < 64) a.span = 64;
  for (int64_t t = 0; t < num_tokens; t += at_once) {
    a.t0 = (int)t;
    a.t1 = (int)(t + at_once < num_tokens ? t + at_once : num_tokens);
    if (a.b.max_blocks > 0 && num_seqs > 0) {
      const dim3 grid((uint32_t)tiles, (uint32_t)num_kv_heads, (uint32_t)((a.columns + a.span - 1) / a.span));
#define BI_CASE(DIM)                                                              \
  if (d == DIM) {                                                                 \
    if (dtype == AKV_F16) bi_scores_kernel<DIM, AKV_F16><<<grid, 256, 0, s>>>(a); \
    else bi_scores_kernel<DIM, AKV_BF16><<<grid, 256, 0, s>>>(a);                 \
  }
      BI_CASE(64) BI_CASE(128) BI_CASE(256)
#undef BI_CASE
      AKV_LAUNCH_CHECK("bi_scores_kernel");
    }
    const int64_t rows = (int64_t)(a.t1 - a.t0) * num_kv_heads;
    bi_select_kernel<<<(uint32_t)((rows + 3) / 4), 256, 0, s>>>(a);
    AKV_LAUNCH_CHECK("bi_select_kernel");
  }
  return AKV_OK;
}
