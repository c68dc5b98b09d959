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
// 8192 tokens of 8 heads of 128 take 7.8 us, 2.2 TB/s: half of it are three trips to memory, lengths, table and keys, one after the other.
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
  typedef uint16_t raw __attribute__((ext_vector_type(N < 2 ? 2 : N)));
  const uint16_t* q = (const uint16_t*)a.q + (int64_t)token * a.qs_tok + (int64_t)head * a.G * a.qs_head + N * lane;
  double sum[N] = {};
  for (int g0 = 0; g0 < a.G; g0 += 4) {          // four heads are requested together
    uint16_t v[4][N];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const uint16_t* p = q + (int64_t)min(g0 + g, a.G - 1) * a.qs_head;
      if constexpr (N == 1) v[g][0] = *p;
      else {
        const raw r = *(const raw*)p;
#pragma unroll
        for (int i = 0; i < N; ++i) v[g][i] = r[i];
      }
    }
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int i = 0; i < N; ++i) sum[i] += g0 + g < a.G ? (double)ab_math<DT>::low(v[g][i]) : 0.0;
  }
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
// A lane holds the scores of one column of every sixteen and four of the tokens, in registers where tables have no more than W x HELD tiles;
// HELD = 0: made anew for each of the passes.  A column that is not free to be chosen has a NaN in its place, since a score may be any other number: one past the
// largest float32 number is infinite.  The k-th largest score of a token is found by a histogram over equal parts of the range of its scores (a part's
// number does not fall as the score rises, so whatever is rounded on the way the parts are in order), then among the scores of the one part in
// which the count passes k; where these are more than fit (scores that are alike), by halving the range of all scores bit by
// bit.  Columns above it, and those that equal it, are marked in two bitmaps a token, from which the lists are written in order.
//
// The vector unit bounds it: a wavefront's instruction takes four clocks, and with the scores of a lane for one token and four columns, their
// scales from other lanes, a hundred of them a score cost 98 us for 2048 tokens over 1920 blocks, where this takes 60 (vector unit 62 % of clocks, LDS
// 32 %).  One token of each of 16 sequences, up to 2560 blocks, takes 19 us: a workgroup a head reads 320 KB of codes at the 36 bytes a clock that a CU takes
// in, and waits for its code.  (A kernel for one token, with orders in LDS and products four at a time, took as long.)
#define BI_PARTS 256
#define BI_CANDIDATES 64
struct bi_row {                         // of a token
  float scale, shift;                   // of the histogram: part = score x scale + shift
  int part, taken, candidates, tied;    // the part in which the count passes k, how many of it are taken; scores in it; taken ones of those marked as equal
  uint32_t order;                       // of the threshold, as far as it is known, where the count goes bit by bit
  float threshold;
};
template <int D, int DT, int W, int HELD> __global__ __launch_bounds__(64 * W, 4) void bi_pick_kernel(bi_rank_args a) {
  constexpr int KS = D / 64, ROW = D + 16, T = 64 * W, HIST = BI_PARTS + 1;
  constexpr int LANES = D / 16, AT_ONCE = 64 / LANES, LOADS = 16 / AT_ONCE;      // of a tile's codes: lanes a row, rows a load, loads
  constexpr int BATCH = 4, STAGED = D == 256 ? 1 : 2;                            // tiles looked up together; tiles in LDS together
  static_assert(HELD % 2 == 0 && (W == 16 || W == 8), "whole batches; a wavefront a token");
  __shared__ __align__(16) int8_t qc[16 * ROW];
  __shared__ int hist[16 * HIST];
  __shared__ float2 cand[16 * BI_CANDIDATES];      // score, column
  __shared__ float range[2][W][16];
  __shared__ bi_row rows[16];
  __shared__ int again;
  __shared__ __align__(16) uint8_t stage[W][STAGED * 16 * D];
  extern __shared__ uint16_t marks[];   // [16][2 words][2]: columns above, and those at, the threshold
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
  const int pos0 = seq < a.b.S ? ab_ctx(a.b, seq) - (s1 - first) : -tokens;
  auto columns_of = [&](int t) { return t >= tokens || pos0 + t < 0 ? 0 : (pos0 + t) / bs + 1; };
  const int columns = columns_of(tokens - 1), need = a.k - a.sinks - a.recent;      // up to the last token's own; those that are chosen

  // ---- lists that take all there is; queries in 8 bits
  auto listed = [&](int t) { return columns_of(t) > a.k; };      // (the others' lists are written here)
  auto list_of = [&](int t) { return a.out + ((int64_t)(first + t) * a.KVH + head) * a.k; };
  for (int t = wave; t < tokens; t += W) {
    const int n = columns_of(t);
    if (n > a.k) continue;
    int32_t* out = list_of(t);
    for (int i = lane; i < a.k; i += 64) out[i] = i < n ? i : -1;
  }
  if (columns <= a.k) return;
#pragma unroll
  for (int t = wave; t < 16; t += W) {
    int8_t c[KS] = {};
    if (listed(t)) bi_quantize<D, DT>(a, first + t, head, c);
#pragma unroll
    for (int i = 0; i < KS; ++i) qc[t * ROW + KS * lane + i] = c[i];
  }
  for (int i = tid; i < 16 * HIST; i += T) hist[i] = 0;
  if (tid == 0) again = 0;
  __syncthreads();

  // ---- scores
  ab_i4 q[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) q[ks] = *(const ab_i4*)(qc + col * ROW + 64 * ks + 16 * hq);
  const int tiles = (columns + 15) / 16, half_words = 2 * ((columns + 31) / 32);
  // columns sinks .. to - 1 of a token are free to be chosen; whole tiles that are free for every token need no mask
  int shortest = 0;                     // of the tokens that choose, the first
  while (columns_of(shortest) <= a.k) ++shortest;
  const int free_tiles = (columns_of(shortest) - a.recent) / 16;
  float lo[4], hi[4];
  int free_to[4];                       // of the lane's tokens; 0: one that does not choose
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    lo[e] = INFINITY, hi[e] = -INFINITY;
    const int m = columns_of(4 * hq + e);
    free_to[e] = m > a.k ? m - a.recent : 0;
  }
  // Codes go from memory to LDS row by row, sixteen bytes a lane side by side, and from there to the operand: memory serves four lanes a
  // clock where they read one line, and in the operand's order, a row a lane, one (120 tiles 25000 clocks).
  const int8_t* const codes = a.codes + (int64_t)head * D + 16 * (lane % LANES);
  uint8_t* const st = stage[wave];
  const int my_row = lane / LANES;
  // entries of the tiles tile0, tile0 + W, ... + (BATCH - 1) W: of tile lane / 16, column lane % 16
  auto look = [&](int tile0) { return ab_look(a.b, seq, min(16 * (tile0 + W * hq) + col, columns - 1)); };
  struct rows_of_codes { ab_u4 v[STAGED][LOADS]; };
  auto request = [&](int blk, int i0, rows_of_codes& r) {      // tiles i0 .. i0 + STAGED - 1 of a batch
#pragma unroll
    for (int i = 0; i < STAGED; ++i)
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int from = __shfl(blk, 16 * (i0 + i) + AT_ONCE * j + my_row, 64);
        r.v[i][j] = *(const ab_u4*)(codes + (int64_t)from * a.KVH * D);
      }
  };
  auto to_stage = [&](const rows_of_codes& c) {
    akv_wave_sync();                    // (what was there has been read)
#pragma unroll
    for (int i = 0; i < STAGED; ++i)
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int r = AT_ONCE * j + my_row;
        *(ab_u4*)(st + (16 * i + r) * D + 16 * ((lane % LANES) ^ (r & (LANES < 8 ? LANES - 1 : 7)))) = c.v[i][j];
      }
    akv_wave_sync();
  };
  auto score = [&](int tile, int i0, int i, float scale, ab_f4& x) {
    ab_i4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(q[ks], *(const ab_i4*)(st + (16 * i + col) * D + 16 * ((4 * ks + hq) ^ (col & (LANES < 8 ? LANES - 1 : 7)))), acc, 0, 0, 0);
    const float f = __shfl(scale, 16 * (i0 + i) + col, 64);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = akv_mul_rn((float)acc[e], f);
    if (16 * tile < a.sinks || tile >= free_tiles) {
      const int cc = 16 * tile + col;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool free = cc >= a.sinks && cc < free_to[e];
        lo[e] = fminf(lo[e], free ? x[e] : INFINITY);
        x[e] = free ? x[e] : NAN;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) lo[e] = fminf(lo[e], x[e]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) hi[e] = fmaxf(hi[e], x[e]);
  };
  constexpr bool fits = HELD > 0;       // (the tables' width says so)
  ab_f4 held[HELD > 0 ? HELD : 1];
  if constexpr (fits) {
    constexpr int BATCHES = (HELD + BATCH - 1) / BATCH;
    // entries are all requested before the first is needed, then scales; codes a step ahead
    ab_entry entry[BATCHES];
    int blk[BATCHES];
    float scale[BATCHES];
#pragma unroll
    for (int i = 0; i < BATCHES; ++i) entry[i] = look(wave + W * BATCH * i);
#pragma unroll
    for (int i = 0; i < BATCHES; ++i) {
      blk[i] = (int)ab_block(a.b, entry[i]);
      scale[i] = a.scales[(int64_t)blk[i] * a.KVH + head];
    }
    rows_of_codes c[2];
    request(blk[0], 0, c[0]);
#pragma unroll
    for (int i = 0; i < HELD; i += STAGED) {
      held[i] = (ab_f4)(NAN);
      if (STAGED == 2) held[i + 1] = (ab_f4)(NAN);
      if (wave + W * i >= tiles) continue;
      const int next = i + STAGED < HELD ? i + STAGED : i;
      if (next > i) request(blk[next / BATCH], next % BATCH, c[next / STAGED & 1]);
      to_stage(c[i / STAGED & 1]);
#pragma unroll
      for (int j = 0; j < STAGED; ++j) score(wave + W * (i + j), i % BATCH, j, scale[i / BATCH], held[i + j]);
    }
  }

  // ---- passes over the scores.  (One loop with the pass as a variable: there is one copy of the code that makes scores anew.)
  enum { RANGE, PARTS, CANDIDATES, BITS, MARKS };
  float scale[4], shift[4];
  int part[4], bit = 31;
  // (the median of a NaN and two numbers is the lesser one: what is not free has the lowest part, and so has an infinite score, whose token has a scale of 0 and one part)
  auto part_of = [&](float s, int e) { return (int)__builtin_amdgcn_fmed3f(fmaf(s, scale[e], shift[e]), 0.f, BI_PARTS - 1.f); };
  int row0 = 4 * hq, my_col = col;      // the lane's first token, its column of a tile
  // sixteen columns of token 4 hq + e: a lane of the token writes their marks
  auto mark = [&](int tile, int e, uint64_t lanes, int which) {
    const uint32_t mine = hq < 2 ? (uint32_t)lanes : (uint32_t)(lanes >> 32);
    marks[(2 * (row0 + e) + which) * half_words + tile] = (uint16_t)(mine >> (16 * (hq & 1)));
  };
  auto take = [&](int pass, int tile, const ab_f4& s) {
    if (pass == PARTS) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        // (what is not free counts in the lowest part, above which no count starts)
        if (free_to[e] > 0) atomicAdd(hist + (row0 + e) * HIST + part_of(s[e], e), 1);
    } else if (pass == CANDIDATES) {
      uint64_t above[4] = {};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int p = part_of(s[e], e);
        above[e] = __ballot(p > part[e]);
        if (p == part[e] && s[e] == s[e]) {
          const int at = atomicAdd(&rows[row0 + e].candidates, 1);
          if (at < BI_CANDIDATES) cand[(row0 + e) * BI_CANDIDATES + at] = make_float2(s[e], __int_as_float(16 * tile + my_col));
        }
      }
      if (my_col == 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          mark(tile, e, above[e], 0);
      }
    } else if (pass == BITS) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (s[e] == s[e] && bi_order(s[e]) >= (rows[row0 + e].order | 1u << bit)) atomicAdd(hist + row0 + e, 1);
    } else if (pass == MARKS) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float threshold = rows[row0 + e].threshold;
        const uint64_t above = __ballot(s[e] > threshold), equal = __ballot(s[e] == threshold);
        if (my_col == 0 && rows[row0 + e].candidates > BI_CANDIDATES) {
          mark(tile, e, above, 0);
          mark(tile, e, equal, 1);
        }
      }
    }
  };
  int pass = fits ? PARTS : RANGE;      // (the range of scores that are held is known)
#pragma unroll 1
  for (;;) {
    if (pass == PARTS) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float l = lo[e], h = hi[e];
        l = fminf(l, akv_lane_xor<1>(l)); l = fminf(l, akv_lane_xor<2>(l)); l = fminf(l, akv_lane_xor<4>(l)); l = fminf(l, akv_lane_xor<8>(l));
        h = fmaxf(h, akv_lane_xor<1>(h)); h = fmaxf(h, akv_lane_xor<2>(h)); h = fmaxf(h, akv_lane_xor<4>(h)); h = fmaxf(h, akv_lane_xor<8>(h));
        if (col == 0) {
          range[0][wave][4 * hq + e] = l;
          range[1][wave][4 * hq + e] = h;
        }
      }
      __syncthreads();
      if (tid < 16) {
        float l = INFINITY, h = -INFINITY;
        for (int w = 0; w < W; ++w) {
          l = fminf(l, range[0][w][tid]);
          h = fmaxf(h, range[1][w][tid]);
        }
        const float f = BI_PARTS / (h - l);
        const bool fine = f < INFINITY && fabsf(l * f) < INFINITY;      // (scores that are all alike, or nearly, or infinite: one part; and none where h < l)
        rows[tid].scale = fine ? f : 0.f;
        rows[tid].shift = fine ? -l * f : 0.f;
        rows[tid].candidates = rows[tid].tied = 0;
        rows[tid].part = BI_PARTS;
      }
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        scale[e] = rows[4 * hq + e].scale;
        shift[e] = rows[4 * hq + e].shift;
      }
    }
    // (what a pass makes of a score is not made before the loop and kept: registers hold the scores)
#pragma unroll
    for (int i = 0; i < HELD; ++i) asm volatile("" : "+v"(held[i]));
    asm volatile("" : "+v"(row0), "+v"(my_col));
    if constexpr (fits) {
#define BI_PASS(P)                                   \
  case P:                                            \
    _Pragma("unroll") for (int i = 0; i < HELD; ++i) \
        if (wave + W * i < tiles) take(P, wave + W * i, held[i]); \
    break;
      switch (pass) { BI_PASS(PARTS) BI_PASS(CANDIDATES) BI_PASS(BITS) BI_PASS(MARKS) }
#undef BI_PASS
    } else {
#pragma unroll 1
      for (int tile = wave; tile < tiles; tile += W * BATCH) {
        const int blk = (int)ab_block(a.b, look(tile));
        const float scale = a.scales[(int64_t)blk * a.KVH + head];
        rows_of_codes c[2];
        request(blk, 0, c[0]);
#pragma unroll
        for (int i = 0; i < BATCH; i += STAGED) {
          if (i + STAGED < BATCH) request(blk, i + STAGED, c[(i / STAGED + 1) & 1]);
          to_stage(c[i / STAGED & 1]);
#pragma unroll
          for (int j = 0; j < STAGED; ++j) {
            ab_f4 s;
            score(tile + W * (i + j), i, j, scale, s);
            if (tile + W * (i + j) < tiles) take(pass, tile + W * (i + j), s);
          }
        }
      }
    }
    __syncthreads();
    if (pass == MARKS) break;
    if (pass == RANGE) {
      pass = PARTS;
    } else if (pass == PARTS) {
      for (int t = wave; t < 16; t += W) {
        if (!listed(t) || need == 0) continue;
        // a lane four parts, the first lane the uppermost
        const int* h = hist + t * HIST + BI_PARTS - 4 - 4 * lane;
        const int c[4] = {h[3], h[2], h[1], h[0]}, sum = c[0] + c[1] + c[2] + c[3], inc = akv_wave_inclusive_scan(sum);
        int before = inc - sum;
        if (before < need && need <= inc) {
          int i = 0;
#pragma unroll
          for (int j = 0; j < 3; ++j)
            if (i == j && before + c[j] < need) before += c[j], ++i;
          rows[t].part = BI_PARTS - 1 - 4 * lane - i;
          rows[t].taken = need - before;
        }
      }
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 4; ++e) part[e] = rows[4 * hq + e].part;
      pass = CANDIDATES;
    } else if (pass == CANDIDATES) {
      for (int t = wave; t < 16; t += W) {
        if (!listed(t) || need == 0) continue;
        const int have = rows[t].candidates, want = rows[t].taken;
        if (have > BI_CANDIDATES) {
          if (lane == 0) again = 1;
        } else {
          // rank among them, of equal ones the lower column first
          const float2* c = cand + t * BI_CANDIDATES;
          for (int i0 = 0; i0 < have; i0 += 64) {
            const float2 mine = c[min(i0 + lane, have - 1)];
            const int mine_col = __float_as_int(mine.y);
            int above = 0;
            for (int i = 0; i < have; ++i) above += c[i].x > mine.x || (c[i].x == mine.x && __float_as_int(c[i].y) < mine_col);
            if (above < want && i0 + lane < have) atomicOr((uint32_t*)marks + t * half_words + (mine_col >> 5), 1u << (mine_col & 31));
          }
        }
      }
      __syncthreads();
      if (!again) break;
      if (tid < 16) {
        rows[tid].order = 0u;
        hist[tid] = 0;
      }
      __syncthreads();
      pass = BITS;
    } else {
      // (the counts of all tokens; those that have their marks let them pass)
      if (tid < 16) {
        bi_row& r = rows[tid];
        const int c = hist[tid];
        if (c >= need) r.order |= 1u << bit;
        else r.tied = need - c;         // not above the threshold, in the end
        if (bit == 0) r.threshold = __uint_as_float(r.order ^ ((r.order >> 31) ? 0x80000000u : 0xffffffffu));
        if (bit == 0 && r.candidates <= BI_CANDIDATES) r.tied = 0;
        hist[tid] = 0;
      }
      __syncthreads();
      if (--bit < 0) pass = MARKS;
    }
  }
  // ---- lists: what is listed anyway, what is marked, and the first of those that equal the threshold
  for (int t = wave; t < tokens; t += W) {
    if (!listed(t)) continue;
    const int n = columns_of(t);
    int32_t* out = list_of(t);
    const uint32_t* above = (const uint32_t*)marks + t * half_words;      // (half_words words a token: two bitmaps)
    const uint32_t* equal = above + half_words / 2;
    int tied = rows[t].tied, at = 0;
    for (int w0 = 0; 32 * w0 < n; w0 += 64) {
      const int w = w0 + lane, c0 = 32 * w;
      // bits below column c of the word
      auto below = [&](int c) { return c <= c0 ? 0u : c - c0 >= 32 ? ~0u : (1u << (c - c0)) - 1; };
      const uint32_t free = below(n - a.recent) & ~below(a.sinks);
      uint32_t take = below(n) & ~free, same = 0u;
      if (need > 0 && free) {
        take |= above[w] & free;
        if (tied > 0) same = equal[w] & free;
      }
      if (tied > 0) {
        const int s = __popc(same), inc = akv_wave_inclusive_scan(s);
        for (int left = min(s, tied - (inc - s)); left > 0; --left) {
          take |= same & -same;
          same &= same - 1;
        }
        tied -= __builtin_amdgcn_readlane(inc, 63);
      }
      const int c = __popc(take), inc = akv_wave_inclusive_scan(c);
      int to = at + inc - c;
      for (; take; take &= take - 1) out[to++] = c0 + __ffs(take) - 1;
      at += __builtin_amdgcn_readlane(inc, 63);
    }
  }
}

// Wider tables go the long way over scores in memory.
#define BI_WIDE 16384
template <int D, int DT, int W, int HELD> static int bi_pick(const bi_rank_args& a, int64_t units, int bytes, hipStream_t stream) {
  int dev = 0;
  AKV_HIP(hipGetDevice(&dev));
  static akv_device_once once;
  if (const int rc = once(dev, [&]() -> int { return ab_lds((const void*)bi_pick_kernel<D, DT, W, HELD>, 16 * BI_WIDE / 4); })) return rc;
  bi_pick_kernel<D, DT, W, HELD><<<(uint32_t)units, 64 * W, bytes, stream>>>(a);
  AKV_LAUNCH_CHECK("bi_pick_kernel");
  return AKV_OK;
}
template <int D, int DT> static int bi_pick(const bi_rank_args& a, int64_t max_blocks, hipStream_t stream) {
  const int64_t units = ((int64_t)a.b.T / 16 + a.b.S + 1) * a.KVH, tiles = (max_blocks + 15) / 16;
  const int bytes = (int)(16 * ((max_blocks + 31) / 32) * 8);
  if (units > 0x7fffffff) return akv_fail(AKV_ERR_UNSUPPORTED, "akv_block_index_select: more than 2^31 rows");
  // Two workgroups of 8 wavefronts a CU, where there are workgroups for them, or one of 16 (registers hold as many scores): 2048 tokens over 1920 blocks 59.8 us
  // against 82.8, 512 tokens 24.5 against 23.9, 64 tokens 22.6 against 20.6.
  if (tiles <= 8 * 16 && units > ab_cus()) return bi_pick<D, DT, 8, 16>(a, units, bytes, stream);
  if (tiles <= 16 * 8) return bi_pick<D, DT, 16, 8>(a, units, bytes, stream);
  if (tiles <= 16 * 14) return bi_pick<D, DT, 16, 14>(a, units, bytes, stream);
  return bi_pick<D, DT, 16, 0>(a, units, bytes, stream);
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
