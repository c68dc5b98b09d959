// Tokens of a paged cache given up: of every sequence and kv head the first and last tokens and the heaviest others stay, and their rows
// move to the front of the sequence, in order.
//
//   akv_evict_select   which ones: weights -> the keep-th largest -> positions, ascending, and the weights they had
//   akv_evict_move     rows of any caches [blocks][positions][heads][bytes], by these positions
#include "akv_batch.h"
#include "akv_device_once.h"

// ---- select ------------------------------------------------------------------------------------------------------------------------------
struct ev_args {
  const float* w; int64_t ws_seq, ws_head;
  const void* lens; int lens_it;
  int32_t* kept; int64_t ks_seq, ks_head;
  float* out; int64_t os_seq, os_head;
  void* out_lens;
  int64_t length;                       // weights of a row
  int keep, sinks, recent;
};
// order of weights as whole numbers: a zero is a zero, a NaN stands with -infinity
__device__ __forceinline__ uint32_t ev_order(float x) {
  const uint32_t u = __float_as_uint(x == x ? x + 0.f : -INFINITY);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// One workgroup of 16 wavefronts a (kv head, sequence), each of which takes a run of the positions, NR of every lane in registers (NR = 0: read
// again and again).  The keep-th largest order is found by halving its range, bit by bit; what is above it stays, and the first ones that equal it.
#define EV_THREADS 1024
template <int NR> __global__ __launch_bounds__(EV_THREADS) void ev_select_kernel(ev_args a) {
  constexpr int WAVES = EV_THREADS / 64;
  __shared__ int sums[2][WAVES], ties[WAVES];
  const int kvh = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = ab_clamp(akv_load_index(a.lens, a.lens_it, seq), a.length);
  const float* w = a.w + (int64_t)seq * a.ws_seq + (int64_t)kvh * a.ws_head;
  int32_t* kept = a.kept + (int64_t)seq * a.ks_seq + (int64_t)kvh * a.ks_head;
  float* out = a.out + (int64_t)seq * a.os_seq + (int64_t)kvh * a.os_head;
  const int stay = min(n, a.keep);
  if (kvh == 0 && tid == 0) {
    if (a.lens_it == AKV_I64) ((int64_t*)a.out_lens)[seq] = stay;
    else ((int32_t*)a.out_lens)[seq] = stay;
  }
  for (int i = stay + tid; i < a.keep; i += EV_THREADS) kept[i] = -1;
  for (int64_t i = stay + tid; i < a.length; i += EV_THREADS) out[i] = 0.f;
  if (n <= a.keep) {
    for (int i = tid; i < n; i += EV_THREADS) {
      kept[i] = i;
      out[i] = w[i];
    }
    return;
  }
  const int each = (n + EV_THREADS - 1) / EV_THREADS, first = wave * each * 64;      // positions of a lane; of the wavefront the first
  auto order = [&](int i) { return i >= n ? 0u : i < a.sinks || i >= n - a.recent ? 0xffffffffu : ev_order(w[i]); };
  uint32_t held[NR > 0 ? NR : 1];
#pragma unroll
  for (int c = 0; c < NR; ++c) held[c] = c < each ? order(first + 64 * c + lane) : 0u;
  auto count = [&](auto test) {           // lanes of the wavefront's positions that pass
    int k = 0;
    if constexpr (NR > 0) {
#pragma unroll
      for (int c = 0; c < NR; ++c) k += __popcll(__ballot(test(held[c])));
    } else {
      for (int c = 0; c < each; ++c) k += __popcll(__ballot(test(order(first + 64 * c + lane))));
    }
    return k;
  };
  uint32_t t = 0u;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t c = t | 1u << bit;
    const int mine = count([&](uint32_t o) { return o >= c; });
    if (lane == 0) sums[bit & 1][wave] = mine;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int v = 0; v < WAVES; ++v) all += sums[bit & 1][v];
    if (all >= a.keep) t = c;
    if (all == a.keep) break;             // (the same in every thread)
  }
  // (order 0 is no position's: t > 0)
  const int above = count([&](uint32_t o) { return o > t; }), tied = count([&](uint32_t o) { return o == t; });
  __syncthreads();
  if (lane == 0) {
    sums[0][wave] = above;
    ties[wave] = tied;
  }
  __syncthreads();
  int all = 0, before = 0, tied_before = 0;
  for (int v = 0; v < WAVES; ++v) {
    all += sums[0][v];
    if (v < wave) before += sums[0][v], tied_before += ties[v];
  }
  int equal = max(0, a.keep - all - tied_before), at = before + min(a.keep - all, tied_before);
  const uint64_t below = (1ull << lane) - 1;
  auto put = [&](int c, uint32_t o) {
    const uint64_t same = __ballot(o == t);
    const bool take = o > t || (o == t && __popcll(same & below) < equal);
    const uint64_t taken = __ballot(take);
    if (take) {
      const int i = first + 64 * c + lane, to = at + __popcll(taken & below);
      kept[to] = i;
      out[to] = w[i];
    }
    at += __popcll(taken);
    equal -= min(equal, (int)__popcll(same));
  };
  if constexpr (NR > 0) {
#pragma unroll
    for (int c = 0; c < NR; ++c) put(c, held[c]);
  } else {
    for (int c = 0; c < each; ++c) put(c, order(first + 64 * c + lane));
  }
}

extern "C" int akv_evict_select(const float* weights, int64_t ws_seq, int64_t ws_head, int64_t length, const void* context_lens, int cl_itype, int num_seqs, int num_kv_heads, int keep,
                                int num_sink, int num_recent, int32_t* kept, int64_t ks_seq, int64_t ks_head, float* kept_weights, int64_t os_seq, int64_t os_head, void* kept_lens,
                                void* stream) {
  const char* name = "akv_evict_select";
  AKV_REQUIRE(akv_valid_itype(cl_itype), "%s: bad index type", name);
  AKV_REQUIRE(num_seqs >= 0 && num_kv_heads > 0 && length >= 0, "%s: %d sequences, %d kv heads, rows of %lld weights", name, num_seqs, num_kv_heads, (long long)length);
  AKV_REQUIRE(keep > 0 && num_sink >= 0 && num_recent >= 0 && num_sink <= keep - num_recent, "%s: %d tokens cannot hold the first %d and last %d", name, keep, num_sink, num_recent);
  if (num_seqs == 0) return AKV_OK;
  AKV_REQUIRE(context_lens && kept && kept_lens && (length == 0 || (weights && kept_weights)), "%s: null pointer", name);
  if (num_seqs > 65535) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: more than 65535 sequences", name);
  if (length > AB_MOST_TOKENS) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: rows of 2^31 weights", name);
  ev_args a = {};
  a.w = weights; a.ws_seq = ws_seq; a.ws_head = ws_head; a.lens = context_lens; a.lens_it = cl_itype;
  a.kept = kept; a.ks_seq = ks_seq; a.ks_head = ks_head; a.out = kept_weights; a.os_seq = os_seq; a.os_head = os_head; a.out_lens = kept_lens;
  a.length = length; a.keep = keep; a.sinks = num_sink; a.recent = num_recent;
  const dim3 grid((uint32_t)num_kv_heads, (uint32_t)num_seqs);
  const hipStream_t s = (hipStream_t)stream;
  if (length <= 8 * EV_THREADS) ev_select_kernel<8><<<grid, EV_THREADS, 0, s>>>(a);
  else if (length <= 32 * EV_THREADS) ev_select_kernel<32><<<grid, EV_THREADS, 0, s>>>(a);
  else ev_select_kernel<0><<<grid, EV_THREADS, 0, s>>>(a);
  AKV_LAUNCH_CHECK("ev_select_kernel");
  return AKV_OK;
}

// ---- move --------------------------------------------------------------------------------------------------------------------------------
#define EV_CACHES AKV_EVICT_CACHES
struct ev_cache {
  uint8_t* p; int64_t blk, pos, head;   // bytes
  int units, log;                       // of a row: pieces of 2^log bytes
  int slice, first;                     // pieces of a slice; number of the cache's first slice or piece
};
struct ev_move_args {
  ab_batch b;                           // lens: tokens that stay
  const void* to_tables; int to_it; int64_t to_stride, to_blocks;
  const int32_t* kept; int64_t ks_seq, ks_head;
  ev_cache c[EV_CACHES];
  int caches, keep, pieces;
};
struct ev_row { int64_t blk; uint32_t pos; };
__device__ __forceinline__ ev_row ev_row_of(const ev_move_args& a, int seq, int position, bool to) {
  ev_row r;
  const int64_t col = akv_div32((uint32_t)position, (uint32_t)a.b.block_size, a.b.bs_recip, r.pos);
  r.blk = to ? akv_clamp_block(akv_load_index(a.to_tables, a.to_it, (int64_t)seq * a.to_stride + col), a.b.num_blocks) : ab_block(a.b, seq, col);
  return r;
}
__device__ __forceinline__ uint8_t* ev_at(const ev_cache& c, ev_row r, int head, int unit) {
  return c.p + r.blk * c.blk + (int64_t)r.pos * c.pos + (int64_t)head * c.head + ((int64_t)unit << c.log);
}
struct ev_piece { ab_u4 v; };
__device__ __forceinline__ void ev_load(ev_piece& x, const uint8_t* p, int log) {
  if (log == 4) x.v = *(const ab_u4*)p;
  else if (log == 3) { const ab_u2 y = *(const ab_u2*)p; x.v[0] = y[0]; x.v[1] = y[1]; }
  else if (log == 2) x.v[0] = *(const uint32_t*)p;
  else if (log == 1) x.v[0] = *(const uint16_t*)p;
  else x.v[0] = *p;
}
__device__ __forceinline__ void ev_store(const ev_piece& x, uint8_t* p, int log) {
  if (log == 4) *(ab_u4*)p = x.v;
  else if (log == 3) *(ab_u2*)p = (ab_u2){x.v[0], x.v[1]};
  else if (log == 2) *(uint32_t*)p = x.v[0];
  else if (log == 1) *(uint16_t*)p = (uint16_t)x.v[0];
  else *p = (uint8_t)x.v[0];
}

// To blocks that nobody reads: a thread a piece.
__global__ __launch_bounds__(256) void ev_copy_kernel(ev_move_args a) {
  const int head = blockIdx.y, seq = blockIdx.z;
  const int n = min(ab_clamp(akv_load_index(a.b.lens, a.b.lens_it, seq), AB_MOST_TOKENS), a.keep);
  const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int j = (int)(x / a.pieces);
  if (j >= n) return;
  int piece = (int)(x - (int64_t)j * a.pieces), i = 0;
  while (i + 1 < a.caches && piece >= a.c[i + 1].first) ++i;
  const ev_cache& c = a.c[i];
  const int from = a.kept[(int64_t)seq * a.ks_seq + (int64_t)head * a.ks_head + j];
  if (from < 0 || from >= a.b.max_blocks * a.b.block_size || j >= a.to_blocks * a.b.block_size) return;
  ev_piece v;
  ev_load(v, ev_at(c, ev_row_of(a, seq, from, false), head, piece - c.first), c.log);
  ev_store(v, ev_at(c, ev_row_of(a, seq, j, true), head, piece - c.first), c.log);
}

// In place.  A token never moves back, so what a tile of tokens writes lies before everything that later tiles read, and a workgroup that walks
// the tiles in order needs only to have read a tile before it writes it.  Slices of the rows are independent of each other, and
// so are heads and sequences: a workgroup each.
#define EV_HELD 8
__global__ __launch_bounds__(256) void ev_compact_kernel(ev_move_args a) {
  const int head = blockIdx.y, seq = blockIdx.z, tid = threadIdx.x;
  int i = 0;
  while (i + 1 < a.caches && (int)blockIdx.x >= a.c[i + 1].first) ++i;
  const ev_cache& c = a.c[i];
  const int u0 = ((int)blockIdx.x - c.first) * c.slice, units = min(c.slice, c.units - u0);
  const int64_t cap = min(a.b.max_blocks, a.to_blocks) * a.b.block_size;
  const int n = min(ab_clamp(akv_load_index(a.b.lens, a.b.lens_it, seq), cap < AB_MOST_TOKENS ? cap : AB_MOST_TOKENS), a.keep);
  const int32_t* kept = a.kept + (int64_t)seq * a.ks_seq + (int64_t)head * a.ks_head;
  const int tile = 256 * EV_HELD / units;        // tokens
  for (int j0 = 0; j0 < n; j0 += tile) {
    ev_piece v[EV_HELD];
    uint8_t* to[EV_HELD];
#pragma unroll
    for (int k = 0; k < EV_HELD; ++k) {
      const int x = 256 * k + tid, t = x / units, j = j0 + t, unit = u0 + x - t * units;
      to[k] = nullptr;
      if (t >= tile || j >= n) continue;
      const int from = kept[j];
      if (from <= j || from >= a.b.max_blocks * a.b.block_size) continue;      // (where it is already)
      to[k] = ev_at(c, ev_row_of(a, seq, j, true), head, unit);
      ev_load(v[k], ev_at(c, ev_row_of(a, seq, from, false), head, unit), c.log);
    }
    // every load of the workgroup has its value before the first store
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int k = 0; k < EV_HELD; ++k)
      if (to[k]) ev_store(v[k], to[k], c.log);
  }
}

extern "C" int akv_evict_move(const int32_t* kept, int64_t ks_seq, int64_t ks_head, const void* kept_lens, int kl_itype, int keep, const void* block_tables, int bt_itype, int64_t bt_stride,
                              int64_t max_blocks_per_seq, const void* out_tables, int ot_itype, int64_t ot_stride, int64_t out_blocks_per_seq, const akv_evict_cache* caches, int num_caches,
                              int num_seqs, int num_kv_heads, int block_size, int64_t num_blocks, void* stream) {
  const char* name = "akv_evict_move";
  const int rc = ab_check(name, block_tables, bt_itype, kept_lens, kl_itype, nullptr, AKV_I32, num_seqs, 0, num_kv_heads, block_size, num_blocks, max_blocks_per_seq);
  if (rc) return rc;
  AKV_REQUIRE(keep > 0 && num_caches >= 0 && (num_caches == 0 || caches), "%s: keep %d, %d caches", name, keep, num_caches);
  AKV_REQUIRE(!out_tables || (akv_valid_itype(ot_itype) && out_blocks_per_seq >= 0), "%s: bad table of outputs", name);
  if (num_caches > EV_CACHES) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: more than %d caches", name, EV_CACHES);
  if (num_seqs == 0 || num_caches == 0 || num_blocks == 0 || max_blocks_per_seq == 0) return AKV_OK;
  AKV_REQUIRE(kept, "%s: null pointer", name);
  if (num_seqs > 65535 || num_kv_heads > 65535) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: more than 65535 sequences or kv heads", name);
  ev_move_args a = {};
  a.b = ab_make(block_tables, bt_itype, bt_stride, kept_lens, kl_itype, nullptr, AKV_I32, num_seqs, 0, block_size, num_blocks, max_blocks_per_seq);
  a.to_tables = out_tables ? out_tables : block_tables; a.to_it = out_tables ? ot_itype : bt_itype;
  a.to_stride = out_tables ? ot_stride : bt_stride; a.to_blocks = out_tables ? out_blocks_per_seq : max_blocks_per_seq;
  a.kept = kept; a.ks_seq = ks_seq; a.ks_head = ks_head; a.caches = num_caches; a.keep = keep;
  int64_t slices = 0, pieces = 0;
  for (int i = 0; i < num_caches; ++i) {
    const akv_evict_cache& x = caches[i];
    AKV_REQUIRE(x.data && x.row_bytes > 0, "%s: cache %d: null pointer or rows of %lld bytes", name, i, (long long)x.row_bytes);
    if (x.row_bytes > 1 << 20) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: rows of more than 2^20 bytes", name);
    ev_cache& c = a.c[i];
    c.p = (uint8_t*)x.data; c.blk = x.s_blk; c.pos = x.s_pos; c.head = x.s_head;
    // pieces as wide as rows, their places and their ends allow
    const uint64_t all = (uint64_t)(uintptr_t)x.data | (uint64_t)x.s_blk | (uint64_t)x.s_pos | (uint64_t)x.s_head | (uint64_t)x.row_bytes;
    for (c.log = 4; all & ((1u << c.log) - 1); --c.log) {}
    c.units = (int)(x.row_bytes >> c.log);
    c.slice = c.units < 4 ? c.units : 4;
    c.first = (int)(out_tables ? pieces : slices);
    slices += (c.units + c.slice - 1) / c.slice;
    pieces += c.units;
  }
  a.pieces = (int)pieces;
  const hipStream_t s = (hipStream_t)stream;
  if (out_tables) {
    const int64_t most = out_blocks_per_seq * block_size < keep ? out_blocks_per_seq * block_size : keep, groups = (most * pieces + 255) / 256;
    if (groups > 0x7fffffff) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: more than 2^39 pieces", name);
    if (groups == 0) return AKV_OK;
    ev_copy_kernel<<<dim3((uint32_t)groups, (uint32_t)num_kv_heads, (uint32_t)num_seqs), 256, 0, s>>>(a);
    AKV_LAUNCH_CHECK("ev_copy_kernel");
  } else {
    ev_compact_kernel<<<dim3((uint32_t)slices, (uint32_t)num_kv_heads, (uint32_t)num_seqs), 256, 0, s>>>(a);
    AKV_LAUNCH_CHECK("ev_compact_kernel");
  }
  return AKV_OK;
}
