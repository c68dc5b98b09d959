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

// One workgroup of 16 wavefronts a (kv head, sequence), each of which takes a run of the positions.  Orders lie in LDS (where they fit, otherwise they are
// made again from the weights).  The keep-th largest is found eight bits at a time, from the highest in which the orders differ: a histogram of
// the next eight bits of those that share the bits known so far.  What is above it stays, and the first ones that equal it.
//
// Few workgroups have much to do here, so that each waits for its code too: the loops are short.  Weights are alike in their upper bits, so that counters have
// copies; when few share the known bits they are listed, and later levels read the list alone.  8 heads of 32768 positions take 32 us: a bit at a time with
// orders in registers 42, one copy of a counter and no list 36.  (Counters take some 2.5 lanes a clock; eleven bits at a time with two
// copies took as long.)  16 sequences of 8 heads, up to 9000 positions, take 15 us.
#define EV_THREADS 1024
#define EV_HELD 32768                   // orders in LDS
#define EV_COPIES 16                    // of a counter: weights are alike, and lanes that add to one word wait for each other
#define EV_LIST 2048                    // those that share the known bits, once they are few
__global__ __launch_bounds__(EV_THREADS) void ev_select_kernel(ev_args a, int room) {
  constexpr int WAVES = EV_THREADS / 64;
  static_assert(256 * EV_COPIES == 4 * EV_THREADS && EV_COPIES == 16, "counters");
  extern __shared__ uint32_t orders[];   // [room], then the list
  __shared__ __attribute__((aligned(16))) int hist[256 * EV_COPIES], sums[WAVES], ties[WAVES], found[3], listed;
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
  // zeros behind
  const int64_t even = min(a.length, stay + (int64_t)(-((int64_t)((uintptr_t)(out + stay) >> 2)) & 3));      // from here on sixteen bytes at a time
  if (tid < even - stay) out[stay + tid] = 0.f;
  for (int64_t i = even + 4 * tid; i < a.length; i += 4 * EV_THREADS) {
    if (i + 3 < a.length) *(ab_f4*)(out + i) = (ab_f4){0.f, 0.f, 0.f, 0.f};
    else
      for (int64_t k = i; k < a.length; ++k) out[k] = 0.f;
  }
  if (n <= a.keep) {
    for (int i = tid; i < a.keep; i += EV_THREADS) {
      kept[i] = i < n ? i : -1;
      if (i < n) out[i] = w[i];
    }
    return;
  }
  const bool held = n <= room, wide = ((uintptr_t)w & 15) == 0;
  // orders of four positions i .. i + 3 (0 past the last); what stays anyway is above all others
  auto rank = [&](int i, float x) { return i >= n ? 0u : i < a.sinks || i >= n - a.recent ? 0xffffffffu : ev_order(x); };
  auto weights = [&](int i) {
    if (wide && i + 3 < n) return *(const ab_f4*)(w + i);
    ab_f4 x;
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = w[min(i + k, n - 1)];
    return x;
  };
  auto made = [&](int i) {
    const ab_f4 x = weights(i);
    ab_u4 o;
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = rank(i + k, x[k]);
    return o;
  };
  auto order = [&](int i) { return held ? *(const ab_u4*)(orders + i) : made(i); };
  constexpr int ROUND = 4 * EV_THREADS;
  const int rounds = (n + ROUND - 1) / ROUND;
  // the bits that all others share: those above the highest in which some differ
  uint32_t both = 0xffffffffu, any = 0u;
  for (int r = 0; r < rounds; r += 4) {
    ab_f4 x[4];                         // (on their way together)
#pragma unroll
    for (int q = 0; q < 4; ++q) x[q] = weights(min((r + q) * ROUND + 4 * tid, (n - 1) & ~3));
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (r + q >= rounds) break;
      const int i = (r + q) * ROUND + 4 * tid;
      ab_u4 o;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        o[k] = rank(i + k, x[q][k]);
        both &= o[k] + 1u > 1u ? o[k] : 0xffffffffu;
        any |= o[k] + 1u > 1u ? o[k] : 0u;
      }
      if (held) *(ab_u4*)(orders + i) = o;
    }
  }
#pragma unroll
  for (int m = 1; m < 64; m *= 2) {
    both &= __shfl_xor(both, m, 64);
    any |= __shfl_xor(any, m, 64);
  }
  if (lane == 0) {
    sums[wave] = (int)both;
    ties[wave] = (int)any;
  }
  __syncthreads();
  for (int v = 0; v < WAVES; ++v) {
    both &= (uint32_t)sums[v];
    any |= (uint32_t)ties[v];
  }
  int need = a.keep - a.sinks - a.recent;      // how many of those that share the known bits stay
  int unknown = any > both ? 32 - __clz(any ^ both) : 0, sharing = n - a.sinks - a.recent;
  // the threshold, as far as it is known
  uint32_t t = need == 0 ? 0xffffffffu : unknown == 32 ? 0u : both >> unknown << unknown;
  if (need == 0) sharing = unknown = 0;
  uint32_t* const list = orders + room;
  bool gathered = false;
  int in_list = 0;
  while (unknown > 0 && need != sharing) {     // (all that share the bits stay: the search is over)
    const int width = min(8, unknown), shift = unknown - width;
    __syncthreads();
    *(ab_u4*)(hist + 4 * tid) = (ab_u4){0u, 0u, 0u, 0u};
    if (tid == 0) listed = 0;
    __syncthreads();
    const uint32_t range = unknown == 32 ? 0xffffffffu : (1u << unknown) - 1;
    auto take = [&](uint32_t o) { atomicAdd(hist + (o >> shift & ((1u << width) - 1)) * EV_COPIES + (lane & (EV_COPIES - 1)), 1); };
    auto shares = [&](uint32_t o) { return (o ^ t) <= range && o + 1u > 1u; };      // (neither what stays anyway nor what is past the last)
    if (gathered) {
      for (int i = tid; i < in_list; i += EV_THREADS)
        if (shares(list[i])) take(list[i]);
    } else {
      const bool gather = unknown < 32 && sharing <= EV_LIST;
#pragma unroll 2
      for (int r = 0; r < rounds; ++r) {
        const ab_u4 o = order(r * ROUND + 4 * tid);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (shares(o[k])) {
            take(o[k]);
            if (gather) list[min(atomicAdd(&listed, 1), EV_LIST - 1)] = o[k];
          }
      }
      gathered = gather;
      in_list = sharing;
    }
    __syncthreads();
    {
      // copies together: four of them a thread, a counter four threads
      const ab_u4 x = *(const ab_u4*)(hist + 4 * tid);
      int sum = (int)(x[0] + x[1] + x[2] + x[3]);
      sum += __shfl_xor(sum, 1, 64);
      sum += __shfl_xor(sum, 2, 64);
      __syncthreads();
      if ((tid & 3) == 0) hist[tid >> 2] = sum;
    }
    __syncthreads();
    if (wave == 0) {
      // a lane four values, the first lane the uppermost
      const int* h = hist + 252 - 4 * lane;
      const int c[4] = {h[3], h[2], h[1], h[0]}, sum = c[0] + c[1] + c[2] + c[3], inc = akv_wave_inclusive_scan(sum);
      int before = inc - sum;
      if (before < need && need <= inc) {
        int i = 0;
#pragma unroll
        for (int k = 0; k < 3; ++k)
          if (i == k && before + c[k] < need) before += c[k], ++i;
        found[0] = 255 - 4 * lane - i;
        found[1] = need - before;
        found[2] = i == 0 ? c[0] : i == 1 ? c[1] : i == 2 ? c[2] : c[3];
      }
    }
    __syncthreads();
    t |= (uint32_t)found[0] << shift;
    need = found[1];
    sharing = found[2];
    unknown = shift;
  }
  // (where the search ended early everything from t on stays, and nothing has to be counted as equal)
  const bool exact = need != sharing;
  const uint32_t from = exact ? t + 1 : t;     // what stays whatever is equal (with need > 0 t is below 0xffffffff)
  const int each = (rounds * ROUND) / WAVES, first = wave * each;      // the wavefront's run of positions
  int above = 0, tied = 0;
  for (int i = first; i < first + each; i += 256) {
    const ab_u4 o = order(i + 4 * lane);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      above += o[k] >= from;
      tied += exact && o[k] == t;
    }
  }
  above = akv_wave_sum(above);
  tied = akv_wave_sum(tied);
  __syncthreads();
  if (lane == 0) {
    sums[wave] = above;
    ties[wave] = tied;
  }
  __syncthreads();
  int at = 0, equal = exact ? need : 0;
  for (int v = 0; v < wave; ++v) {
    at += sums[v] + min(equal, ties[v]);
    equal -= min(equal, ties[v]);
  }
  for (int i0 = first; i0 < first + each && i0 < n; i0 += 256) {
    const int i = i0 + 4 * lane;
    const ab_u4 o = order(i);
    int left = 0;                       // equal ones that the lanes before leave
    if (exact) {
      int mine = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) mine += o[k] == t;
      const int inc = akv_wave_inclusive_scan(mine);
      left = equal - (inc - mine);
      equal -= min(equal, __builtin_amdgcn_readlane(inc, 63));
    }
    uint32_t take = 0u;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool same = exact && o[k] == t;
      take |= (uint32_t)(o[k] >= from || (same && left > 0)) << k;
      left -= same;
    }
    const int mine = __popc(take), inc = akv_wave_inclusive_scan(mine);
    int to = at + inc - mine;
    at += __builtin_amdgcn_readlane(inc, 63);
    // the weight from its order, but where that does not tell (a weight read again is waited for)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (!(take >> k & 1)) continue;
      float x = __uint_as_float(o[k] ^ ((o[k] >> 31) ? 0x80000000u : 0xffffffffu));
      if (o[k] == 0xffffffffu || o[k] == 0x80000000u || o[k] == 0x007fffffu) x = w[i + k];
      kept[to] = i + k;
      out[to++] = x;
    }
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
  int dev = 0;
  AKV_HIP(hipGetDevice(&dev));
  static akv_device_once once;
  if (const int rc = once(dev, [&]() -> int { return ab_lds((const void*)ev_select_kernel, 4 * (EV_HELD + EV_LIST)); })) return rc;
  const int room = (int)(length < EV_HELD ? (length + 4095) / 4096 * 4096 : EV_HELD);      // (whole rounds of the kernel)
  ev_select_kernel<<<dim3((uint32_t)num_kv_heads, (uint32_t)num_seqs), EV_THREADS, 4 * (size_t)(room + EV_LIST), (hipStream_t)stream>>>(a, room);
  AKV_LAUNCH_CHECK("ev_select_kernel");
  return AKV_OK;
}

// ---- move --------------------------------------------------------------------------------------------------------------------------------
#define EV_CACHES AKV_EVICT_CACHES
struct ev_cache {
  uint8_t* p; int64_t blk, pos, head;   // bytes
  int units, log, per;                  // of a row: units of 2^log bytes; units of a piece
  int pieces, slice, first;             // of a row; pieces of a slice; number of the cache's first slice or piece
};
struct ev_move_args {
  ab_batch b;                           // lens: tokens that stay
  const void* to_tables; int to_it; int64_t to_stride, to_blocks;
  const int32_t* kept; int64_t ks_seq, ks_head;
  ev_cache c[EV_CACHES];
  int caches, keep, pieces, heads;      // pieces: of a token and head
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
// up to sixteen bytes, as units of 2^log bytes
struct ev_piece { ab_u4 v; };
struct __attribute__((packed, aligned(4))) ev_words { uint32_t v[4]; };
__device__ __forceinline__ void ev_load(ev_piece& x, const uint8_t* p, int log, int units) {
  if (log == 4) x.v = *(const ab_u4*)p;
  else if (log == 2 && units >= 4) x.v = __builtin_bit_cast(ab_u4, *(const ev_words*)p);
  else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < units) x.v[k] = log == 2 ? ((const uint32_t*)p)[k] : log == 1 ? ((const uint16_t*)p)[k] : p[k];
  }
}
__device__ __forceinline__ void ev_store(const ev_piece& x, uint8_t* p, int log, int units) {
  if (log == 4) *(ab_u4*)p = x.v;
  else if (log == 2 && units >= 4) *(ev_words*)p = __builtin_bit_cast(ev_words, x.v);
  else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < units) {
        if (log == 2) ((uint32_t*)p)[k] = x.v[k];
        else if (log == 1) ((uint16_t*)p)[k] = (uint16_t)x.v[k];
        else p[k] = (uint8_t)x.v[k];
      }
  }
}

// To blocks that nobody reads: a thread a piece of a row, heads of a token side by side, as the rows lie where they go to.
// 16 sequences of 2048 tokens of 4 bits take 34 us: 125 MB read, since most lines of 128 bytes hold a row of another head or token as well, and 40 MB written,
// 4.8 TB/s, what a large copy reaches.  (With four bytes a thread and a division of 64 bits for it 68 us; four tokens a thread, all loads on their way
// together, 38: neighbouring tokens share lines.)
__global__ __launch_bounds__(256) void ev_copy_kernel(ev_move_args a) {
  const int seq = blockIdx.y;
  const int n = min(ab_clamp(akv_load_index(a.b.lens, a.b.lens_it, seq), AB_MOST_TOKENS), a.keep);
  const uint32_t x = blockIdx.x * 256 + threadIdx.x, per = (uint32_t)a.heads * (uint32_t)a.pieces;
  const uint32_t j = x / per, rest = x - j * per, head = rest / (uint32_t)a.pieces;
  if ((int64_t)j >= n) return;
  const int piece = (int)(rest - head * (uint32_t)a.pieces);
  int i = 0;
  while (i + 1 < a.caches && piece >= a.c[i + 1].first) ++i;
  const ev_cache& c = a.c[i];
  const int from = a.kept[(int64_t)seq * a.ks_seq + (int64_t)head * a.ks_head + j];
  if (from < 0 || from >= a.b.max_blocks * a.b.block_size || (int64_t)j >= a.to_blocks * a.b.block_size) return;
  const int unit = c.per * (piece - c.first), units = min(c.per, c.units - unit);
  ev_piece v;
  ev_load(v, ev_at(c, ev_row_of(a, seq, from, false), (int)head, unit), c.log, units);
  ev_store(v, ev_at(c, ev_row_of(a, seq, (int)j, true), (int)head, unit), c.log, units);
}

// In place.  A token never moves back, so what a tile of tokens writes lies before everything that later tiles read, and a workgroup that walks
// the tiles in order needs only to have read a tile before it writes it.  Slices of the rows are independent of each other, and
// so are heads and sequences: a workgroup each.
// 16 sequences of 2048 tokens of 4 bits take 52 us and one of 4096 tokens of 8 heads of 128 62, where ev_copy_kernel takes 31 and 9.4: few workgroups (512 and 64), each of
// which waits for a tile's positions, table entries and rows one after the other.
#define EV_PIECES 8
__global__ __launch_bounds__(256) void ev_compact_kernel(ev_move_args a) {
  const int head = blockIdx.y, seq = blockIdx.z, tid = threadIdx.x;
  int i = 0;
  while (i + 1 < a.caches && (int)blockIdx.x >= a.c[i + 1].first) ++i;
  const ev_cache& c = a.c[i];
  const int p0 = ((int)blockIdx.x - c.first) * c.slice, pieces = min(c.slice, c.pieces - p0);      // of a row
  const int64_t cap = min(a.b.max_blocks, a.to_blocks) * a.b.block_size;
  const int n = min(ab_clamp(akv_load_index(a.b.lens, a.b.lens_it, seq), cap < AB_MOST_TOKENS ? cap : AB_MOST_TOKENS), a.keep);
  const int32_t* kept = a.kept + (int64_t)seq * a.ks_seq + (int64_t)head * a.ks_head;
  const int tile = 256 * EV_PIECES / pieces;      // tokens
  for (int j0 = 0; j0 < n; j0 += tile) {
    ev_piece v[EV_PIECES];
    uint8_t* to[EV_PIECES];
    int count[EV_PIECES];               // units
#pragma unroll
    for (int k = 0; k < EV_PIECES; ++k) {
      const int x = 256 * k + tid, t = x / pieces, j = j0 + t, unit = c.per * (p0 + x - t * pieces);
      count[k] = min(c.per, c.units - unit);
      to[k] = nullptr;
      if (t >= tile || j >= n) continue;
      const int from = kept[j];
      if (from <= j || from >= a.b.max_blocks * a.b.block_size) continue;      // (where it is already)
      to[k] = ev_at(c, ev_row_of(a, seq, j, true), head, unit);
      ev_load(v[k], ev_at(c, ev_row_of(a, seq, from, false), head, unit), c.log, count[k]);
    }
    // every load of the workgroup has its value before the first store
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int k = 0; k < EV_PIECES; ++k)
      if (to[k]) ev_store(v[k], to[k], c.log, count[k]);
  }
}

// Whether a row of cache x and one of cache y share a byte (or two rows of one cache), over `counts` blocks, positions and heads.  A dimension of the same stride in both
// moves the one against the other by multiples of it, the widest first; what has unlike strides is taken as one piece from end to end.
static bool ev_meet(const __int128* stride, const int64_t* reach, int dims, __int128 lo, __int128 hi, bool other) {
  if (dims == 0) return other && lo <= 0 && 0 <= hi;
  __int128 rest = 0;                    // what the dimensions behind move
  for (int i = 1; i < dims; ++i) rest += stride[i] * reach[i];
  auto floor = [](__int128 a, __int128 b) { return a / b - (a % b < 0); };
  __int128 from = -floor(rest - lo, *stride), to = floor(hi + rest, *stride);
  if (from < -*reach) from = -*reach;
  if (to > *reach) to = *reach;
  if (to - from > 64) return true;      // (of strides that are no layout of rows side by side)
  for (__int128 d = from; d <= to; ++d)
    if (ev_meet(stride + 1, reach + 1, dims - 1, lo - d * *stride, hi - d * *stride, other || d != 0)) return true;
  return false;
}
static bool ev_share(const akv_evict_cache& x, const akv_evict_cache& y, bool same, const int64_t* counts) {
  const int64_t xs[3] = {x.s_blk, x.s_pos, x.s_head}, ys[3] = {y.s_blk, y.s_pos, y.s_head};
  __int128 stride[3], x0 = (intptr_t)x.data, x1 = x0 + x.row_bytes, y0 = (intptr_t)y.data, y1 = y0 + y.row_bytes, ways = 0;
  int64_t reach[3];
  int dims = 0;
  for (int i = 0; i < 3; ++i) {
    const int64_t n = counts[i] - 1;
    if (n == 0) continue;
    if (xs[i] != ys[i]) {
      (xs[i] < 0 ? x0 : x1) += (__int128)xs[i] * n;
      (ys[i] < 0 ? y0 : y1) += (__int128)ys[i] * n;
    } else if (xs[i] != 0) {
      const __int128 s = xs[i] < 0 ? -(__int128)xs[i] : xs[i];
      int at = dims++;
      for (; at > 0 && stride[at - 1] < s; --at) stride[at] = stride[at - 1], reach[at] = reach[at - 1];
      stride[at] = s;
      reach[at] = n;
      ways += s * n;
    } else if (same) return true;
  }
  if (x0 - ways >= y1 || y0 - ways >= x1) return false;
  return ev_meet(stride, reach, dims, y0 - x1 + 1, y1 - x0 - 1, !same);
}

// The launch of a move: `groups` workgroups (0: nothing to do)
struct ev_plan { ev_move_args a; dim3 groups; bool in_place; };
static int ev_prepare(ev_plan& plan, const int32_t* kept, int64_t ks_seq, int64_t ks_head, const void* kept_lens, int kl_itype, int keep, const void* block_tables, int bt_itype,
                      int64_t bt_stride, int64_t max_blocks_per_seq, const void* out_tables, int ot_itype, int64_t ot_stride, int64_t out_blocks_per_seq, const akv_evict_cache* caches,
                      int num_caches, int num_seqs, int num_kv_heads, int block_size, int64_t num_blocks) {
  plan.groups = dim3(0);
  plan.in_place = !out_tables;
  const char* name = "akv_evict_move";
  const int rc = ab_check(name, block_tables, bt_itype, kept_lens, kl_itype, nullptr, AKV_I32, num_seqs, 0, num_kv_heads, block_size, num_blocks, max_blocks_per_seq);
  if (rc) return rc;
  AKV_REQUIRE(keep > 0 && num_caches >= 0 && (num_caches == 0 || caches), "%s: keep %d, %d caches", name, keep, num_caches);
  AKV_REQUIRE(!out_tables || (akv_valid_itype(ot_itype) && out_blocks_per_seq >= 0), "%s: bad table of outputs", name);
  if (num_caches > EV_CACHES) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: more than %d caches", name, EV_CACHES);
  if (num_seqs == 0 || num_caches == 0 || num_blocks == 0 || max_blocks_per_seq == 0) return AKV_OK;
  AKV_REQUIRE(kept, "%s: null pointer", name);
  if (num_seqs > 65535 || num_kv_heads > 65535) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: more than 65535 sequences or kv heads", name);
  ev_move_args& a = plan.a;
  a = ev_move_args{};
  a.b = ab_make(block_tables, bt_itype, bt_stride, kept_lens, kl_itype, nullptr, AKV_I32, num_seqs, 0, block_size, num_blocks, max_blocks_per_seq);
  a.to_tables = out_tables ? out_tables : block_tables; a.to_it = out_tables ? ot_itype : bt_itype;
  a.to_stride = out_tables ? ot_stride : bt_stride; a.to_blocks = out_tables ? out_blocks_per_seq : max_blocks_per_seq;
  a.kept = kept; a.ks_seq = ks_seq; a.ks_head = ks_head; a.caches = num_caches; a.keep = keep;
  int64_t slices = 0, pieces = 0;
  for (int i = 0; i < num_caches; ++i) {
    const akv_evict_cache& x = caches[i];
    AKV_REQUIRE(x.data && x.row_bytes > 0, "%s: cache %d: null pointer or rows of %lld bytes", name, i, (long long)x.row_bytes);
    if (x.row_bytes > 1 << 20) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: rows of more than 2^20 bytes", name);
    // (a row in two places would be moved twice at the same time)
    const int64_t counts[3] = {num_blocks, block_size, num_kv_heads};
    AKV_REQUIRE(!ev_share(x, x, true, counts), "%s: rows of cache %d share memory", name, i);
    for (int j = 0; j < i; ++j) AKV_REQUIRE(!ev_share(x, caches[j], false, counts), "%s: caches %d and %d share rows", name, j, i);
    ev_cache& c = a.c[i];
    c.p = (uint8_t*)x.data; c.blk = x.s_blk; c.pos = x.s_pos; c.head = x.s_head;
    // units as wide as rows, their places and their ends allow
    const uint64_t all = (uint64_t)(uintptr_t)x.data | (uint64_t)x.s_blk | (uint64_t)x.s_pos | (uint64_t)x.s_head | (uint64_t)x.row_bytes;
    c.log = all & 1 ? 0 : all & 3 ? 1 : all & 15 ? 2 : 4;
    c.units = (int)(x.row_bytes >> c.log);
    c.per = c.log == 4 ? 1 : 4;
    c.pieces = (c.units + c.per - 1) / c.per;
    c.slice = c.pieces < 4 ? c.pieces : 4;
    c.first = (int)(out_tables ? pieces : slices);
    slices += (c.pieces + c.slice - 1) / c.slice;
    pieces += c.pieces;
  }
  a.pieces = (int)pieces; a.heads = num_kv_heads;
  if (out_tables) {
    const int64_t most = out_blocks_per_seq * block_size < keep ? out_blocks_per_seq * block_size : keep, all = most * pieces * num_kv_heads;
    if (all > 0xffffff00ll) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: more than 2^32 pieces a sequence", name);
    plan.groups = dim3((uint32_t)((all + 255) / 256), (uint32_t)num_seqs);
  } else {
    plan.groups = dim3((uint32_t)slices, (uint32_t)num_kv_heads, (uint32_t)num_seqs);
  }
  return AKV_OK;
}
static int ev_move(const ev_plan& plan, void* stream) {
  if (plan.groups.x == 0) return AKV_OK;
  if (plan.in_place) ev_compact_kernel<<<plan.groups, 256, 0, (hipStream_t)stream>>>(plan.a);
  else ev_copy_kernel<<<plan.groups, 256, 0, (hipStream_t)stream>>>(plan.a);
  AKV_LAUNCH_CHECK(plan.in_place ? "ev_compact_kernel" : "ev_copy_kernel");
  return AKV_OK;
}

extern "C" int akv_evict_move(const int32_t* kept, int64_t ks_seq, int64_t ks_head, const void* kept_lens, int kl_itype, int keep, const void* block_tables, int bt_itype, int64_t bt_stride,
                              int64_t max_blocks_per_seq, const void* out_tables, int ot_itype, int64_t ot_stride, int64_t out_blocks_per_seq, const akv_evict_cache* caches, int num_caches,
                              int num_seqs, int num_kv_heads, int block_size, int64_t num_blocks, void* stream) {
  ev_plan plan;
  const int rc = ev_prepare(plan, kept, ks_seq, ks_head, kept_lens, kl_itype, keep, block_tables, bt_itype, bt_stride, max_blocks_per_seq, out_tables, ot_itype, ot_stride,
                            out_blocks_per_seq, caches, num_caches, num_seqs, num_kv_heads, block_size, num_blocks);
  return rc ? rc : ev_move(plan, stream);
}

extern "C" int akv_evict(const float* weights, int64_t ws_seq, int64_t ws_head, int64_t length, const void* context_lens, int cl_itype, int num_seqs, int num_kv_heads, int keep,
                         int num_sink, int num_recent, int32_t* kept, int64_t ks_seq, int64_t ks_head, float* kept_weights, int64_t os_seq, int64_t os_head, void* kept_lens,
                         const void* block_tables, int bt_itype, int64_t bt_stride, int64_t max_blocks_per_seq, const void* out_tables, int ot_itype, int64_t ot_stride,
                         int64_t out_blocks_per_seq, const akv_evict_cache* caches, int num_caches, int block_size, int64_t num_blocks, void* stream) {
  // (what is refused is refused before anything runs)
  ev_plan plan;
  int rc = ev_prepare(plan, kept, ks_seq, ks_head, kept_lens, cl_itype, keep, block_tables, bt_itype, bt_stride, max_blocks_per_seq, out_tables, ot_itype, ot_stride, out_blocks_per_seq,
                      caches, num_caches, num_seqs, num_kv_heads, block_size, num_blocks);
  if (rc == AKV_OK)
    rc = akv_evict_select(weights, ws_seq, ws_head, length, context_lens, cl_itype, num_seqs, num_kv_heads, keep, num_sink, num_recent, kept, ks_seq, ks_head, kept_weights, os_seq, os_head,
                          kept_lens, stream);
  return rc ? rc : ev_move(plan, stream);
}
