// akv_paged_chunk_attn: attention of a chunk of new tokens over the packed cache.
#include "akv_chunk_kernels.h"

// The rotation's tables in the order of the operand, a thread each sixteen bytes (akv_chunk_rotate.h): Pi, then Pi^T.
__global__ __launch_bounds__(256) void ck_tables_kernel(const float* __restrict__ pi, int d, const akv_prep_scale* __restrict__ scale, uint4* __restrict__ to) {
  const int per = d * d / 8, t = blockIdx.x * 256 + threadIdx.x;
  if (t >= 2 * per) return;
  const bool out = t >= per;
  const int i = out ? t - per : t, lane = i & 63, ks = (i >> 6) % (d / 16), dt = (i >> 6) / (d / 16);
  const int n = 32 * dt + (lane & 31), h = lane >> 5;
  const float f = CK_TURN * scale->down;
  uint32_t hi[4], lo[4];
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    hi[p] = lo[p] = 0u;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int j = 2 * p + e, k = 16 * ks + (out ? ck_result_k(h, j) : 8 * h + j);
      const float v = (out ? pi[(size_t)k * d + n] : pi[(size_t)n * d + k]) * f;
      const __half a = __float2half_rn(v), b = __float2half_rn(v - __half2float(a));
      hi[p] |= (uint32_t)__half_as_ushort(a) << (16 * e);
      lo[p] |= (uint32_t)__half_as_ushort(b) << (16 * e);
    }
  }
  uint4* at = to + (size_t)(out ? 2 * per : 0) + i;
  at[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
  at[per] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
}
int akv_prepare_chunk(int d, void* prep, hipStream_t stream) {
  if (d == 512) return AKV_OK;
  ck_tables_kernel<<<(d * d / 4 + 255) / 256, 256, 0, stream>>>((const float*)prep, d, (const akv_prep_scale*)((const char*)prep + AKV_PREP_SCALE_OFFSET(d)),
                                                               (uint4*)((char*)prep + AKV_PREP_CHUNK_OFFSET(d)));
  AKV_LAUNCH_CHECK("ck_tables_kernel");
  return AKV_OK;
}

extern "C" size_t akv_paged_chunk_attn_workspace_bytes(int d) { return d == 64 || d == 128 || d == 256 ? ck_scratch_layout(d).bytes : 0; }

extern "C" int akv_paged_chunk_attn(const void* query, int dtype, int64_t qs_tok, int64_t qs_head,
                                    const uint8_t* k_packed, int64_t kps_blk, int64_t kps_pos, int64_t kps_head, const float* k_norms, int64_t kns_blk, int64_t kns_pos, int64_t kns_head,
                                    const uint8_t* v_packed, int64_t vps_blk, int64_t vps_pos, int64_t vps_head, const float* v_norms, int64_t vns_blk, int64_t vns_pos, int64_t vns_head,
                                    const void* block_tables, int bt_itype, int64_t bt_stride, const void* context_lens, int cl_itype,
                                    const void* query_starts, int qs_itype, const void* rot_prep, const float* centroids, int bits,
                                    void* out, int64_t os_tok, int64_t os_head, int zero_tail,
                                    int num_seqs, int64_t num_tokens, int num_q_heads, int num_kv_heads, int d, int block_size,
                                    int64_t num_blocks, int64_t max_blocks_per_seq, int max_query_len, float scale,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  const char* name = "akv_paged_chunk_attn";
  const int rc = ck_check_batch(name, query, dtype, block_tables, bt_itype, context_lens, cl_itype, query_starts, qs_itype, out, num_seqs, num_tokens,
                                num_q_heads, num_kv_heads, d, block_size, num_blocks, max_blocks_per_seq, scale);
  AKV_REQUIRE(rc || (bits >= 2 && bits <= 4), "%s: bits must be 2, 3 or 4, got %d", name, bits);
  if (rc || num_tokens == 0) return rc;
  AKV_REQUIRE(rot_prep && centroids, "%s: null pointer", name);
  AKV_REQUIRE(num_blocks == 0 || (k_packed && v_packed && k_norms && v_norms), "%s: null pointer", name);
  if (!ck_aligned(query, 16) || !ck_aligned(out, 8) || ((qs_tok | qs_head) & 7) || ((os_tok | os_head) & 3))
    return akv_fail(AKV_ERR_UNSUPPORTED, "%s: queries must lie at multiples of 16 bytes, outputs of 8", name);
  if (!ck_aligned(k_packed, 4) || !ck_aligned(v_packed, 4) || ((kps_blk | kps_pos | kps_head | vps_blk | vps_pos | vps_head) & 3))
    return akv_fail(AKV_ERR_UNSUPPORTED, "%s: packed rows must lie at multiples of 4 bytes", name);
  const size_t need = ck_scratch_layout(d).bytes;
  if (!workspace || workspace_bytes < need || !ck_aligned(workspace, 256)) return akv_fail(AKV_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", name, need);
  ck_args a = {};
  a.q = query; a.qs_tok = qs_tok; a.qs_head = qs_head;
  a.k = k_packed; a.k_blk = kps_blk; a.k_pos = kps_pos; a.k_head = kps_head;
  a.v = v_packed; a.v_blk = vps_blk; a.v_pos = vps_pos; a.v_head = vps_head;
  a.kn = k_norms; a.kn_blk = kns_blk; a.kn_pos = kns_pos; a.kn_head = kns_head;
  a.vn = v_norms; a.vn_blk = vns_blk; a.vn_pos = vns_pos; a.vn_head = vns_head;
  a.centroids = centroids;
  a.kv_alike = kps_blk == vps_blk && kps_pos == vps_pos && kps_head == vps_head && kns_blk == vns_blk && kns_pos == vns_pos && kns_head == vns_head;
  a.turn_in = (const uint4*)((const char*)rot_prep + AKV_PREP_CHUNK_OFFSET(d));
  a.turn_out = a.turn_in + (size_t)d * d / 4;
  a.turn_scale = (const akv_prep_scale*)((const char*)rot_prep + AKV_PREP_SCALE_OFFSET(d));
  a.dtype = dtype;
  a.out = out; a.os_tok = os_tok; a.os_head = os_head;
  a.tables = block_tables; a.tables_it = bt_itype; a.bt_stride = bt_stride;
  a.lens = context_lens; a.lens_it = cl_itype; a.starts = query_starts; a.starts_it = qs_itype;
  a.S = num_seqs; a.T = (int)num_tokens; a.QH = num_q_heads; a.KVH = num_kv_heads; a.G = num_q_heads / num_kv_heads;
  a.block_size = block_size; a.bs_recip = ck_reciprocal(block_size);
  a.max_blocks = num_blocks > 0 ? max_blocks_per_seq : 0; a.num_blocks = num_blocks;
  a.tail = zero_tail; a.scale2 = scale * 1.44269504088896341f;
  const hipStream_t s = (hipStream_t)stream;
#define CK_CASE(DIM)                                                                             \
  if (d == DIM) return bits == 4   ? ck_launch<DIM, 4>(a, max_query_len, workspace, s)           \
                       : bits == 3 ? ck_launch<DIM, 3>(a, max_query_len, workspace, s)           \
                                   : ck_launch<DIM, 2>(a, max_query_len, workspace, s);
  CK_CASE(64) CK_CASE(128) CK_CASE(256)
#undef CK_CASE
  return AKV_ERR_UNSUPPORTED;
}
