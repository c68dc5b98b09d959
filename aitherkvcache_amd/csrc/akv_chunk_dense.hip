// akv_dense_chunk_attn: attention of a chunk of new tokens over a paged cache of float16 or bfloat16 rows.
#include "akv_chunk_kernels.h"

extern "C" size_t akv_dense_chunk_attn_workspace_bytes(int d) { return d == 64 || d == 128 || d == 256 ? ck_scratch_layout(d).bytes : 0; }

extern "C" int akv_dense_chunk_attn(const void* query, int dtype, int64_t qs_tok, int64_t qs_head,
                                    const void* key_cache, int64_t ks_blk, int64_t ks_pos, int64_t ks_head,
                                    const void* value_cache, int64_t vs_blk, int64_t vs_pos, int64_t vs_head,
                                    const void* block_tables, int bt_itype, int64_t bt_stride, const void* context_lens, int cl_itype,
                                    const void* query_starts, int qs_itype, void* out, int64_t os_tok, int64_t os_head, int zero_tail,
                                    int num_seqs, int64_t num_tokens, int num_q_heads, int num_kv_heads, int d, int block_size,
                                    int64_t num_blocks, int64_t max_blocks_per_seq, int window, int max_query_len, float scale,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  const char* name = "akv_dense_chunk_attn";
  const int rc = ck_check_batch(name, query, dtype, block_tables, bt_itype, context_lens, cl_itype, query_starts, qs_itype, out, num_seqs, num_tokens,
                                num_q_heads, num_kv_heads, d, block_size, num_blocks, max_blocks_per_seq, scale);
  if (rc || num_tokens == 0) return rc;
  AKV_REQUIRE(num_blocks == 0 || (key_cache && value_cache), "%s: null pointer", name);
  AKV_REQUIRE(window >= 0, "%s: negative window", name);
  if (!ck_aligned(query, 16) || !ck_aligned(key_cache, 16) || !ck_aligned(value_cache, 16) || !ck_aligned(out, 8) || ((qs_tok | qs_head | ks_blk | ks_pos | ks_head | vs_blk | vs_pos | vs_head) & 7) || ((os_tok | os_head) & 3))
    return akv_fail(AKV_ERR_UNSUPPORTED, "%s: rows must lie at multiples of 16 bytes (outputs of 8)", name);
  if (!workspace || workspace_bytes < ck_scratch_layout(d).bytes || !ck_aligned(workspace, 256)) return akv_fail(AKV_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", name, ck_scratch_layout(d).bytes);
  ck_args a = {};
  a.q = query; a.qs_tok = qs_tok; a.qs_head = qs_head;
  a.k = (const uint8_t*)key_cache; a.k_blk = 2 * ks_blk; a.k_pos = 2 * ks_pos; a.k_head = 2 * ks_head;
  a.v = (const uint8_t*)value_cache; a.v_blk = 2 * vs_blk; a.v_pos = 2 * vs_pos; a.v_head = 2 * vs_head;
  a.tables = block_tables; a.tables_it = bt_itype; a.bt_stride = bt_stride;
  a.lens = context_lens; a.lens_it = cl_itype; a.starts = query_starts; a.starts_it = qs_itype;
  a.out = out; a.os_tok = os_tok; a.os_head = os_head;
  a.S = num_seqs; a.T = (int)num_tokens; a.QH = num_q_heads; a.KVH = num_kv_heads; a.G = num_q_heads / num_kv_heads;
  a.block_size = block_size; a.bs_recip = ck_reciprocal(block_size);
  a.max_blocks = num_blocks > 0 ? max_blocks_per_seq : 0; a.num_blocks = num_blocks;
  a.kv_alike = ks_blk == vs_blk && ks_pos == vs_pos && ks_head == vs_head;
  // a window that reaches as far as the tables (and lengths, ck_ctx_of) is none
  const int64_t longest = a.max_blocks * block_size;
  a.window = window < (longest < 0x7fff0000 ? longest : 0x7fff0000) ? window : 0;
  if (a.window > 1 << 30) return akv_fail(AKV_ERR_UNSUPPORTED, "%s: windows of more than 2^30 tokens over longer tables", name);
  a.tail = zero_tail; a.scale2 = scale * 1.44269504088896341f;
  const hipStream_t s = (hipStream_t)stream;
#define CK_CASE(DIM) if (d == DIM) return dtype == AKV_F16 ? ck_launch<DIM, CK_F16>(a, max_query_len, workspace, s) : ck_launch<DIM, CK_BF16>(a, max_query_len, workspace, s);
  CK_CASE(64) CK_CASE(128) CK_CASE(256)
#undef CK_CASE
  return AKV_ERR_UNSUPPORTED;
}
