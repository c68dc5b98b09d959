// akv_paged_chunk_attn: attention of a chunk of new tokens over the packed cache.
#include "akv_chunk_rotate.h"

struct ck_packed_layout { size_t scratch, q, fac, out, bytes; };
static inline ck_packed_layout ck_packed_scratch(int64_t T, int QH, int D) {
  ck_packed_layout w;
  w.scratch = 0;
  w.q = akv_align256(ck_scratch_layout(D).bytes);
  w.fac = w.q + akv_align256((size_t)T * QH * D * 2);
  w.out = w.fac + akv_align256((size_t)T * QH * 4);
  w.bytes = w.out + akv_align256((size_t)T * QH * D * 4);
  return w;
}
extern "C" size_t akv_paged_chunk_attn_workspace_bytes(int64_t num_tokens, int num_q_heads, int d) {
  return num_tokens >= 0 && num_q_heads > 0 && (d == 64 || d == 128 || d == 256) ? ck_packed_scratch(num_tokens, num_q_heads, d).bytes : 0;
}

template <int D, int BITS>
static int ck_run(ck_args a, int dtype, const void* prep, void* out, int64_t os_tok, int64_t os_head, int most_new, void* workspace, hipStream_t stream) {
  const ck_packed_layout w = ck_packed_scratch(a.T, a.QH, D);
  const float* pi = (const float*)prep;
  const akv_prep_scale* ps = (const akv_prep_scale*)((const char*)prep + AKV_PREP_SCALE_OFFSET(D));
  uint16_t* qr = (uint16_t*)((char*)workspace + w.q);
  float* fac = (float*)((char*)workspace + w.fac);
  float* turned = (float*)((char*)workspace + w.out);
  const int64_t rows = (int64_t)a.T * a.QH, tiles = (rows + 15) / 16;
  const int most = ck_groups(4) / (D / 64);
  const dim3 grid((unsigned)(tiles < most ? tiles : most), D / 64);
  const void* q = a.q;
  const int64_t qs_tok = a.qs_tok, qs_head = a.qs_head;
  if (dtype == AKV_F16) ck_rotate_kernel<D, AKV_F16, true, AKV_F16><<<grid, 256, 0, stream>>>(q, qs_tok, qs_head, rows, a.QH, pi, ps, qr, 0, 0, fac, a.scale2, a.starts, a.starts_it, a.S, a.tail);
  else ck_rotate_kernel<D, AKV_BF16, true, AKV_F16><<<grid, 256, 0, stream>>>(q, qs_tok, qs_head, rows, a.QH, pi, ps, qr, 0, 0, fac, a.scale2, a.starts, a.starts_it, a.S, a.tail);
  AKV_LAUNCH_CHECK("ck_rotate_kernel");
  a.q = qr; a.qs_tok = (int64_t)a.QH * D; a.qs_head = D; a.qfac = fac;
  a.out = turned; a.os_tok = (int64_t)a.QH * D; a.os_head = D;
  const int rc = ck_launch<D, BITS>(a, most_new, (char*)workspace + w.scratch, stream);
  if (rc) return rc;
  const float* pit = pi + (size_t)D * D;
  if (dtype == AKV_F16) ck_rotate_kernel<D, AKV_F32, false, AKV_F16><<<grid, 256, 0, stream>>>(turned, a.os_tok, a.os_head, rows, a.QH, pit, ps, out, os_tok, os_head, nullptr, 0.f, a.starts, a.starts_it, a.S, a.tail);
  else ck_rotate_kernel<D, AKV_F32, false, AKV_BF16><<<grid, 256, 0, stream>>>(turned, a.os_tok, a.os_head, rows, a.QH, pit, ps, out, os_tok, os_head, nullptr, 0.f, a.starts, a.starts_it, a.S, a.tail);
  AKV_LAUNCH_CHECK("ck_rotate_kernel");
  return AKV_OK;
}

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
  if (!ck_aligned(k_packed, 4) || !ck_aligned(v_packed, 4) || ((kps_blk | kps_pos | kps_head | vps_blk | vps_pos | vps_head) & 3))
    return akv_fail(AKV_ERR_UNSUPPORTED, "%s: packed rows must lie at multiples of 4 bytes", name);
  const size_t need = ck_packed_scratch(num_tokens, num_q_heads, d).bytes;
  if (!workspace || workspace_bytes < need || !ck_aligned(workspace, 256)) return akv_fail(AKV_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", name, need);
  ck_args a = {};
  a.q = query; a.qs_tok = qs_tok; a.qs_head = qs_head;
  a.k = k_packed; a.k_blk = kps_blk; a.k_pos = kps_pos; a.k_head = kps_head;
  a.v = v_packed; a.v_blk = vps_blk; a.v_pos = vps_pos; a.v_head = vps_head;
  a.kn = k_norms; a.kn_blk = kns_blk; a.kn_pos = kns_pos; a.kn_head = kns_head;
  a.vn = v_norms; a.vn_blk = vns_blk; a.vn_pos = vns_pos; a.vn_head = vns_head;
  a.centroids = centroids;
  a.tables = block_tables; a.tables_it = bt_itype; a.bt_stride = bt_stride;
  a.lens = context_lens; a.lens_it = cl_itype; a.starts = query_starts; a.starts_it = qs_itype;
  a.S = num_seqs; a.T = (int)num_tokens; a.QH = num_q_heads; a.KVH = num_kv_heads; a.G = num_q_heads / num_kv_heads;
  a.block_size = block_size; a.bs_recip = ck_reciprocal(block_size);
  a.max_blocks = num_blocks > 0 ? max_blocks_per_seq : 0; a.num_blocks = num_blocks;
  a.tail = zero_tail; a.scale2 = scale * 1.44269504088896341f;
  const hipStream_t s = (hipStream_t)stream;
#define CK_CASE(DIM)                                                                                                                  \
  if (d == DIM) return bits == 4   ? ck_run<DIM, 4>(a, dtype, rot_prep, out, os_tok, os_head, max_query_len, workspace, s)            \
                       : bits == 3 ? ck_run<DIM, 3>(a, dtype, rot_prep, out, os_tok, os_head, max_query_len, workspace, s)            \
                                   : ck_run<DIM, 2>(a, dtype, rot_prep, out, os_tok, os_head, max_query_len, workspace, s);
  CK_CASE(64) CK_CASE(128) CK_CASE(256)
#undef CK_CASE
  return AKV_ERR_UNSUPPORTED;
}
