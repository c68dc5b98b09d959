"""Paged decode attention straight from the TurboQuant-compressed cache, in the rotated
domain: q' = Pi q once, score_t = |k_t| <q', c[codes_t]> / sqrt(d), out = Pi^T (sum_t w_t |v_t|
c[codes_t]) -- the computation of the reference's TQPagedAttentionRef
(aither_kvcache/fused_attention.py:91-185) behind the interface of its TQPagedAttention
(:538-748).  Pre-rotation, the stream-K split over long contexts, the merge and the inverse
rotation all run on the GPU through one C-ABI call; 2-, 3- and 4-bit caches are handled by
kernels (the reference runs a Python loop for 2/3-bit).
"""
import math
import os
from typing import Optional

import torch

from . import _lib

HAS_HIP = _lib.available()
HAS_TRITON = HAS_HIP


class TQPagedAttention:
    """attn = TQPagedAttention(tq, num_query_heads=32)
    out = attn.forward(query, k_packed, k_norms, v_packed, v_norms, block_tables, context_lens)
    """

    # Kept for call compatibility (fused_attention.py:632-633).  The split over the context is
    # decided on the device from context_lens, so these two no longer steer anything.
    SPLITK_THRESHOLD = int(os.environ.get("AITHER_TQ_SPLITK_THRESHOLD", "64"))
    SPLITK_NUM_SPLITS = int(os.environ.get("AITHER_TQ_SPLITK_SPLITS", "16"))

    def __init__(self, tq, num_query_heads: int, block_selector=None):
        self._tq = tq
        self.rotation = tq.rotation
        self.centroids = tq.centroids
        self.scale = 1.0 / math.sqrt(tq.head_dim)   # always 1/sqrt(d), as the reference (:563)
        self.head_dim = tq.head_dim
        self.num_levels = tq.num_levels
        self.bits = tq.bits
        self.packed_dim = tq._packed_dim
        self.num_query_heads = num_query_heads
        self._block_selector = block_selector
        self._workspace: Optional[torch.Tensor] = None
        self._use_hip = True
        self._use_triton = False

    def _get_workspace(self, num_seqs: int, device) -> torch.Tensor:
        need = _lib.lib().akv_paged_attn_workspace_bytes(num_seqs, self.num_query_heads, self.head_dim)
        ws = self._workspace
        if ws is None or ws.numel() < need or ws.device != device:
            ws = torch.empty(need, dtype=torch.uint8, device=device)
            self._workspace = ws
        return ws

    def forward_no_alloc(self, query, k_packed, k_norms, v_packed, v_norms, block_tables, context_lens,
                         out: torch.Tensor, block_size: int = 16, num_kv_heads: Optional[int] = None) -> torch.Tensor:
        """forward() for callers that may not allocate (under graph capture, in a loop that forbids
        it): the result goes into `out` (same shape as `query`, float16 / bfloat16 / float32) and the
        library works in a fixed scratch array of its own instead of a workspace tensor.  Inputs must
        already be in the form the kernels take (float query with contiguous rows, float32 norms,
        contiguous table rows); batches too large for the built-in array raise.  No block selector."""
        if self._block_selector is not None:
            raise ValueError("forward_no_alloc does not run the block selector (it allocates)")
        return self.forward(query, k_packed, k_norms, v_packed, v_norms, block_tables, context_lens,
                            block_size, num_kv_heads, _static_out=out)

    def forward(self, query, k_packed, k_norms, v_packed, v_norms, block_tables, context_lens,
                block_size: int = 16, num_kv_heads: Optional[int] = None, _static_out=None) -> torch.Tensor:
        """query [num_seqs, num_query_heads, head_dim] -> same shape and dtype.

        k/v_packed [num_blocks, block_size, num_kv_heads, >= packed_dim] uint8 (may be strided
        views with 4-byte aligned rows), k/v_norms [num_blocks, block_size, num_kv_heads] float32,
        block_tables [num_seqs, max_blocks_per_seq] int32/int64, context_lens [num_seqs]."""
        tq = self._tq
        if tq.rotation is not self.rotation:     # the quantizer's matrix was reassigned: follow it
            self.rotation = tq.rotation
        if _static_out is None and self._block_selector is None and self._workspace is not None:
            out = _lib.calls().uniform_attention(query, k_packed, k_norms, v_packed, v_norms, block_tables, context_lens, self.centroids,
                                                 self._workspace, tq.prepared_rotation().ptr, num_kv_heads, self.num_query_heads,
                                                 self.head_dim, self.packed_dim, self.bits, block_size, self.scale)
            if out is not None:
                if type(out) is int:
                    _lib.check(out)
                self._last_static = None
                return out
        if num_kv_heads is None:
            num_kv_heads = k_packed.shape[2]
        if self._block_selector is not None:
            # as in the reference (:659-668): even / odd coordinates of the rotated query score the blocks,
            # the kernel then walks the filtered table
            q_rot = torch.matmul(query.float(), self.rotation.T)
            block_tables, context_lens = self._block_selector.select(
                q_rot[..., 0::2].contiguous(), q_rot[..., 1::2].contiguous(), block_tables, context_lens,
                query.shape[1] // num_kv_heads, block_size)
        dev = _lib.require_gpu(query, k_packed, k_norms, v_packed, v_norms, block_tables, context_lens)
        num_seqs, num_q_heads, head_dim = query.shape
        if head_dim != self.head_dim or num_q_heads != self.num_query_heads:
            raise ValueError(f"query shape {tuple(query.shape)} does not match heads="
                             f"{self.num_query_heads}, head_dim={self.head_dim}")
        q = query
        if q.dtype not in (torch.float16, torch.bfloat16, torch.float32):
            q = q.float()
        if q.stride(-1) != 1:
            q = q.contiguous()
        if _static_out is not None:
            out = _static_out
            if out.shape != query.shape or out.stride(-1) != 1 or not out.is_cuda:
                raise ValueError("out must be a device tensor of the query's shape with contiguous rows")
        else:
            out = torch.empty((num_seqs, num_q_heads, head_dim), dtype=q.dtype, device=dev)
        if num_seqs == 0:
            return out if _static_out is not None else out.to(query.dtype)
        for name, t in (("k_packed", k_packed), ("v_packed", v_packed)):
            if t.dtype != torch.uint8 or t.stride(-1) != 1 or t.shape[-1] < self.packed_dim:
                raise ValueError(f"{name} must be uint8 with contiguous rows of >= {self.packed_dim} bytes")
        _lib.check_caches(block_size, num_kv_heads, k_packed, k_norms, v_packed, v_norms)
        _lib.check_batch(num_seqs, block_tables, context_lens)
        if _static_out is not None and (k_norms.dtype != torch.float32 or v_norms.dtype != torch.float32):
            raise ValueError("forward_no_alloc needs float32 norms (a conversion would allocate)")
        k_norms = k_norms if k_norms.dtype == torch.float32 else k_norms.float()
        v_norms = v_norms if v_norms.dtype == torch.float32 else v_norms.float()
        bt = block_tables if block_tables.stride(-1) == 1 else block_tables.contiguous()
        cl = context_lens if context_lens.is_contiguous() else context_lens.contiguous()
        num_blocks = min(k_packed.shape[0], k_norms.shape[0], v_packed.shape[0], v_norms.shape[0])
        if _static_out is not None:
            if q is not query or bt is not block_tables or cl is not context_lens:
                raise ValueError("forward_no_alloc needs inputs that take no conversion")
            _lib.check(_lib.lib().akv_paged_attn_static(
                q.data_ptr(), _lib.dtype_code(q), q.stride(0), q.stride(1),
                k_packed.data_ptr(), k_packed.stride(0), k_packed.stride(1), k_packed.stride(2),
                k_norms.data_ptr(), k_norms.stride(0), k_norms.stride(1), k_norms.stride(2),
                v_packed.data_ptr(), v_packed.stride(0), v_packed.stride(1), v_packed.stride(2),
                v_norms.data_ptr(), v_norms.stride(0), v_norms.stride(1), v_norms.stride(2),
                bt.data_ptr(), _lib.itype_code(bt), bt.stride(0), cl.data_ptr(), _lib.itype_code(cl),
                self._tq.prepared_rotation().ptr, self.centroids.data_ptr(), self.bits,
                out.data_ptr(), _lib.dtype_code(out), out.stride(0), out.stride(1),
                num_seqs, num_q_heads, num_kv_heads, head_dim, block_size, num_blocks, bt.shape[1], self.scale,
                _lib.stream_ptr(dev)))
            self._last_static = dev
            return out
        self._last_static = None
        ws = self._get_workspace(num_seqs, dev)
        _lib.check(_lib.lib().akv_paged_attn(
            q.data_ptr(), _lib.dtype_code(q), q.stride(0), q.stride(1),
            k_packed.data_ptr(), k_packed.stride(0), k_packed.stride(1), k_packed.stride(2),
            k_norms.data_ptr(), k_norms.stride(0), k_norms.stride(1), k_norms.stride(2),
            v_packed.data_ptr(), v_packed.stride(0), v_packed.stride(1), v_packed.stride(2),
            v_norms.data_ptr(), v_norms.stride(0), v_norms.stride(1), v_norms.stride(2),
            bt.data_ptr(), _lib.itype_code(bt), bt.stride(0), cl.data_ptr(), _lib.itype_code(cl),
            tq.prepared_rotation().ptr, self.centroids.data_ptr(), self.bits,
            out.data_ptr(), _lib.dtype_code(out), out.stride(0), out.stride(1),
            num_seqs, num_q_heads, num_kv_heads, head_dim, block_size, num_blocks, bt.shape[1], self.scale,
            ws.data_ptr(), ws.numel(), _lib.stream_ptr(dev)))
        return out if out.dtype == query.dtype else out.to(query.dtype)

    def forward_chunk(self, query, k_packed, k_norms, v_packed, v_norms, block_tables, context_lens, query_start_loc,
                      block_size: int = 16, num_kv_heads: Optional[int] = None, out: Optional[torch.Tensor] = None,
                      max_query_len: Optional[int] = None) -> torch.Tensor:
        """Causal attention of a chunk of new tokens a sequence (a draft to verify, a prompt that goes on) over the packed cache,
        which holds the chunk's own tokens already; a chunk of one token is forward().

        query           [num_tokens, num_query_heads, head_dim] float16 / bfloat16, the chunks of all sequences one after the other
        query_start_loc [num_seqs + 1]: sequence i owns query rows query_start_loc[i] .. query_start_loc[i + 1] - 1, the newest of
                        its context_lens[i] tokens; token j of n stands at position context_len - n + j and sees the
                        keys up to there (none: zeros)
        out             where the result goes (shape and type of query; rows before the first sequence or behind the last are left
                        as they were); without it a new tensor, zero in such rows
        max_query_len   the longest chunk, if known on the host: what is launched goes by it, the result but for its last rounding does not

        Caches, norms and tables as in forward(); head_dim 64, 128 or 256, rows at multiples of 4 bytes.  No block selector.
        Norms of the sequences' tokens must be finite; past a context the caches and tables may hold anything.
        Rounded on the way, whatever the query's type: levels and weights to float16 (weights also by 2^-30 of the row's largest),
        rotated queries to one float16 term, or to two where the query is float16 or chunks are short; sums are float32."""
        from .chunk_attention import _check_out, _longest, check_chunk, check_query
        if self._block_selector is not None:
            raise ValueError("forward_chunk does not run the block selector")
        tq = self._tq
        if tq.rotation is not self.rotation:
            self.rotation = tq.rotation
        if query.is_cuda:
            result = _lib.calls().packed_chunk(query, k_packed, k_norms, v_packed, v_norms, block_tables, context_lens, query_start_loc,
                                               self.centroids, tq.prepared_rotation().ptr, num_kv_heads, self.num_query_heads, self.head_dim,
                                               self.packed_dim, self.bits, block_size, max_query_len, self.scale, out)
            if result is not None:
                return result if type(result) is not int else _lib.check(result)
        check_query(query)
        if k_packed.dim() != 4 or v_packed.dim() != 4 or k_norms.dim() != 3 or v_norms.dim() != 3:
            raise ValueError("expected caches [blocks, block_size, heads, bytes] and norms [blocks, block_size, heads]")
        dev = _lib.require_gpu(query, k_packed, k_norms, v_packed, v_norms, block_tables, context_lens, query_start_loc, out, self.centroids, tq.rotation)
        if self.centroids.numel() != 1 << self.bits:
            raise ValueError(f"a codebook of {self.bits} bits has {1 << self.bits} levels, got shape {tuple(self.centroids.shape)}")
        centroids = self.centroids.float().contiguous()
        num_tokens, num_q_heads, d = query.shape
        if d != self.head_dim or num_q_heads != self.num_query_heads:
            raise ValueError(f"query shape {tuple(query.shape)} does not match heads={self.num_query_heads}, head_dim={self.head_dim}")
        if num_kv_heads is None:
            num_kv_heads = k_packed.shape[2]
        for name, t in (("k_packed", k_packed), ("v_packed", v_packed)):
            if t.dtype != torch.uint8 or t.stride(-1) != 1 or t.shape[-1] < self.packed_dim:
                raise ValueError(f"{name} must be uint8 with contiguous rows of >= {self.packed_dim} bytes")
        _lib.check_caches(block_size, num_kv_heads, k_packed, k_norms, v_packed, v_norms)
        num_seqs, q, bt, lens, starts = check_chunk(query, num_kv_heads, block_tables, context_lens, query_start_loc)
        k_norms = k_norms if k_norms.dtype == torch.float32 else k_norms.float()
        v_norms = v_norms if v_norms.dtype == torch.float32 else v_norms.float()
        if out is not None:
            _check_out("out", out, query)
        result = out if out is not None else torch.empty((num_tokens, num_q_heads, d), dtype=query.dtype, device=dev)
        L = _lib.lib()
        ws = torch.empty(L.akv_paged_chunk_attn_workspace_bytes(d), dtype=torch.uint8, device=dev)
        blocks = min(k_packed.shape[0], k_norms.shape[0], v_packed.shape[0], v_norms.shape[0])
        with _lib.on_device(dev):
            _lib.check(L.akv_paged_chunk_attn(
                q.data_ptr(), _lib.dtype_code(q), q.stride(0), q.stride(1),
                k_packed.data_ptr(), k_packed.stride(0), k_packed.stride(1), k_packed.stride(2),
                k_norms.data_ptr(), k_norms.stride(0), k_norms.stride(1), k_norms.stride(2),
                v_packed.data_ptr(), v_packed.stride(0), v_packed.stride(1), v_packed.stride(2),
                v_norms.data_ptr(), v_norms.stride(0), v_norms.stride(1), v_norms.stride(2),
                bt.data_ptr(), _lib.itype_code(bt), bt.stride(0), lens.data_ptr(), _lib.itype_code(lens),
                starts.data_ptr(), _lib.itype_code(starts), tq.prepared_rotation().ptr, centroids.data_ptr(), self.bits,
                result.data_ptr(), result.stride(0), result.stride(1), int(out is None),
                num_seqs, num_tokens, num_q_heads, num_kv_heads, d, block_size, blocks, bt.shape[1],
                _longest(max_query_len), self.scale, ws.data_ptr(), ws.numel(), _lib.stream_ptr(dev)))
        return result

    def key_weights(self, query, k_packed, k_norms, block_tables, context_lens, query_start_loc, block_size: int = 16,
                    num_kv_heads: Optional[int] = None, accumulated: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The softmax weight that every key of the packed cache gets from its sequence's newest tokens (causal, as forward_chunk weighs
        them; a chunk of one token as forward), summed over these tokens and over the query heads of a kv head:
        [num_seqs, num_kv_heads, length] float32, a key at its position.

        query, k_packed, k_norms, block_tables, context_lens, query_start_loc as in forward_chunk
        accumulated  as in paged_key_weights: float32, added to and returned; without it a new tensor as long as the tables

        head_dim 64, 128 or 256, rows at multiples of 4 bytes, at most 65535 sequences; queries and norms of the sequences' tokens must be finite.  Scores, weights and sums
        are float32, levels and rotated queries two float16 terms each (2^-22)."""
        from .chunk_attention import check_chunk, check_query
        from .eviction import weights_for
        tq = self._tq
        if tq.rotation is not self.rotation:
            self.rotation = tq.rotation
        if query.is_cuda:
            result = _lib.calls().packed_weights(query, k_packed, k_norms, block_tables, context_lens, query_start_loc, self.centroids, accumulated,
                                                 tq.prepared_rotation().ptr, num_kv_heads, self.num_query_heads, self.head_dim, self.packed_dim,
                                                 self.bits, block_size, self.scale)
            if result is not None:
                return result if type(result) is not int else _lib.check(result)
        check_query(query)
        if k_packed.dim() != 4 or k_norms.dim() != 3:
            raise ValueError("expected a cache [blocks, block_size, heads, bytes] and norms [blocks, block_size, heads]")
        num_tokens, num_q_heads, d = query.shape
        if d != self.head_dim or num_q_heads != self.num_query_heads:
            raise ValueError(f"query shape {tuple(query.shape)} does not match heads={self.num_query_heads}, head_dim={self.head_dim}")
        if self.centroids.numel() != 1 << self.bits:
            raise ValueError(f"a codebook of {self.bits} bits has {1 << self.bits} levels, got shape {tuple(self.centroids.shape)}")
        if k_packed.dtype != torch.uint8 or k_packed.stride(-1) != 1 or k_packed.shape[-1] < self.packed_dim:
            raise ValueError(f"k_packed must be uint8 with contiguous rows of >= {self.packed_dim} bytes")
        if num_kv_heads is None:
            num_kv_heads = k_packed.shape[2]
        if block_size < 1:
            raise ValueError(f"block_size {block_size}")
        _lib.check_caches(block_size, num_kv_heads, k_packed, k_norms)
        num_seqs, q, bt, lens, starts = check_chunk(query, num_kv_heads, block_tables, context_lens, query_start_loc)
        dev = _lib.require_gpu(query, k_packed, k_norms, block_tables, context_lens, query_start_loc, accumulated, self.centroids, tq.rotation)
        centroids = self.centroids.float().contiguous()
        k_norms = k_norms if k_norms.dtype == torch.float32 else k_norms.float()
        w = weights_for(accumulated, num_seqs, num_kv_heads, bt.shape[1] * block_size, dev)
        L = _lib.lib()
        ws = torch.empty(L.akv_packed_key_weights_workspace_bytes(num_tokens, num_seqs, num_q_heads, num_kv_heads, d, w.shape[2]), dtype=torch.uint8, device=dev)
        with _lib.on_device(dev):
            _lib.check(L.akv_packed_key_weights(
                q.data_ptr(), _lib.dtype_code(q), q.stride(0), q.stride(1), k_packed.data_ptr(), k_packed.stride(0), k_packed.stride(1), k_packed.stride(2),
                k_norms.data_ptr(), k_norms.stride(0), k_norms.stride(1), k_norms.stride(2), bt.data_ptr(), _lib.itype_code(bt), bt.stride(0),
                lens.data_ptr(), _lib.itype_code(lens), starts.data_ptr(), _lib.itype_code(starts), tq.prepared_rotation().ptr, centroids.data_ptr(), self.bits,
                w.data_ptr(), w.stride(0), w.stride(1), w.shape[2], int(accumulated is not None), num_seqs, num_tokens, num_q_heads, num_kv_heads, d, block_size,
                min(k_packed.shape[0], k_norms.shape[0]), bt.shape[1], self.scale, ws.data_ptr(), ws.numel(), _lib.stream_ptr(dev)))
        return w

    def last_call_status(self) -> int:
        """0 when the most recent forward() / forward_no_alloc() ran clean; bit 0 set when it failed on the device (its
        outputs are NaN).  Synchronises the stream."""
        if getattr(self, "_last_static", None) is not None:
            return _lib.attn_status_static(self._last_static)       # the library's built-in scratch array
        return _lib.attn_status(self._workspace)


class _RotationHolder:
    """What TQPagedAttention reads from a quantizer, for callers that bring the rotation and the codebook
    themselves."""

    def __init__(self, rotation: torch.Tensor, centroids: torch.Tensor, head_dim: int, bits: int):
        from .packing import packed_size
        self.rotation = rotation
        self.centroids = centroids.to(torch.float32).contiguous()
        self.head_dim = head_dim
        self.bits = bits
        self.num_levels = 1 << bits
        self._packed_dim = packed_size(head_dim, bits)

    def prepared_rotation(self):
        from .quantizer import prepared_rotation_for
        return prepared_rotation_for(self.rotation)


class TQPagedAttentionRef:
    """Constructor and forward() of the reference's pure-PyTorch class (fused_attention.py:53-185): rotation
    [head_dim, head_dim], centroids [2**bits], an explicit score scale, fixed head counts and block size.
    Here it runs the same HIP kernels as TQPagedAttention (there is no CPU path: tensors must live on the GPU);
    the results are those the golden vectors of the reference's class are checked against."""

    def __init__(self, rotation: torch.Tensor, centroids: torch.Tensor, scale: float, num_kv_heads: int,
                 num_query_heads: int, head_dim: int, block_size: int, bits: int = 4):
        self.rotation = rotation
        self.centroids = centroids
        self.scale = scale
        self.num_kv_heads = num_kv_heads
        self.num_query_heads = num_query_heads
        self.gqa_ratio = num_query_heads // num_kv_heads
        self.head_dim = head_dim
        self.block_size = block_size
        self.bits = bits
        self._impl = TQPagedAttention(_RotationHolder(rotation, centroids, head_dim, bits), num_query_heads)
        self._impl.scale = float(scale)

    def forward(self, query, k_packed, k_norms, v_packed, v_norms, block_tables, context_lens) -> torch.Tensor:
        """query [num_seqs, num_query_heads, head_dim] -> same shape and dtype."""
        return self._impl.forward(query, k_packed, k_norms, v_packed, v_norms, block_tables, context_lens,
                                  block_size=self.block_size, num_kv_heads=self.num_kv_heads)

