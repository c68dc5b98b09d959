"""Attention of new tokens over a part of an uncompressed paged cache: each token and kv head reads the blocks whose mean key its query
likes best.

BlockIndex keeps the mean key of every block in 8 bits and selects blocks by it; paged_sparse_attention attends over what was selected.
The reference scores blocks too (aither_kvcache/block_selector.py), for a packed cache, one list a sequence and one token at a time; that is
BlockSelector in block_selector.py.  Here every token of a chunk and every kv head has its own list, and prompts take part.
"""
import math
from typing import Optional

import torch

from . import _lib
from .chunk_attention import _check_out, _check_rows, check_chunk, check_query

__all__ = ["BlockIndex", "paged_sparse_attention"]


class BlockIndex:
    """What the blocks of a cache of keys look like from afar: per block and kv head the mean of its keys in 8 bits.

    codes  [num_blocks, num_kv_heads, head_dim] int8;  scales [num_blocks, num_kv_heads] float32: the mean is codes x scale

    index = BlockIndex(num_blocks, num_kv_heads, head_dim, device)
    index.update(key_cache, block_tables, context_lens, query_start_loc)        # after a chunk's keys have been written
    selected = index.select(query, block_tables, context_lens, query_start_loc, block_size, num_selected=64)
    out = paged_sparse_attention(query, key_cache, value_cache, block_tables, context_lens, query_start_loc, selected)

    head_dim is 64, 128 or 256."""

    def __init__(self, num_blocks: int, num_kv_heads: int, head_dim: int, device):
        if num_blocks < 0 or num_kv_heads < 1 or head_dim < 1:
            raise ValueError(f"{num_blocks} blocks of {num_kv_heads} kv heads of {head_dim}")
        self.num_blocks, self.num_kv_heads, self.head_dim = num_blocks, num_kv_heads, head_dim
        self.codes = torch.zeros(num_blocks, num_kv_heads, head_dim, dtype=torch.int8, device=device)
        self.scales = torch.zeros(num_blocks, num_kv_heads, dtype=torch.float32, device=device)

    def _check(self) -> None:
        shape = (self.num_blocks, self.num_kv_heads, self.head_dim)
        for name, t, dims, dtype in (("codes", self.codes, shape, torch.int8), ("scales", self.scales, shape[:2], torch.float32)):
            if tuple(t.shape) != dims or t.dtype != dtype or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous {dtype} of shape {dims}, got {t.dtype} {tuple(t.shape)}")

    def dequantized(self) -> torch.Tensor:
        """The means as float32, [num_blocks, num_kv_heads, head_dim]."""
        return self.codes * self.scales[..., None]

    def update(self, key_cache: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor,
               query_start_loc: Optional[torch.Tensor] = None) -> None:
        """Take the means of the blocks that the sequences' newest tokens came to, from the keys these blocks hold now.

        key_cache       [num_blocks, block_size, num_kv_heads, head_dim] float16 / bfloat16 (strides honoured)
        block_tables    [num_seqs, blocks] int32 / int64;  context_lens [num_seqs] tokens of a sequence, the newest included
        query_start_loc [num_seqs + 1]: sequence i has query_start_loc[i + 1] - query_start_loc[i] new tokens (the first start may be any:
                        a part of a batch); None: the means of all blocks of every sequence (the cache was filled or rearranged by other means)

        A last block that is not full has the mean of the keys in it; a mean that is not finite is kept as zeros.  Sums are 64 bits."""
        result = _lib.calls().index_update(key_cache, block_tables, context_lens, query_start_loc, self.codes, self.scales, self.num_blocks,
                                           self.num_kv_heads, self.head_dim)
        if result is not None:
            return _lib.check(result)
        _check_rows("key_cache", key_cache, 4)
        if key_cache.dtype not in (torch.float16, torch.bfloat16):
            raise NotImplementedError(f"keys are float16 or bfloat16, got {key_cache.dtype}")
        blocks, block_size, kv_heads, d = key_cache.shape
        if (blocks, kv_heads, d) != (self.num_blocks, self.num_kv_heads, self.head_dim):
            raise ValueError(f"a cache of shape {tuple(key_cache.shape)} does not fit an index of {self.num_blocks} blocks of {self.num_kv_heads} heads of {self.head_dim}")
        self._check()
        dev = _lib.require_gpu(key_cache, block_tables, context_lens, query_start_loc, self.codes, self.scales)
        num_seqs, bt, lens, starts = check_sequences(block_tables, context_lens, query_start_loc)
        # (starts may lie behind the rows of sequences that are not of this call: as many tokens as a batch can have)
        tokens = 0 if starts is None else (1 << 30) - 1
        with _lib.on_device(dev):
            _lib.check(_lib.lib().akv_block_index_update(
                key_cache.data_ptr(), _lib.dtype_code(key_cache), key_cache.stride(0), key_cache.stride(1), key_cache.stride(2),
                bt.data_ptr(), _lib.itype_code(bt), bt.stride(0), lens.data_ptr(), _lib.itype_code(lens),
                None if starts is None else starts.data_ptr(), 0 if starts is None else _lib.itype_code(starts),
                self.codes.data_ptr(), self.scales.data_ptr(), num_seqs, tokens, kv_heads, d, block_size, blocks, bt.shape[1], _lib.stream_ptr(dev)))

    def select(self, query: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor, query_start_loc: torch.Tensor, block_size: int,
               num_selected: int, num_sink_blocks: int = 1, num_recent_blocks: int = 2, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The blocks that each new token and kv head reads: [num_tokens, num_kv_heads, num_selected] int32 columns of the block tables,
        ascending, -1 behind the last where a token has fewer blocks.

        query            [num_tokens, num_query_heads, head_dim] float16 / bfloat16, the chunks of all sequences one after the other
        block_tables, context_lens, query_start_loc as in paged_chunk_attention
        num_selected     blocks a list, among them the first num_sink_blocks of the context and the last num_recent_blocks up to the
                         token's own (at least 1: its own block is always read); the others are those of largest (c_q . codes) scale with
                         c_q the sum of the group's queries in 8 bits, a float32 number (infinite past the largest); equal scores: the
                         lower column
        out              where the result goes (that shape, int32, contiguous)

        Products are of whole numbers: the result does not hang on the order of a sum."""
        result = _lib.calls().index_select(query, block_tables, context_lens, query_start_loc, self.codes, self.scales, out, self.num_blocks,
                                           self.num_kv_heads, self.head_dim, block_size, num_selected, num_sink_blocks, num_recent_blocks)
        if result is not None:
            return result if type(result) is not int else _lib.check(result)
        check_query(query)
        num_tokens, num_q_heads, d = query.shape
        if d != self.head_dim:
            raise ValueError(f"queries of {d} coordinates on an index of {self.head_dim}")
        if block_size < 1:
            raise ValueError(f"block_size {block_size}")
        if num_sink_blocks < 0 or num_recent_blocks < 1 or num_selected < num_sink_blocks + num_recent_blocks:
            raise ValueError(f"{num_selected} blocks cannot hold the first {num_sink_blocks} and the last {num_recent_blocks} (at least 1)")
        self._check()
        num_seqs, q, bt, lens, starts = check_chunk(query, self.num_kv_heads, block_tables, context_lens, query_start_loc)
        shape = (num_tokens, self.num_kv_heads, num_selected)
        if out is not None and (tuple(out.shape) != shape or out.dtype != torch.int32 or not out.is_contiguous()):
            raise ValueError(f"out must be contiguous int32 of shape {shape}, got {out.dtype} {tuple(out.shape)}")
        dev = _lib.require_gpu(query, block_tables, context_lens, query_start_loc, self.codes, self.scales, out)
        result = out if out is not None else torch.empty(shape, dtype=torch.int32, device=dev)
        L = _lib.lib()
        ws = torch.empty(L.akv_block_index_select_workspace_bytes(num_tokens, self.num_kv_heads, bt.shape[1]), dtype=torch.uint8, device=dev)
        with _lib.on_device(dev):
            _lib.check(L.akv_block_index_select(
                q.data_ptr(), _lib.dtype_code(q), q.stride(0), q.stride(1), self.codes.data_ptr(), self.scales.data_ptr(),
                bt.data_ptr(), _lib.itype_code(bt), bt.stride(0), lens.data_ptr(), _lib.itype_code(lens), starts.data_ptr(), _lib.itype_code(starts),
                result.data_ptr(), num_seqs, num_tokens, num_q_heads, self.num_kv_heads, d, block_size, self.num_blocks, bt.shape[1],
                num_selected, num_sink_blocks, num_recent_blocks, ws.data_ptr(), ws.numel(), _lib.stream_ptr(dev)))
        return result


def check_sequences(block_tables: torch.Tensor, context_lens: torch.Tensor, query_start_loc: Optional[torch.Tensor]):
    """Tables, lengths and starts (or None) of a batch in the form the kernels take, and how many sequences it has."""
    if block_tables.dim() != 2 or context_lens.dim() != 1 or (query_start_loc is not None and (query_start_loc.dim() != 1 or query_start_loc.numel() < 1)):
        raise ValueError("expected block_tables [num_seqs, blocks], context_lens [num_seqs] and query_start_loc [num_seqs + 1]")
    num_seqs = context_lens.numel() if query_start_loc is None else query_start_loc.numel() - 1
    _lib.check_batch(num_seqs, block_tables, context_lens)
    bt = block_tables if block_tables.stride(-1) == 1 or block_tables.shape[1] < 2 else block_tables.contiguous()
    return num_seqs, bt, context_lens.contiguous(), None if query_start_loc is None else query_start_loc.contiguous()


def paged_sparse_attention(query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, block_tables: torch.Tensor,
                           context_lens: torch.Tensor, query_start_loc: torch.Tensor, selected: torch.Tensor, scale: Optional[float] = None,
                           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of every sequence's newest tokens over the blocks that each token and kv head has selected.

    query, key_cache, value_cache, block_tables, context_lens, query_start_loc, scale, out as in paged_chunk_attention
    selected  [num_tokens, num_kv_heads, entries] int32: columns of the sequence's block table, as BlockIndex.select gives them.  A set:
              order and repetition do not matter; entries below 0, or past the token's own block, are skipped.  At most 4096 entries

    A token sees the keys of its selected blocks up to its own position; one without a key gets zeros.  head_dim is 64, 128 or 256.
    Past a context, and in blocks that are not selected, the caches may hold anything; a value that is not finite reaches only tokens that
    see it.  A block has at most 4096 tokens, less than 256 MB apart, and a table at most some 800000 columns.  Scores and sums are float32; a key's weight is rounded to the query's type before it meets its value
    (in float16 also by 2^-30 of the row's largest), and so is the result."""
    result = _lib.calls().sparse_attention(query, key_cache, value_cache, block_tables, context_lens, query_start_loc, selected, scale, out)
    if result is not None:
        return result if type(result) is not int else _lib.check(result)
    check_query(query)
    _check_rows("key_cache", key_cache, 4)
    _check_rows("value_cache", value_cache, 4)
    num_tokens, num_q_heads, d = query.shape
    blocks, block_size, kv_heads = key_cache.shape[:3]
    if value_cache.shape[1:] != key_cache.shape[1:] or key_cache.shape[3] != d:
        raise ValueError(f"caches of shape {tuple(key_cache.shape)} and {tuple(value_cache.shape)} do not fit queries of {d} coordinates")
    if key_cache.dtype != query.dtype or value_cache.dtype != query.dtype:
        raise ValueError(f"queries are {query.dtype}, caches {key_cache.dtype} and {value_cache.dtype}: they must agree")
    num_seqs, q, bt, lens, starts = check_chunk(query, kv_heads, block_tables, context_lens, query_start_loc)
    if selected.dim() != 3 or tuple(selected.shape[:2]) != (num_tokens, kv_heads) or selected.dtype != torch.int32:
        raise ValueError(f"selected must be int32 [{num_tokens}, {kv_heads}, entries], got {selected.dtype} {tuple(selected.shape)}")
    sel = selected if selected.stride(2) == 1 or selected.shape[2] < 2 else selected.contiguous()
    if out is not None:
        _check_out("out", out, query)
    dev = _lib.require_gpu(query, key_cache, value_cache, block_tables, context_lens, query_start_loc, selected, out)
    result = out if out is not None else torch.empty((num_tokens, num_q_heads, d), dtype=query.dtype, device=dev)
    L = _lib.lib()
    ws = torch.empty(L.akv_sparse_attn_workspace_bytes(num_tokens, num_seqs, num_q_heads, kv_heads, d, block_size, sel.shape[2]), dtype=torch.uint8, device=dev)
    with _lib.on_device(dev):
        _lib.check(L.akv_sparse_attn(
            q.data_ptr(), _lib.dtype_code(q), q.stride(0), q.stride(1),
            key_cache.data_ptr(), key_cache.stride(0), key_cache.stride(1), key_cache.stride(2),
            value_cache.data_ptr(), value_cache.stride(0), value_cache.stride(1), value_cache.stride(2),
            bt.data_ptr(), _lib.itype_code(bt), bt.stride(0), lens.data_ptr(), _lib.itype_code(lens), starts.data_ptr(), _lib.itype_code(starts),
            sel.data_ptr(), sel.stride(0), sel.stride(1), sel.shape[2], result.data_ptr(), result.stride(0), result.stride(1), int(out is None),
            num_seqs, num_tokens, num_q_heads, kv_heads, d, block_size, min(blocks, value_cache.shape[0]), bt.shape[1],
            1.0 / math.sqrt(d) if scale is None else scale, ws.data_ptr(), ws.numel(), _lib.stream_ptr(dev)))
    return result
