"""A chunk of new tokens against an uncompressed paged cache: rotary positions with the append, and causal attention.

rope_append turns a chunk's queries and keys by their positions and writes keys and values to their slots;
paged_chunk_attention attends from every sequence's newest tokens over the cache.  The reference has neither: its prefill
scatters rows with torch indexing (aither_kvcache/vllm/backend.py:1247-1272) and calls its engine's dense kernel
(:1200-1236).  Attention of a chunk over the packed cache is TQPagedAttention.forward_chunk.
"""
import ctypes as C
import math
from typing import Optional, Sequence

import torch

from . import _lib

__all__ = ["rope_append", "paged_chunk_attention"]


def _check_rows(name: str, t: torch.Tensor, dims: int) -> None:
    if t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions, got shape {tuple(t.shape)}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")


def _check_out(name: str, out: torch.Tensor, like: torch.Tensor) -> None:
    _check_rows(name, out, like.dim())
    if out.shape != like.shape or out.dtype != like.dtype:
        raise ValueError(f"{name} must be {like.dtype} of shape {tuple(like.shape)}, got {out.dtype} {tuple(out.shape)}")


_INT_MAX = (1 << 31) - 1


def _longest(max_query_len: Optional[int]) -> int:
    return 0 if max_query_len is None else max(0, min(max_query_len, _INT_MAX))


def check_query(query: torch.Tensor) -> None:
    if query.dim() != 3:
        raise ValueError(f"query must be [tokens, heads, head_dim], got shape {tuple(query.shape)}")
    if query.dtype not in (torch.float16, torch.bfloat16):
        raise NotImplementedError(f"queries of a chunk are float16 or bfloat16, got {query.dtype}")


def check_chunk(query: torch.Tensor, num_kv_heads: int, block_tables: torch.Tensor, context_lens: torch.Tensor,
                query_start_loc: torch.Tensor):
    """What both attentions of a chunk ask of their batch; returns the tensors in the form the kernels take."""
    if num_kv_heads < 1 or query.shape[1] % num_kv_heads != 0:
        raise ValueError(f"{query.shape[1]} query heads on {num_kv_heads} kv heads")
    if block_tables.dim() != 2 or context_lens.dim() != 1 or query_start_loc.dim() != 1 or query_start_loc.numel() < 1:
        raise ValueError("expected block_tables [num_seqs, blocks], context_lens [num_seqs] and query_start_loc [num_seqs + 1]")
    num_seqs = query_start_loc.numel() - 1
    _lib.check_batch(num_seqs, block_tables, context_lens)
    q = query
    if query.stride(-1) != 1 or query.data_ptr() % 16 or query.stride(0) % 8 or query.stride(1) % 8:
        q = query.contiguous()
        if q.data_ptr() % 16:
            q = query.clone(memory_format=torch.contiguous_format)
    bt = block_tables if block_tables.stride(-1) == 1 or block_tables.shape[1] < 2 else block_tables.contiguous()
    return (num_seqs, q, bt, context_lens if context_lens.is_contiguous() else context_lens.contiguous(),
            query_start_loc if query_start_loc.is_contiguous() else query_start_loc.contiguous())


def paged_chunk_attention(query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, block_tables: torch.Tensor,
                          context_lens: torch.Tensor, query_start_loc: torch.Tensor, scale: Optional[float] = None, window: int = 0,
                          out: Optional[torch.Tensor] = None, max_query_len: Optional[int] = None) -> torch.Tensor:
    """Causal attention of every sequence's newest tokens over a paged cache that holds them already.

    query           [num_tokens, num_query_heads, head_dim] float16 / bfloat16, the chunks of all sequences one after the other
    key_cache, value_cache [num_blocks, block_size, num_kv_heads, head_dim] of the query's type (strides honoured)
    block_tables    [num_seqs, blocks] int32 / int64;  context_lens [num_seqs] tokens of a sequence, its chunk included
    query_start_loc [num_seqs + 1]: sequence i owns query rows query_start_loc[i] .. query_start_loc[i + 1] - 1
    scale           of the scores (1 / sqrt(head_dim));  window > 0: a token sees the newest `window` keys, its own among them
    out             where the result goes (same shape and type as query; rows before the first sequence or behind the last are left as
                    they were); without it a new tensor, zero in such rows
    max_query_len   the longest chunk, if known on the host: what is launched goes by it, the result but for its last rounding does not

    Token j of n stands at position context_len - n + j; one without a key gets zeros.  head_dim is 64, 128 or 256.
    Values that some token of a sequence's chunk sees must be finite; past a context, or before every token's window, the caches and
    tables may hold anything.  Scores and sums are float32; a key's weight is rounded to the query's type before it meets its value
    (in float16 also by 2^-30 of the row's largest), and so is the result."""
    result = _lib.calls().dense_chunk(query, key_cache, value_cache, block_tables, context_lens, query_start_loc, scale, window, out,
                                      max_query_len)
    if result is not None:
        return result if type(result) is not int else _lib.check(result)
    check_query(query)
    _check_rows("key_cache", key_cache, 4)
    _check_rows("value_cache", value_cache, 4)
    dev = _lib.require_gpu(query, key_cache, value_cache, block_tables, context_lens, query_start_loc, out)
    num_tokens, num_q_heads, d = query.shape
    blocks, block_size, kv_heads = key_cache.shape[:3]
    if value_cache.shape[1:] != key_cache.shape[1:] or key_cache.shape[3] != d:
        raise ValueError(f"caches of shape {tuple(key_cache.shape)} and {tuple(value_cache.shape)} do not fit queries of {d} coordinates")
    if key_cache.dtype != query.dtype or value_cache.dtype != query.dtype:
        raise ValueError(f"queries are {query.dtype}, caches {key_cache.dtype} and {value_cache.dtype}: they must agree")
    num_seqs, q, bt, lens, starts = check_chunk(query, kv_heads, block_tables, context_lens, query_start_loc)
    if out is not None:
        _check_out("out", out, query)
    result = out if out is not None else torch.empty((num_tokens, num_q_heads, d), dtype=query.dtype, device=dev)
    L = _lib.lib()
    ws = torch.empty(L.akv_dense_chunk_attn_workspace_bytes(d), dtype=torch.uint8, device=dev)
    with _lib.on_device(dev):
        _lib.check(L.akv_dense_chunk_attn(
            q.data_ptr(), _lib.dtype_code(q), q.stride(0), q.stride(1),
            key_cache.data_ptr(), key_cache.stride(0), key_cache.stride(1), key_cache.stride(2),
            value_cache.data_ptr(), value_cache.stride(0), value_cache.stride(1), value_cache.stride(2),
            bt.data_ptr(), _lib.itype_code(bt), bt.stride(0), lens.data_ptr(), _lib.itype_code(lens), starts.data_ptr(), _lib.itype_code(starts),
            result.data_ptr(), result.stride(0), result.stride(1), int(out is None),
            num_seqs, num_tokens, num_q_heads, kv_heads, d, block_size, min(blocks, value_cache.shape[0]), bt.shape[1], min(window, _INT_MAX),
            _longest(max_query_len), 1.0 / math.sqrt(d) if scale is None else scale, ws.data_ptr(), ws.numel(), _lib.stream_ptr(dev)))
    return result


def rope_append(query: Optional[torch.Tensor], key: torch.Tensor, value: torch.Tensor, positions: Optional[torch.Tensor],
                cos_sin: Optional[torch.Tensor], slot_mapping: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                sections: Optional[Sequence[int]] = None, interleaved: bool = False,
                query_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Rotate a chunk's queries and keys by their positions and append keys and values to a paged cache, in one launch.

    query        [num_tokens, num_query_heads, head_dim] or None;  key, value [num_tokens, num_kv_heads, head_dim], one type
    positions    [num_tokens] int32 / int64, or [axes, num_tokens] with `sections`, the pairs that each of up to four axes turns
    cos_sin      [positions, rotary_dim] float32: cosines of the rotary_dim / 2 pairs, then their sines.  None: nothing turns
    interleaved  pairs are neighbours (2p, 2p + 1) instead of (p, p + rotary_dim / 2); coordinates past rotary_dim stay
    slot_mapping [num_tokens]: block * block_size + place; negative slots and slots beyond the cache are skipped, the
                 others must differ
    key_cache, value_cache [num_blocks, block_size, num_kv_heads, head_dim] float16 / bfloat16 / float32, one type
    query_out    where the queries go (may be `query`); without it a new tensor

    Returns the rotated queries (None without queries).  Arithmetic in float32, one rounding to the type stored.  Positions
    outside the table are clamped into it.  head_dim and rotary_dim are multiples of 16."""
    result = _lib.calls().rope_append(query, key, value, positions, cos_sin, slot_mapping, key_cache, value_cache, sections, interleaved,
                                      query_out)
    if result is not None:
        return result if type(result) is not int else _lib.check(result)
    for name, t, dims in (("key", key, 3), ("value", value, 3), ("key_cache", key_cache, 4), ("value_cache", value_cache, 4)):
        if t.dim() != dims:
            raise ValueError(f"{name} must have {dims} dimensions, got shape {tuple(t.shape)}")
    _check_rows("key_cache", key_cache, 4)
    _check_rows("value_cache", value_cache, 4)
    num_tokens, kv_heads, d = key.shape
    if value.shape != key.shape or (query is not None and (query.dim() != 3 or query.shape[0] != num_tokens or query.shape[2] != d)):
        raise ValueError(f"query, key and value do not fit each other: {None if query is None else tuple(query.shape)}, {tuple(key.shape)}, {tuple(value.shape)}")
    if value.dtype != key.dtype or (query is not None and query.dtype != key.dtype) or value_cache.dtype != key_cache.dtype:
        raise ValueError("query, key and value must share a type, and so must the caches")
    if key_cache.shape[2:] != (kv_heads, d) or value_cache.shape[1:] != key_cache.shape[1:]:
        raise ValueError(f"caches of shape {tuple(key_cache.shape)} and {tuple(value_cache.shape)} do not fit {kv_heads} heads of {d}")
    if cos_sin is not None and positions is None:
        raise ValueError("a table without positions")
    dev = _lib.require_gpu(query, key, value, positions if cos_sin is not None else None, cos_sin, slot_mapping, key_cache, value_cache, query_out)
    _lib.check_slots(num_tokens, slot_mapping)
    if slot_mapping.dim() != 1:
        raise ValueError("slot_mapping must have one dimension")
    rotary, axes, counts = 0, 1, None
    if cos_sin is not None:
        if cos_sin.dim() != 2 or cos_sin.dtype != torch.float32 or not cos_sin.is_contiguous() or cos_sin.shape[0] == 0:
            raise ValueError("cos_sin must be a contiguous float32 table [positions, rotary_dim]")
        rotary = cos_sin.shape[1]
        if sections is not None:
            axes = len(sections)
            if not 1 <= axes <= 4:
                raise ValueError(f"one to four axes, got {axes} sections")
            counts = (C.c_int * axes)(*sections)
            if positions.dim() != 2 or positions.shape[0] != axes:
                raise ValueError(f"{axes} sections, but positions of shape {tuple(positions.shape)}")
            if min(sections) < 0 or sum(sections) != rotary // 2:
                raise ValueError(f"sections {tuple(sections)} do not make up {rotary // 2} pairs")
            positions = positions if positions.stride(1) == 1 else positions.contiguous()
        elif positions.dim() != 1:
            raise ValueError(f"positions of shape {tuple(positions.shape)} need sections")
        if positions.shape[-1] < num_tokens:
            raise ValueError(f"{num_tokens} tokens, but positions {tuple(positions.shape)}")
        positions = positions if positions.stride(-1) == 1 else positions.contiguous()
    key, value = (t if t.stride(2) == 1 else t.contiguous() for t in (key, value))
    slots = slot_mapping if slot_mapping.is_contiguous() else slot_mapping.contiguous()
    result = None
    if query is not None:
        q = query if query.stride(2) == 1 else query.contiguous()
        if query_out is not None:
            _check_out("query_out", query_out, query)
        result = query_out if query_out is not None else torch.empty(query.shape, dtype=query.dtype, device=dev)
    with _lib.on_device(dev):
        _lib.check(_lib.lib().akv_rope_append(
            None if query is None else q.data_ptr(), 0 if query is None else q.stride(0), 0 if query is None else q.stride(1),
            None if query is None else result.data_ptr(), 0 if query is None else result.stride(0), 0 if query is None else result.stride(1),
            key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(), value.stride(0), value.stride(1), _lib.dtype_code(key),
            positions.data_ptr() if rotary else None, _lib.itype_code(positions) if rotary else 0, positions.stride(0) if axes > 1 else 0,
            cos_sin.data_ptr() if rotary else None, cos_sin.shape[0] if rotary else 0, rotary, counts, axes, int(interleaved),
            slots.data_ptr(), _lib.itype_code(slots),
            key_cache.data_ptr(), key_cache.stride(0), key_cache.stride(1), key_cache.stride(2),
            value_cache.data_ptr(), value_cache.stride(0), value_cache.stride(1), value_cache.stride(2), _lib.dtype_code(key_cache),
            num_tokens, 0 if query is None else query.shape[1], kv_heads, d, key_cache.shape[1], min(key_cache.shape[0], value_cache.shape[0]),
            _lib.stream_ptr(dev)))
    return result
