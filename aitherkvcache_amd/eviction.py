"""Tokens of a paged cache given up by the attention weight they get.

paged_key_weights (over packed codes TQPagedAttention.key_weights) adds up the attention weight that every cached key gets from new
tokens; evict_tokens keeps the heaviest tokens of each sequence and kv head and moves their rows to the front.  The reference has neither.
"""
import math
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from .chunk_attention import _check_rows, check_chunk, check_query

__all__ = ["paged_key_weights", "evict_tokens"]


def weights_for(accumulated: Optional[torch.Tensor], num_seqs: int, kv_heads: int, length: int, device) -> torch.Tensor:
    """Where a call's weights go: `accumulated`, or a new tensor."""
    if accumulated is None:
        return torch.empty(num_seqs, kv_heads, length, dtype=torch.float32, device=device)
    check_weights("accumulated", accumulated, num_seqs, kv_heads, length)
    # (weights are added row by row, by workgroups of their own)
    end = accumulated.shape[2]
    for stride, count in sorted(zip(accumulated.stride()[:2], accumulated.shape[:2])):
        if count > 1 and stride < end:
            raise ValueError("accumulated has rows that share memory")
        end += stride * (count - 1)
    return accumulated


def check_weights(name: str, t: torch.Tensor, num_seqs: int, kv_heads: Optional[int], length: int) -> None:
    if t.dim() != 3 or t.dtype != torch.float32 or t.shape[0] < num_seqs or (kv_heads is not None and t.shape[1] != kv_heads) or t.shape[2] < length:
        raise ValueError(f"{name} must be float32 [{num_seqs}, {'kv heads' if kv_heads is None else kv_heads}, {length} or more], got {t.dtype} {tuple(t.shape)}")
    if t.stride(2) != 1 and t.shape[2] > 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")
    if t.stride(0) == 0 and t.shape[0] > 1 or t.stride(1) == 0 and t.shape[1] > 1:
        raise ValueError(f"{name} has rows that share memory")


def paged_key_weights(query: torch.Tensor, key_cache: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor,
                      query_start_loc: torch.Tensor, accumulated: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """The softmax weight that every cached key gets from its sequence's newest tokens (causal, as paged_chunk_attention weighs them),
    summed over these tokens and over the query heads of a kv head: [num_seqs, num_kv_heads, length] float32, a key at its position.

    query, key_cache, block_tables, context_lens, query_start_loc, scale as in paged_chunk_attention
    accumulated  [num_seqs, num_kv_heads, length] float32, rows apart in memory: the weights are added to what is there, and it is returned; its
                 length is at least that of the tables, and positions past a context are left as they are.  Without it a new tensor as long as the tables,
                 zero past a context

    To weigh a prompt by its last tokens pass those tokens only.  head_dim is 64, 128 or 256, sequences and kv heads at most 65535.  Keys of a
    context and queries must be finite; past it the cache may hold anything.  Scores, weights and sums are float32."""
    result = _lib.calls().key_weights(query, key_cache, block_tables, context_lens, query_start_loc, accumulated, scale)
    if result is not None:
        return result if type(result) is not int else _lib.check(result)
    check_query(query)
    _check_rows("key_cache", key_cache, 4)
    num_tokens, num_q_heads, d = query.shape
    blocks, block_size, kv_heads = key_cache.shape[:3]
    if key_cache.shape[3] != d or key_cache.dtype != query.dtype:
        raise ValueError(f"a cache of {key_cache.dtype} {tuple(key_cache.shape)} does not fit queries of {query.dtype} with {d} coordinates")
    num_seqs, q, bt, lens, starts = check_chunk(query, kv_heads, block_tables, context_lens, query_start_loc)
    dev = _lib.require_gpu(query, key_cache, block_tables, context_lens, query_start_loc, accumulated)
    w = weights_for(accumulated, num_seqs, kv_heads, bt.shape[1] * block_size, dev)
    L = _lib.lib()
    ws = torch.empty(L.akv_key_weights_workspace_bytes(num_tokens, num_seqs, num_q_heads, kv_heads, d, w.shape[2]), dtype=torch.uint8, device=dev)
    with _lib.on_device(dev):
        _lib.check(L.akv_key_weights(
            q.data_ptr(), _lib.dtype_code(q), q.stride(0), q.stride(1), key_cache.data_ptr(), key_cache.stride(0), key_cache.stride(1), key_cache.stride(2),
            bt.data_ptr(), _lib.itype_code(bt), bt.stride(0), lens.data_ptr(), _lib.itype_code(lens), starts.data_ptr(), _lib.itype_code(starts),
            w.data_ptr(), w.stride(0), w.stride(1), w.shape[2], int(accumulated is not None), num_seqs, num_tokens, num_q_heads, kv_heads, d, block_size,
            blocks, bt.shape[1], 1.0 / math.sqrt(d) if scale is None else scale, ws.data_ptr(), ws.numel(), _lib.stream_ptr(dev)))
    return w


def _bytes_of(name: str, t: torch.Tensor, block_size: int, kv_heads: int):
    """A cache [blocks, positions, heads, ...] as strides and rows of bytes."""
    if t.dim() < 3:
        raise ValueError(f"{name} must be [blocks, block_size, heads, ...], got shape {tuple(t.shape)}")
    _lib.check_caches(block_size, kv_heads, t)
    row = t[0, 0, 0] if t.shape[0] else t.new_empty(t.shape[3:])
    if row.dim() and not row.is_contiguous():
        raise ValueError(f"the rows of {name} must be contiguous")
    size = t.element_size()
    return [s * size for s in t.stride()[:3]], row.numel() * size


def evict_tokens(weights: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor, caches: Sequence[torch.Tensor], keep: int,
                 num_sink: int = 4, num_recent: int = 32, out_tables: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Keep the heaviest `keep` tokens of every sequence, for each kv head its own, and move their rows to the front, in order.

    weights       [num_seqs, num_kv_heads, length] float32, as paged_key_weights adds them up (length at least that of the tables)
    block_tables  [num_seqs, blocks] int32 / int64;  context_lens [num_seqs]
    caches        up to 8 tensors [num_blocks, block_size, num_kv_heads, ...] of any type: keys, values, packed rows, norms; strides are
                  honoured, rows must be contiguous and share no memory with others.  Position kept[j] of a sequence and head goes to position j of each
    keep          tokens that stay (of a shorter sequence all), among them the first num_sink and the last num_recent; equal weights: the
                  earlier token; a NaN counts as -infinity
    out_tables    [num_seqs, blocks of `keep` tokens or more]: blocks that the rows move to and that no sequence of the call reads, for
                  sequences that share blocks.  None: in place, and no block may belong to two sequences or stand twice in a table

    Returns (kept [num_seqs, num_kv_heads, keep] int32: positions in ascending order, -1 behind the last; the sequences' lengths now, in
    the type of context_lens; weights of the tokens that stayed, at their new positions, zeros behind, in a new tensor).  Rows behind the
    tokens that stayed are left as they were.  Positions that are part of a key (rotary ones) stay in it."""
    result = _lib.calls().evict(weights, block_tables, context_lens, caches, keep, num_sink, num_recent, out_tables)
    if result is not None:
        return result if type(result) is not int else _lib.check(result)
    check_weights("weights", weights, 0, None, 0)
    if block_tables.dim() != 2 or context_lens.dim() != 1:
        raise ValueError("expected block_tables [num_seqs, blocks] and context_lens [num_seqs]")
    num_seqs, kv_heads = context_lens.numel(), weights.shape[1]
    _lib.check_batch(num_seqs, block_tables, context_lens)
    if keep < 1 or keep > 1 << 30 or num_sink < 0 or num_recent < 0 or keep < num_sink + num_recent:
        raise ValueError(f"keep {keep} tokens, among them the first {num_sink} and the last {num_recent}")
    if not 1 <= len(caches) <= _lib.EVICT_CACHES:
        raise ValueError(f"one to {_lib.EVICT_CACHES} caches, got {len(caches)}")
    if kv_heads < 1 or caches[0].dim() < 3:
        raise ValueError(f"weights of shape {tuple(weights.shape)} and a cache of shape {tuple(caches[0].shape)}")
    block_size = caches[0].shape[1]
    blocks = min(t.shape[0] for t in caches)
    rows = [_bytes_of(f"caches[{i}]", t, block_size, kv_heads) for i, t in enumerate(caches)]
    if any(t.shape[1] != block_size or t.shape[2] != kv_heads for t in caches):
        raise ValueError(f"caches of shape {[tuple(t.shape) for t in caches]} do not fit each other and {kv_heads} kv heads")
    check_weights("weights", weights, num_seqs, kv_heads, block_tables.shape[1] * block_size)
    if out_tables is not None and (out_tables.dim() != 2 or out_tables.shape[0] < num_seqs or out_tables.shape[1] * block_size < min(keep, block_tables.shape[1] * block_size)):
        raise ValueError(f"out_tables of shape {tuple(out_tables.shape)} do not hold {num_seqs} sequences of {keep} tokens")
    dev = _lib.require_gpu(weights, block_tables, context_lens, out_tables, *caches)
    bt = block_tables if block_tables.stride(-1) == 1 or block_tables.shape[1] < 2 else block_tables.contiguous()
    ot = out_tables if out_tables is None or out_tables.stride(-1) == 1 or out_tables.shape[1] < 2 else out_tables.contiguous()
    lens = context_lens.contiguous()
    itype, bt_itype, ot_itype = _lib.itype_code(lens), _lib.itype_code(bt), 0 if ot is None else _lib.itype_code(ot)
    kept = torch.empty(num_seqs, kv_heads, keep, dtype=torch.int32, device=dev)
    left = torch.empty(num_seqs, kv_heads, weights.shape[2], dtype=torch.float32, device=dev)
    now = torch.empty(num_seqs, dtype=lens.dtype, device=dev)
    # (no further than the tables: what lies behind is not theirs)
    length = min(weights.shape[2], bt.shape[1] * block_size) if blocks else 0
    if length < left.shape[2]:
        left.zero_()
    L = _lib.lib()
    moved = [_lib.EvictCache(t.data_ptr(), *strides, size) for t, (strides, size) in zip(caches, rows) if size]      # (a row of nothing stays where it is)
    chosen = (weights.data_ptr(), weights.stride(0), weights.stride(1), length, lens.data_ptr(), itype, num_seqs, kv_heads, keep, num_sink, num_recent,
              kept.data_ptr(), kept.stride(0), kept.stride(1), left.data_ptr(), left.stride(0), left.stride(1), now.data_ptr())
    with _lib.on_device(dev):
        stream = _lib.stream_ptr(dev)
        if not blocks or not moved:
            _lib.check(L.akv_evict_select(*chosen, stream))
        else:
            held = (_lib.EvictCache * len(moved))(*moved)
            _lib.check(L.akv_evict(*chosen, bt.data_ptr(), bt_itype, bt.stride(0), bt.shape[1], None if ot is None else ot.data_ptr(), ot_itype,
                                   0 if ot is None else ot.stride(0), 0 if ot is None else ot.shape[1], held, len(moved), block_size, blocks, stream))
    return kept, now, left
