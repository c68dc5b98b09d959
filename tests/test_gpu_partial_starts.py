"""BlockIndex.update over a part of a batch: starts that lie far behind the rows of other sequences say how many new tokens a sequence has, and
nothing else.  Codes and scales as in test_gpu_partial.py: equal to the plain form's."""
import pytest
import torch

import aitherkvcache_amd as akv
from tests.test_gpu_chunk import BF, FP, Batch
from tests.test_gpu_chunk_use import binding
from tests.test_gpu_partial import index_of, vectors

pytestmark = pytest.mark.gpu

LENS = [(1000, 1000), (10, 40), (20, 20), (0, 30), (5, 7), (1, 64), (33, 50)]


@pytest.mark.parametrize("take", [True, False])
@pytest.mark.parametrize("dtype,index", [(BF, torch.int32), (FP, torch.int64)])
@pytest.mark.parametrize("first,shift", [(1, 0), (2, 0), (5, 0), (1, 100), (1, 1 << 29)])
def test_update_of_a_part_of_a_batch(dev, monkeypatch, first, shift, dtype, index, take):
    b = Batch(LENS, 16, dev, seed=21, index=index)
    cache = vectors(torch.Generator().manual_seed(first), dtype, dev, b.blocks, 16, 2, 64)
    # (the sequences behind `first` hold 64 tokens at most: four columns)
    tables, ctx, starts = b.tables[first:, :4], b.ctx[first:], b.starts[first:] + shift
    ix = akv.BlockIndex(b.blocks, 2, 64, dev)
    ix.codes.fill_(99)
    ix.scales.fill_(-1.0)
    with binding(monkeypatch, take) as c:
        ix.update(cache, tables, ctx, starts)
        assert c.taken == (1 if take else 0)
    want = index_of(cache, b, [(i, col) for i, (n, c) in enumerate(LENS) for col in range((c - n) // 16, -(-c // 16)) if n and i >= first])
    codes, scales = ix.codes.cpu(), ix.scales.cpu()
    for blk in range(b.blocks):
        if blk in want:
            assert torch.equal(codes[blk].float(), want[blk][0]) and torch.equal(scales[blk], want[blk][1]), blk
        else:
            assert (codes[blk] == 99).all() and (scales[blk] == -1).all(), blk


@pytest.mark.parametrize("take", [True, False])
@pytest.mark.parametrize("starts", [[100, 101], [60, 70], [20, 40]])
def test_update_of_one_sequence_of_a_batch(dev, monkeypatch, starts, take):
    n = starts[1] - starts[0]
    b = Batch([(n, 33)], 16, dev, seed=22, pad_cols=0)
    cache = vectors(torch.Generator().manual_seed(n), BF, dev, b.blocks, 16, 3, 128)
    ix = akv.BlockIndex(b.blocks, 3, 128, dev)
    with binding(monkeypatch, take):
        ix.update(cache, b.tables, b.ctx, torch.tensor(starts, dtype=torch.int32, device=dev))
    for blk, (codes, scales) in index_of(cache, b, [(0, col) for col in range((33 - n) // 16, 3)]).items():
        assert torch.equal(ix.codes[blk].cpu().float(), codes) and torch.equal(ix.scales[blk].cpu(), scales)
    for col in range((33 - n) // 16):
        assert (ix.scales[b.host[0, col]] == 0).all()
