"""BlockIndex.select where scores pass the largest float32 number: they are infinite, and ordered and listed like any other."""
import numpy as np
import pytest
import torch

import aitherkvcache_amd as akv
from tests.test_gpu_chunk import BF, Batch
from tests.test_gpu_partial import in_8_bits, tokens_of

pytestmark = pytest.mark.gpu


def selection(b, index, query, kvh, k, sinks, recent):
    """Plain selection; the first and last blocks go before any score."""
    codes, scales = index.codes.cpu().double(), index.scales.cpu()
    out = torch.full((len(query), kvh, k), -1, dtype=torch.int32)
    cq = in_8_bits(query.cpu().double().view(len(query), kvh, -1, query.shape[2]).sum(2).float())[0].double()
    for i, row, pos in tokens_of(b):
        n = pos // b.block + 1
        blocks = torch.from_numpy(b.host[i, :n])
        col = np.arange(n)
        forced = (col < sinks) | (col >= n - recent)
        for h in range(kvh):
            score = ((codes[blocks, h] @ cq[row, h]).float() * scales[blocks, h]).numpy()
            best = np.sort(np.lexsort((col, -score, ~forced))[:k])
            out[row, h, :len(best)] = torch.from_numpy(best.astype(np.int32))
    return out


@pytest.mark.parametrize("kind", ["below", "both", "most below", "above"])
@pytest.mark.parametrize("context,pad", [(600, 0), (1500, 0), (3000, 2), (7000, 4000), (9000, 20000)])
def test_infinite_scores(dev, context, pad, kind):
    gen = torch.Generator().manual_seed(context)
    b = Batch([(20, context), (3, context // 2)], 1, dev, seed=27, pad_cols=pad)
    index = akv.BlockIndex(b.blocks, 2, 64, dev)
    codes = torch.zeros(b.blocks, 2, 64, dtype=torch.int8)
    codes[:, :, 0] = -120 if kind != "above" else 120
    if kind == "both":
        codes[torch.rand(b.blocks, generator=gen) < 0.3, :, 0] = 120
    # (120 x 127 x 1e36 is past 2^128; 1e30 is not)
    scales = torch.full((b.blocks, 2), 1e36)
    if kind != "below":
        scales[torch.rand(b.blocks, generator=gen) < (0.02 if kind == "most below" else 0.4)] = 1e30
    index.codes.copy_(codes)
    index.scales.copy_(scales)
    query = torch.zeros(b.tokens, 4, 64, dtype=BF, device=dev)
    query[:, :, 0] = 1.0
    for k in (5, 70, 400):
        into = torch.full((b.tokens, 2, k), -77, dtype=torch.int32, device=dev)
        index.select(query, b.tables, b.ctx, b.starts, 1, k, num_sink_blocks=2, num_recent_blocks=2, out=into)
        assert torch.equal(into.cpu(), selection(b, index, query, 2, k, 2, 2)), k


def test_means_next_to_the_largest_number(dev):
    """Keys that bfloat16 holds, as update takes them."""
    gen = torch.Generator().manual_seed(1)
    b = Batch([(9, 900)], 4, dev, seed=28)
    cache = torch.randn(b.blocks, 4, 1, 64, generator=gen).to(BF).to(dev)
    cache[torch.rand(b.blocks, generator=gen).to(dev) < 0.5] *= 1e37
    index = akv.BlockIndex(b.blocks, 1, 64, dev)
    index.update(cache, b.tables, b.ctx, b.starts)
    index.update(cache, b.tables, b.ctx)
    query = torch.randn(9, 4, 64, generator=gen).to(BF).to(dev)
    dots = index.codes.cpu().double()[:, 0] @ in_8_bits(query.cpu().double().sum(1).float())[0].double().T
    scores = dots.float() * index.scales.cpu()
    assert (scores == np.inf).any() and (scores == -np.inf).any() and torch.isfinite(scores).any()
    for k in (10, 150, 200):
        got = index.select(query, b.tables, b.ctx, b.starts, 4, k)
        assert torch.equal(got.cpu(), selection(b, index, query, 1, k, 1, 2))
