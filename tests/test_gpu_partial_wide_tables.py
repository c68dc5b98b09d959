"""Key weights over tables far wider than the contexts, where the scores of few rows find no room: right, with scratch of 258 MB at most.  Bounds as in
test_gpu_partial.py."""
import math

import pytest
import torch

import aitherkvcache_amd as akv
from tests.test_gpu_chunk import BF, FP, Batch, Packed, unpack
from tests.test_gpu_partial import vectors, weights_reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype,heads,kvh,lens,width", [
    # one token, a few and none; slabs of fifteen tokens of less than thirty sequences and of more, and none
    (BF, 32, 8, [(1, 700), (3, 300), (0, 50), (2, 2), (1, 1), (4, 900)] * 4, 1 << 17), (BF, 32, 4, [(1, 100), (17, 40), (0, 50), (1, 1), (0, 0), (1, 200), (2, 300)] * 7, 1 << 17), (FP, 64, 2, [(1, 700), (3, 300), (0, 50), (2, 2), (1, 1), (4, 900)], 1 << 20),
    (BF, 64, 1, [(1, 3000)], 1 << 20), (FP, 16, 16, [(1, 800), (9, 30), (2, 600), (5, 4)], 1 << 22)])
def test_tables_far_wider_than_contexts(dev, dtype, heads, kvh, lens, width, packed):
    d = 64
    b = Batch(lens, 16, dev, seed=33, pad_cols=0)
    b.kvh = kvh
    wide = torch.full((len(lens), width // 16), -5, dtype=torch.int32, device=dev)
    wide[:, :b.tables.shape[1]] = b.tables
    if packed:
        p = Packed(b, d, 4, heads, kvh, dtype, dev, 34)
        call = lambda **more: p.attn.key_weights(p.q, p.k, p.kn, wide, b.ctx, b.starts, **more)  # noqa: E731
        levels, pi = p.tq.centroids.cpu().double(), p.tq.rotation.cpu().double()
        want, _ = weights_reference(b, p.q, lambda i: (levels[unpack(b.rows(p.k, i), 4, d).cpu()].view(-1, kvh, d) @ pi) * b.rows(p.kn, i).cpu().double()[..., None], 1 / math.sqrt(d))
        turned = (p.q.cpu().double().abs() @ pi.abs().T).sum(-1).max().item()
        rel = 2 * turned * levels.abs().max().item() * p.kn[~p.kn.isnan()].max().item() / math.sqrt(d) * (2 * d * 2.0 ** -24 + 3 * 2.0 ** -22) + 2.0 ** -20
    else:
        gen = torch.Generator().manual_seed(3)
        q, k = vectors(gen, dtype, dev, b.tokens, heads, d), vectors(gen, dtype, dev, b.blocks, 16, kvh, d)
        call = lambda **more: akv.paged_key_weights(q, k, wide, b.ctx, b.starts, **more)  # noqa: E731
        want, most = weights_reference(b, q, lambda i: b.rows(k, i), 1 / math.sqrt(d))
        rel = 2 * most * d * 2.0 ** -24 + 2.0 ** -20
    acc = torch.full((len(lens), kvh, width), 0.5, device=dev)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    assert call(accumulated=acc) is acc
    assert torch.cuda.max_memory_allocated() - before <= 259 << 20
    for i, (n, c) in enumerate(lens):
        # (what is added to 0.5, in up to three pieces, is rounded by 2^-24 of the sum each time)
        off = (acc[i, :, :c].cpu().double() - 0.5 - want[i, :, :c]).abs()
        assert (off <= rel * want[i, :, :c] + 3 * 2.0 ** -24 * acc[i, :, :c].cpu()).all() and (acc[i, :, c:] == 0.5).all()
    del acc
    got = call()
    places = want.shape[2]
    off = (got[..., :places].cpu().double() - want).abs()
    assert (got[..., places:] == 0).all() and (off <= rel * want + 1e-30).all() and (off.square().sum() / want.square().sum()).sqrt() < 2e-6
