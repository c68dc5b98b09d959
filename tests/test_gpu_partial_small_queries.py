"""Key weights of packed rows for queries that are zero, or next to it: such a query likes all keys alike.  Bounds as in test_gpu_partial.py."""
import math

import numpy as np
import pytest
import torch

import aitherkvcache_amd as akv
from tests.test_gpu_chunk import BF, FP, Batch, Packed, unpack
from tests.test_gpu_partial import weights_reference

pytestmark = pytest.mark.gpu

FEW = [(1, 700), (2, 300), (3, 3), (1, 1), (4, 40)]
MANY = [(40, 513), (17, 17), (20, 300), (1, 64)]


@pytest.mark.parametrize("bits", [4, 3, 2])
@pytest.mark.parametrize("lens", [FEW, MANY], ids=["few rows", "many rows"])
@pytest.mark.parametrize("d,heads,kvh,dtype", [(128, 8, 2, BF), (64, 8, 2, FP), (256, 4, 2, BF)])
def test_zero_and_tiny_queries(dev, d, heads, kvh, dtype, lens, bits):
    b = Batch(lens, 16, dev, seed=23)
    b.kvh = kvh
    p = Packed(b, d, bits, heads, kvh, dtype, dev, 24)
    q = p.q
    # the smallest numbers of a type, below and at the edge of its normal ones, and zeros of both signs
    tiny = [1e-36, 2.0 ** -126, 2.0 ** -133, 2.0 ** -113, 2.0 ** -112, 2.0 ** -100] if dtype == BF else [2.0 ** -24, 2.0 ** -14, 2.0 ** -20]
    for row in range(b.tokens):
        if row % 3 == 0:
            q[row] = 0.0
        elif row % 3 == 1:
            q[row] *= tiny[row // 3 % len(tiny)]
        q[row, row % heads] = -0.0
    got = p.attn.key_weights(q, p.k, p.kn, b.tables, b.ctx, b.starts)
    levels, pi = p.tq.centroids.cpu().double(), p.tq.rotation.cpu().double()

    def keys(i):
        return (levels[unpack(b.rows(p.k, i), bits, d).cpu()].view(-1, kvh, d) @ pi) * b.rows(p.kn, i).cpu().double()[..., None]

    want, _ = weights_reference(b, q, keys, 1 / math.sqrt(d))
    turned = (q.cpu().double().abs() @ pi.abs().T).sum(-1).max().item()
    most = turned * levels.abs().max().item() * p.kn[~p.kn.isnan()].max().item() / math.sqrt(d)
    rel = 2 * most * (2 * d * 2.0 ** -24 + 3 * 2.0 ** -22) + 2.0 ** -20
    off = (got.cpu().double() - want).abs()
    assert torch.isfinite(got).all() and (off <= rel * want + 1e-30).all()
    acc = torch.full_like(got, 0.25)
    p.attn.key_weights(q, p.k, p.kn, b.tables, b.ctx, b.starts, accumulated=acc)
    for i, (_, c) in enumerate(lens):
        # (rows come in two blocks at most: three additions, each rounded by 2^-24 of what is there)
        assert ((acc[i, :, :c] - 0.25 - got[i, :, :c]).abs() <= 2.0 ** -21 * acc[i, :, :c]).all() and (acc[i, :, c:] == 0.25).all()


@pytest.mark.parametrize("tokens", [1, 200])
def test_queries_of_nothing_but_zeros(dev, tokens):
    """Every key that a row sees has the same weight."""
    b = Batch([(tokens, 230)], 16, dev, seed=25)
    p = Packed(b, 128, 4, 4, 1, FP, dev, 26)
    got = p.attn.key_weights(torch.zeros_like(p.q), p.k, p.kn, b.tables, b.ctx, b.starts)[0, 0].cpu().double().numpy()
    seen = np.arange(230 - tokens, 230) + 1
    want = np.array([4 * (1.0 / seen[seen > key]).sum() for key in range(230)])
    # (a weight is an inverse, rounded by 2^-24, and a sum of up to 800 of them by 2^-24 each in the worst case)
    assert np.abs(got[:230] / want - 1).max() <= (4 * tokens + 2) * 2.0 ** -24 and (got[230:] == 0).all()
