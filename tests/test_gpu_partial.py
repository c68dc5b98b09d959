"""A part of a long context: BlockIndex, paged_sparse_attention, paged_key_weights, TQPagedAttention.key_weights and evict_tokens against
plain implementations in 64 bits.

Tolerances.  Means are sums of 16-bit numbers in 64 bits and one rounding to float32, codes and scales functions of these: equal to the plain
form's.  Selections are whole numbers: equal.  Sparse attention: as for a chunk's attention over plain rows (test_gpu_chunk.py): u is half a
step of the 16-bit type (2^-8 bfloat16, 2^-11 float16), every weight is rounded once (u of itself; float16 weights by up to 2^-25 of the
largest besides, and the sum of weights is at least the largest) and so is the output, so a coordinate is off by at most
(2 u + 2^-14) A + 2^-25 B with A the same attention over |v| and B the sum of |v| over the keys.
Weights: a score is a sum of d products of size |q| |k| scale, each addition rounded by 2^-24: off by at most d 2^-24 E with
E = scale sum_i |q_i k_i| (packed: terms of 2^-22 each for levels and queries besides, and the rotation of a query by sums of d products,
d 2^-24 sum_j |Pi_ij q_j|, so E there is scale |k| sum_i |c_i| sum_j |Pi_ij q_j| and the factor 2 d 2^-24 + 3 2^-22); a weight is off by the
factor exp(2 max E d 2^-24) and some roundings of its own, 2^-20 for the exponents (of scores below 2^4 in size the differences are rounded by
2^-20 at most) and sums."""
import math

import numpy as np
import pytest
import torch

import aitherkvcache_amd as akv
from tests.test_gpu_chunk import BF, FP, HALF, Batch

pytestmark = pytest.mark.gpu


def vectors(gen, dtype, dev, *shape):
    x = torch.randn(shape, generator=gen)
    return (x * torch.exp(0.3 * torch.randn(shape[:-1], generator=gen))[..., None]).to(dtype).to(dev)


def tokens_of(b):
    """(sequence, row, position) of every query row."""
    at = 0
    for i, (n, c) in enumerate(b.lens):
        for j in range(n):
            yield i, at + j, c - n + j
        at += n


# ---- the index ------------------------------------------------------------------------------------------------
def in_8_bits(x):
    """The codes of vectors (as numbers) and their scales, from float32 means."""
    top = x.abs().amax(-1, keepdim=True)
    per = torch.reciprocal(top) * 127
    fine = torch.isfinite(top) & torch.isfinite(per)
    return torch.where(fine, torch.round(x * per), 0.0), torch.where(fine, top * torch.tensor(1 / 127), 0.0)[..., 0]


def index_of(cache, b, columns):
    """Codes and scales of the given (sequence, column) pairs' blocks."""
    out = {}
    for i, col in columns:
        c = min(b.block, b.lens[i][1] - col * b.block)
        blk = b.host[i, col]
        keys = cache[blk, :c].double().cpu()
        out[blk] = in_8_bits((keys.sum(0) / c).float())
    return out


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d,kvh,block", [(64, 1, 16), (128, 8, 16), (256, 5, 32), (128, 2, 7), (64, 4, 1), (128, 3, 100)])
def test_update(dev, d, kvh, block, dtype):
    gen = torch.Generator().manual_seed(d + kvh + block)
    lens = [(1, 1), (5, 40), (0, 33), (130, 130), (16, 64), (1, 17), (0, 0), (3, 200), (33, 90)]
    b = Batch(lens, block, dev, seed=4, index=torch.int64 if kvh == 8 else torch.int32)
    cache = vectors(gen, dtype, dev, b.blocks, block, kvh, d)
    b.unused(math.nan, cache)
    index = akv.BlockIndex(b.blocks, kvh, d, dev)
    index.codes.fill_(99)
    index.scales.fill_(-1.0)
    index.update(cache, b.tables, b.ctx, b.starts)
    touched = [(i, col) for i, (n, c) in enumerate(lens) for col in range((c - n) // block, -(-c // block)) if n]
    want = index_of(cache, b, touched)
    codes, scales = index.codes.cpu(), index.scales.cpu()
    for blk in range(b.blocks):
        if blk in want:
            assert torch.equal(codes[blk].float(), want[blk][0]) and torch.equal(scales[blk], want[blk][1]), blk
        else:
            assert (codes[blk] == 99).all() and (scales[blk] == -1).all(), blk
    # all blocks of every sequence
    index.update(cache, b.tables, b.ctx)
    want = index_of(cache, b, [(i, col) for i, (_, c) in enumerate(lens) for col in range(-(-c // block))])
    for blk, (c, s) in want.items():
        assert torch.equal(index.codes[blk].cpu().float(), c) and torch.equal(index.scales[blk].cpu(), s)
    assert torch.equal(index.dequantized(), index.codes.float() * index.scales[..., None])


def test_update_of_odd_keys(dev):
    """Zeros, infinities, values near a type's ends, and strides."""
    b = Batch([(64, 64)], 16, dev, seed=1, spare=0)
    wide = torch.randn(b.blocks, 4, 16, 128, device=dev).to(BF)
    cache = wide.transpose(1, 2)[:, :, 1:3]
    blk = b.host[0]
    cache[blk[0]] = 0
    cache[blk[1], 3, 0, 5] = math.inf
    cache[blk[2]] = 1e-38
    index = akv.BlockIndex(b.blocks, 2, 128, dev)
    index.update(cache, b.tables, b.ctx, b.starts)
    want = index_of(cache, b, [(0, i) for i in range(4)])
    for n, (c, s) in want.items():
        assert torch.equal(index.codes[n].cpu().float(), c) and torch.equal(index.scales[n].cpu(), s)
    assert (index.codes[blk[0]] == 0).all() and (index.scales[blk[0]] == 0).all() and index.scales[blk[1], 0] == 0 and index.scales[blk[1], 1] > 0


def selection(b, index, query, kvh, k, sinks, recent):
    """Plain selection: every token and head."""
    codes, scales = index.codes.cpu().double(), index.scales.cpu()
    out = torch.full((len(query), kvh, k), -1, dtype=torch.int32)
    q = query.cpu().double().view(len(query), kvh, -1, query.shape[2]).sum(2).float()
    cq = in_8_bits(q)[0].double()
    for i, row, pos in tokens_of(b):
        if pos < 0:
            continue
        n = pos // b.block + 1
        blocks = torch.from_numpy(b.host[i, :n])
        for h in range(kvh):
            score = ((codes[blocks, h] @ cq[row, h]).float() * scales[blocks, h]).numpy()
            col = np.arange(n)
            score = np.where((col < sinks) | (col >= n - recent), np.inf, score)
            best = np.sort(np.lexsort((col, -score))[:k])
            out[row, h, :len(best)] = torch.from_numpy(best.astype(np.int32))
    return out


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d,heads,kvh,block,k,sinks,recent", [
    (128, 32, 8, 16, 8, 1, 2), (64, 28, 4, 32, 3, 0, 1), (256, 16, 16, 16, 12, 2, 3), (128, 8, 1, 7, 20, 3, 1), (64, 40, 8, 1, 30, 0, 30), (128, 4, 2, 16, 1, 0, 1)])
def test_select(dev, d, heads, kvh, block, k, sinks, recent, dtype):
    gen = torch.Generator().manual_seed(d + heads + k)
    lens = [(1, 700), (20, 300), (0, 50), (3, 3), (17, 17), (1, 1), (40, 513), (5, 2), (1, 1200)]
    b = Batch(lens, block, dev, seed=5, index=torch.int64 if kvh == 1 else torch.int32)
    index = akv.BlockIndex(b.blocks, kvh, d, dev)
    # few different means, so that scores tie
    index.codes.copy_(torch.randint(-127, 128, (9, kvh, d), generator=gen)[torch.randint(9, (b.blocks,), generator=gen)].to(torch.int8))
    index.scales.copy_(torch.tensor([0.0, 1e-3, 0.5, 0.5])[torch.randint(4, (b.blocks, 1), generator=gen)].expand(-1, kvh))
    query = vectors(gen, dtype, dev, b.tokens, heads, d)
    query[3] = 0
    got = index.select(query, b.tables, b.ctx, b.starts, block, k, num_sink_blocks=sinks, num_recent_blocks=recent)
    assert torch.equal(got.cpu(), selection(b, index, query, kvh, k, sinks, recent))
    into = torch.full_like(got, 7)
    assert index.select(query, b.tables, b.ctx, b.starts, block, k, sinks, recent, out=into) is into and torch.equal(into, got)
    # rows of no sequence
    part = index.select(query, b.tables[1:3], b.ctx[1:3], b.starts[1:4], block, k, sinks, recent).cpu()
    assert (part[:1] == -1).all() and (part[21:] == -1).all() and torch.equal(part[1:21], got[1:21].cpu())


def test_select_long_tables(dev):
    """More columns than a wavefront holds, and scores in slabs of tokens."""
    b = Batch([(40, 70000)], 2, dev, seed=6, pad_cols=100000)
    gen = torch.Generator().manual_seed(1)
    index = akv.BlockIndex(b.blocks, 16, 64, dev)
    index.codes.copy_(torch.randint(-127, 128, (b.blocks, 16, 64), generator=gen).to(torch.int8))
    index.scales.copy_(torch.rand(b.blocks, 16, generator=gen))
    query = vectors(gen, BF, dev, 40, 16, 64)
    got = index.select(query, b.tables, b.ctx, b.starts, 2, 500)
    assert torch.equal(got.cpu(), selection(b, index, query, 16, 500, 1, 2))


# ---- attention ------------------------------------------------------------------------------------------------
def sparse_reference(b, q, k, v, selected, scale):
    """(attention, attention over |v|, sum of |v| of the keys seen) in 64 bits on the host."""
    q, sel = q.cpu().double(), selected.cpu()
    out, size, total = (torch.zeros(q.shape, dtype=torch.float64) for _ in range(3))
    kvh = k.shape[2]
    group = q.shape[1] // kvh
    held = {i: (b.rows(k, i).cpu().double(), b.rows(v, i).cpu().double()) for i in range(len(b.lens)) if b.lens[i][1]}
    for i, row, pos in tokens_of(b):
        for h in range(kvh):
            cols = {c for c in sel[row, h].tolist() if 0 <= c <= pos // b.block} if pos >= 0 else set()
            at = [p for c in sorted(cols) for p in range(c * b.block, min((c + 1) * b.block, pos + 1))]
            if not at:
                continue
            kk, vv = held[i][0][at, h], held[i][1][at, h]
            w = torch.softmax(q[row, h * group:(h + 1) * group] @ kk.T * scale, -1)
            out[row, h * group:(h + 1) * group] = w @ vv
            size[row, h * group:(h + 1) * group] = w @ vv.abs()
            total[row, h * group:(h + 1) * group] = vv.abs().sum(0)
    return out, size, total


def assert_attention(got, b, q, k, v, selected, scale=None):
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    want, size, total = sparse_reference(b, q, k, v, selected, scale)
    u = HALF[q.dtype]
    off = (got.cpu().double() - want).abs()
    bound = (2 * u + 2.0 ** -14) * size + 2.0 ** -25 * total + 1e-30
    if q.dtype == FP:
        bound += 2.0 ** -25          # (outputs below float16's normal numbers)
    worst = (off / bound).max().item() if off.numel() else 0.0
    print(f"[sparse attention] error / bound {worst:.3f}")
    assert worst <= 1.0


def some_columns(gen, b, kvh, entries):
    """Selected columns in any order, with repetitions, entries below 0 and past the token's own block."""
    sel = torch.full((b.tokens, kvh, entries), -1, dtype=torch.int32)
    for i, row, pos in tokens_of(b):
        most = max(1, pos // b.block + 3)
        sel[row] = torch.randint(-2, most, (kvh, entries), generator=gen).int()
        if row % 3:
            sel[row, :, 0] = max(0, pos // b.block)
    sel[::7] = -1
    return sel


LENS = [(1, 700), (20, 300), (0, 50), (3, 3), (17, 17), (1, 1), (40, 513), (5, 2), (1, 64), (2, 1600)]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d,heads,kvh,block,entries", [
    (128, 32, 8, 16, 8), (64, 28, 4, 32, 5), (256, 16, 4, 16, 9), (128, 8, 8, 16, 30), (64, 64, 1, 16, 6), (128, 40, 2, 7, 13), (256, 5, 1, 1, 40), (64, 6, 2, 100, 3)])
def test_attention(dev, d, heads, kvh, block, entries, dtype):
    gen = torch.Generator().manual_seed(d + heads + block)
    b = Batch(LENS, block, dev, seed=7, index=torch.int64 if kvh == 2 else torch.int32)
    q, k, v = (vectors(gen, dtype, dev, *s) for s in ((b.tokens, heads, d), (b.blocks, block, kvh, d), (b.blocks, block, kvh, d)))
    b.unused(math.nan, k, v)
    sel = some_columns(gen, b, kvh, entries).to(dev)
    got = akv.paged_sparse_attention(q, k, v, b.tables, b.ctx, b.starts, sel)
    assert_attention(got, b, q, k, v, sel)
    # a given place for the result, rows of no sequence: left as they are, and zero in a new tensor
    into = torch.full_like(q, 3.0)
    part = akv.paged_sparse_attention(q, k, v, b.tables[1:3], b.ctx[1:3], b.starts[1:4], sel, out=into)
    assert part is into and torch.equal(part[1:21], got[1:21]) and (part[:1] == 3).all() and (part[21:] == 3).all()
    part = akv.paged_sparse_attention(q, k, v, b.tables[1:3], b.ctx[1:3], b.starts[1:4], sel)
    assert torch.equal(part[1:21], got[1:21]) and (part[:1] == 0).all() and (part[21:] == 0).all()


@pytest.mark.parametrize("dtype", [BF, FP])
def test_attention_over_everything_is_chunk_attention(dev, dtype):
    gen = torch.Generator().manual_seed(3)
    b = Batch(LENS, 16, dev, seed=8)
    q, k, v = (vectors(gen, dtype, dev, *s) for s in ((b.tokens, 16, 128), (b.blocks, 16, 4, 128), (b.blocks, 16, 4, 128)))
    sel = torch.arange(b.tables.shape[1], dtype=torch.int32, device=dev).expand(b.tokens, 4, -1)
    got = akv.paged_sparse_attention(q, k, v, b.tables, b.ctx, b.starts, sel, scale=0.2)
    assert_attention(got, b, q, k, v, sel, scale=0.2)
    dense = akv.paged_chunk_attention(q, k, v, b.tables, b.ctx, b.starts, scale=0.2)
    assert (got.float() - dense.float()).abs().max() < 0.05


def test_attention_large_scores(dev):
    """Scores of some hundred in size, rising and falling: the running maximum moves all the time."""
    gen = torch.Generator().manual_seed(4)
    for dtype in (BF, FP):
        b = Batch([(9, 900)], 16, dev, seed=9)
        q, k, v = (vectors(gen, dtype, dev, *s) for s in ((9, 8, 64), (b.blocks, 16, 2, 64), (b.blocks, 16, 2, 64)))
        q *= 8
        sel = torch.arange(57, dtype=torch.int32, device=dev).expand(9, 2, -1)
        got = akv.paged_sparse_attention(q, k, v, b.tables, b.ctx, b.starts, sel)
        want, size, total = sparse_reference(b, q, k, v, sel, 1 / 8)
        # (scores of 2^8: 64 products, each rounded by 2^-24 of up to 2^9, move a weight by 2^-9 at most)
        assert ((got.cpu().double() - want).abs() <= (2 * HALF[dtype] + 2.0 ** -8) * size + 2.0 ** -25 * total + 2.0 ** -25).all()


# ---- weights --------------------------------------------------------------------------------------------------
def weights_reference(b, q, keys, scale, sizes=None):
    """(weights [seqs, kv heads, length], the largest sum of |products| of a score) in 64 bits; keys(i): of sequence i."""
    length = b.tables.shape[1] * b.block
    q = q.cpu().double()
    out = None
    most = 0.0
    at = 0
    for i, (n, c) in enumerate(b.lens):
        k = keys(i).cpu().double() if c else None
        if out is None:
            kvh = b.kvh
            group = q.shape[1] // kvh
            out = torch.zeros(len(b.lens), kvh, length, dtype=torch.float64)
        if n and c:
            hidden = torch.arange(c)[None] > torch.arange(c - n, c)[:, None]
            for g in range(q.shape[1]):
                s = (q[at:at + n, g] @ k[:, g // group].T * scale).masked_fill(hidden, -math.inf)
                w = torch.softmax(s, 1)
                out[i, g // group, :c] += torch.where(hidden.all(1, keepdim=True), 0.0, w).sum(0)
                e = (q[at:at + n, g].abs() @ k[:, g // group].abs().T * scale).masked_fill(hidden, 0.0)
                most = max(most, e.max().item())
        at += n
    return out, most


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d,heads,kvh,block", [(128, 32, 8, 16), (64, 28, 4, 32), (256, 16, 16, 16), (128, 8, 1, 7), (64, 40, 2, 1), (256, 8, 2, 100)])
def test_weights(dev, d, heads, kvh, block, dtype):
    gen = torch.Generator().manual_seed(d + heads)
    b = Batch(LENS, block, dev, seed=10, index=torch.int64 if kvh == 1 else torch.int32)
    b.kvh = kvh
    q, k = vectors(gen, dtype, dev, b.tokens, heads, d), vectors(gen, dtype, dev, b.blocks, block, kvh, d)
    b.unused(math.nan, k)
    got = akv.paged_key_weights(q, k, b.tables, b.ctx, b.starts)
    want, most = weights_reference(b, q, lambda i: b.rows(k, i), 1 / math.sqrt(d))
    rel = 2 * most * d * 2.0 ** -24 + 2.0 ** -20
    off = (got.cpu().double() - want).abs()
    print(f"[weights] error / bound {(off / (rel * want + 1e-30)).max().item():.3f}")
    # (the bound takes every error at its worst at once; in the mean they are far from it)
    assert got.dtype == torch.float32 and got.shape == want.shape and (off <= rel * want + 1e-30).all() and (off.square().sum() / want.square().sum()).sqrt() < 2e-6
    # a row's weights sum to one: a sequence's to the rows that see a key
    rows = torch.tensor([sum(c - n + j >= 0 for j in range(n)) * heads // kvh for n, c in LENS], dtype=torch.float64)
    assert (got.double().sum(2).cpu() - rows[:, None]).abs().max() <= 2.0 ** -18 * rows.max()
    # added to what is there, and nothing else touched
    acc = torch.full((len(LENS) + 1, kvh, got.shape[2] + 5), 0.5, device=dev)
    assert akv.paged_key_weights(q, k, b.tables, b.ctx, b.starts, accumulated=acc) is acc
    for i, (_, c) in enumerate(LENS):
        assert torch.equal(acc[i, :, :c], 0.5 + got[i, :, :c]) and (acc[i, :, c:] == 0.5).all()
    assert (acc[-1] == 0.5).all()


@pytest.mark.parametrize("bits", [4, 3, 2])
@pytest.mark.parametrize("d,heads,kvh,block,dtype", [(128, 32, 8, 16, FP), (64, 28, 4, 32, BF), (256, 16, 16, 16, FP), (128, 8, 1, 7, BF)])
def test_packed_weights(dev, d, heads, kvh, block, dtype, bits):
    from oracle import tq_oracle as O
    gen = torch.Generator().manual_seed(d + bits)
    b = Batch(LENS, block, dev, seed=11)
    b.kvh = kvh
    tq = akv.TurboQuant(head_dim=d, bits=bits, device=dev)
    row = d * bits // 8
    kp = torch.randint(256, (b.blocks, block, kvh, row + 4), dtype=torch.uint8, generator=gen).to(dev)[..., :row]
    kn = (math.sqrt(d) * torch.exp(0.3 * torch.randn(b.blocks, block, kvh, generator=gen))).to(dev)
    b.unused(math.nan, kn)
    q = vectors(gen, dtype, dev, b.tokens, heads, d)
    attn = akv.TQPagedAttention(tq, heads)
    got = attn.key_weights(q, kp, kn, b.tables, b.ctx, b.starts, block_size=block)
    levels, pi = tq.centroids.cpu().double(), tq.rotation.cpu().double()

    def keys(i):
        codes = O._UNPACK[bits](b.rows(kp, i).cpu().numpy().reshape(-1, row), d)
        return (levels[torch.from_numpy(codes.astype(np.int64))].view(-1, kvh, d) @ pi) * b.rows(kn, i).cpu().double()[..., None]

    want, _ = weights_reference(b, q, keys, 1 / math.sqrt(d))
    turned = (q.cpu().double().abs() @ pi.abs().T).sum(-1).max().item()
    most = turned * levels.abs().max().item() * kn[~kn.isnan()].max().item() / math.sqrt(d)
    rel = 2 * most * (2 * d * 2.0 ** -24 + 3 * 2.0 ** -22) + 2.0 ** -20
    off = (got.cpu().double() - want).abs()
    # the bound takes every error at its worst at once; in the mean they are far from it
    mean = (off.square().sum() / want.square().sum()).sqrt().item()
    print(f"[packed weights] error / bound {(off / (rel * want + 1e-30)).max().item():.4f}, rms {mean:.2e}")
    assert (off <= rel * want + 1e-30).all() and mean < 2e-6
    acc = torch.zeros_like(got)
    attn.key_weights(q, kp, kn, b.tables, b.ctx, b.starts, block_size=block, accumulated=acc)
    assert torch.equal(acc, got)


# ---- eviction -------------------------------------------------------------------------------------------------
def kept_reference(w, n, keep, sinks, recent):
    if n <= keep:
        return np.arange(n)
    w = np.where(np.isnan(w[:n]), -np.inf, w[:n])
    at = np.arange(n)
    forced = (at < sinks) | (at >= n - recent)
    return np.sort(np.lexsort((at, -w, ~forced))[:keep])


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("block,kvh,keep,sinks,recent,index", [(16, 8, 100, 4, 32, torch.int32), (32, 3, 1, 0, 0, torch.int64), (7, 1, 300, 0, 1, torch.int32), (1, 2, 64, 64, 0, torch.int32),
                                                               (100, 4, 999, 5, 500, torch.int64), (16, 2, 5000, 0, 0, torch.int32)])
def test_evict(dev, block, kvh, keep, sinks, recent, index, in_place):
    gen = torch.Generator().manual_seed(block + keep)
    lens = [700, 0, 1, 99, 100, 101, 1024, 1025, 3, 9000, 2000]
    b = Batch([(0, c) for c in lens], block, dev, seed=12, index=index)
    length = b.tables.shape[1] * block + 3
    w = torch.exp(2 * torch.randn(len(lens), kvh, length, generator=gen))
    w[torch.rand(w.shape, generator=gen) < 0.3] = 0.0
    w[:, :, 5::11] = -0.0
    w[0, 0, ::2], w[4], w[5, :, 50], w[6, :, :60] = math.nan, 1.0, math.inf, -math.inf
    w = w.to(dev)
    caches = [torch.randn(b.blocks, block, kvh, 128, generator=gen).to(BF).to(dev), torch.randint(256, (b.blocks, 2, block, kvh, 68), dtype=torch.uint8, generator=gen).to(dev)[:, 1, ..., :64],
              torch.randn(b.blocks, block, kvh, generator=gen).to(dev), torch.randn(b.blocks, kvh, block, 6, generator=gen).half().to(dev).transpose(1, 2),
              torch.randint(256, (b.blocks, block, kvh, 5), dtype=torch.uint8, generator=gen).to(dev)]
    to, host_to = None, b.host
    if not in_place:
        need = [-(-min(c, keep) // block) for c in lens]
        old = b.blocks
        host_to = np.full((len(lens), max(1, -(-min(keep, b.tables.shape[1] * block) // block))), 1 << 20, dtype=np.int64)
        order, at = np.random.default_rng(1).permutation(sum(need)) + old, 0
        for i, n in enumerate(need):
            host_to[i, :n] = order[at:at + n]
            at += n
        caches = [torch.cat([c, torch.zeros_like(c[:1]).expand(sum(need), *c.shape[1:])]) for c in caches]
        to = torch.from_numpy(host_to).to(dev, index)
    before = [c.clone() for c in caches]
    kept, now, left = akv.evict_tokens(w, b.tables, b.ctx, caches, keep, num_sink=sinks, num_recent=recent, out_tables=to)
    assert kept.dtype == torch.int32 and now.dtype == index and left.shape == w.shape
    assert now.tolist() == [min(c, keep) for c in lens]
    kept_host, want = kept.cpu().numpy(), [c.clone().cpu() for c in before]
    left_host, w_host = left.cpu().numpy(), w.cpu().numpy()
    for i, c in enumerate(lens):
        for h in range(kvh):
            ref = kept_reference(w_host[i, h], c, keep, sinks, recent)
            n = len(ref)
            assert np.array_equal(kept_host[i, h, :n], ref) and (kept_host[i, h, n:] == -1).all(), (i, h)
            assert np.array_equal(left_host[i, h, :n], w_host[i, h, ref], equal_nan=True) and (left_host[i, h, n:] == 0).all()
            to_pos = np.arange(n)
            for x, y in zip(before, want):
                y[host_to[i, to_pos // block], to_pos % block, h] = x.cpu()[b.host[i, ref // block], ref % block, h]
    for x, y in zip(caches, want):
        assert torch.equal(x.cpu(), y)


def test_evict_long(dev):
    """More positions than the registers hold, and than one of the smaller forms."""
    for n in (8192, 8200, 32768, 32769, 150000):
        gen = torch.Generator().manual_seed(n)
        w = torch.rand(1, 2, n, generator=gen)
        w[0, 1] = (w[0, 1] * 50).floor()
        b = Batch([(0, n)], 16, dev, seed=13, pad_cols=0)
        w = torch.nn.functional.pad(w, (0, b.tables.shape[1] * 16 - n))
        cache = torch.arange(b.blocks * 16 * 2, device=dev).view(b.blocks, 16, 2)
        before = b.rows(cache, 0).clone()
        kept, now, _ = akv.evict_tokens(w.to(dev), b.tables, b.ctx, [cache], n // 3)
        for h in range(2):
            ref = kept_reference(w[0, h].numpy(), n, n // 3, 4, 32)
            assert np.array_equal(kept[0, h].cpu().numpy(), ref)
            assert torch.equal(b.rows(cache, 0)[:n // 3, h], before[torch.from_numpy(ref).to(dev), h])


@pytest.mark.parametrize("kind", ["alike", "two values", "outlier", "near", "rising"])
def test_select_scores_of_all_kinds(dev, kind):
    """Scores that fall into one part of the histogram, by the hundred or all of them, on tables of every width class."""
    gen = torch.Generator().manual_seed(len(kind))
    for context, pad in ((1500, 0), (3000, 2), (7000, 4000), (9000, 20000)):
        b = Batch([(20, context), (3, context // 2)], 1, dev, seed=14, pad_cols=pad)
        index = akv.BlockIndex(b.blocks, 2, 64, dev)
        codes = torch.zeros(b.blocks, 2, 64, dtype=torch.int8)
        codes[:, :, 0] = 100
        scales = torch.ones(b.blocks, 2)
        if kind == "two values":
            scales[torch.rand(b.blocks, generator=gen) < 0.5] = 0.75
        elif kind == "outlier":
            scales = 1 + torch.rand(b.blocks, 2, generator=gen)
            scales[3], codes[7, :, 0] = 1e30, -100
            scales[7] = 1e30
        elif kind == "near":
            scales = 1 + torch.randint(40, (b.blocks, 2), generator=gen) * 2.0 ** -23
        elif kind == "rising":
            scales = 1.02 ** (torch.arange(b.blocks * 2).view(-1, 2) % 3001) * 1e-20
        index.codes.copy_(codes)
        index.scales.copy_(scales)
        query = torch.zeros(b.tokens, 4, 64, dtype=BF, device=dev)
        query[:, :, 0] = 1.0
        query[1::2] *= -1
        for k in (5, 400):
            got = index.select(query, b.tables, b.ctx, b.starts, 1, k, num_sink_blocks=2, num_recent_blocks=2)
            assert torch.equal(got.cpu(), selection(b, index, query, 2, k, 2, 2)), (context, k)
