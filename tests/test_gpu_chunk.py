"""A chunk of new tokens: rope_append, paged_chunk_attention and TQPagedAttention.forward_chunk against plain implementations in 64 bits.

Tolerances.  u is half a step of the 16-bit type (2^-8 bfloat16, 2^-11 float16).  Attention with exact scores: every weight is rounded
once (u of itself; float16 weights below 2^-14 of the largest by up to 2^-25 of the largest, and the sum of weights is at least the
largest) and so is the output, so a coordinate is off by at most (2 u + 2^-14) A + 2^-25 B with A the same attention over |v| and B
the sum of |v| over the keys; 2^-14 covers what is done in float32 (scores of up to 2^8: 128 products of 2^-24 each and their
exponential, as relative errors of the weights).  Packed rows: queries (rotated) and levels are float16 besides, each off by 2^-11,
which moves a score by at most 2^-10 E with E = scale |k| sum |q'_i c_i|, a weight by the factor exp(2 max E 2^-10), and a value
by 2^-11 |c| in the rotated domain, whose effect on a coordinate is at most 2^-11 sum |Pi_ij| A'_i with A' the attention over |v| |c|."""
import math

import numpy as np
import pytest
import torch

import aitherkvcache_amd as akv

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BF, FP = torch.bfloat16, torch.float16


class Batch:
    """Sequences of (new, context) tokens over a pool of blocks in random order; table entries past a context are out of range."""

    def __init__(self, lens, block, dev, seed, index=torch.int32, spare=2, pad_cols=2):
        rng = np.random.default_rng(seed)
        self.lens, self.block = lens, block
        need = [-(-c // block) for _, c in lens]
        self.blocks = sum(need) + spare
        order = rng.permutation(self.blocks)
        tables = np.full((max(1, len(lens)), max([1] + need) + pad_cols), 1 << 20, dtype=np.int64)
        tables[:, 1::2] = -7
        at = 0
        for i, n in enumerate(need):
            tables[i, :n] = order[at:at + n]
            at += n
        self.host = tables
        self.tables = torch.from_numpy(tables[:len(lens)]).to(dev, index)
        self.ctx = torch.tensor([c for _, c in lens], dtype=index, device=dev)
        self.starts = torch.tensor(np.cumsum([0] + [n for n, _ in lens]), dtype=index, device=dev)
        self.tokens = sum(n for n, _ in lens)

    def rows(self, cache, i):
        """What sequence i holds of a cache, [tokens, ...]."""
        c, bs = self.lens[i][1], self.block
        return cache[torch.from_numpy(self.host[i, :-(-c // bs)]).to(cache.device)].flatten(0, 1)[:c]

    def unused(self, fill, *caches):
        """`fill` into everything that no sequence holds: spare blocks, places behind a context in its last block."""
        for cache in caches:
            used = torch.zeros(cache.shape[:2], dtype=torch.bool, device=cache.device)
            for i, (_, c) in enumerate(self.lens):
                for b in range(-(-c // self.block)):
                    used[self.host[i, b], :min(self.block, c - b * self.block)] = True
            cache[~used] = fill


def hidden_of(n, c, window, dev):
    pos, key = torch.arange(c - n, c, device=dev)[:, None], torch.arange(c, device=dev)[None]
    return (key > pos) | ((key <= pos - window) if window else torch.zeros_like(key > pos))


def softmax_rows(logits, hidden):
    w = torch.softmax(logits.masked_fill(hidden, -math.inf), -1)
    return torch.where(hidden.all(-1, keepdim=True), torch.zeros_like(w), w)


def dense_reference(b, q, kc, vc, scale, window):
    """(out, bound) in float64."""
    u, out, bound = HALF[q.dtype], torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    group, at = q.shape[1] // kc.shape[2], 0
    for i, (n, c) in enumerate(b.lens):
        if c and n:
            k, v = b.rows(kc, i).double(), b.rows(vc, i).double()
            hidden = hidden_of(n, c, window, q.device)
            for h in range(q.shape[1]):
                w = softmax_rows(q[at:at + n, h].double() @ k[:, h // group].T.contiguous() * scale, hidden)
                x = v[:, h // group].contiguous()
                out[at:at + n, h] = w @ x
                small = (~hidden).double() @ x.abs() if q.dtype == FP else 0.0
                bound[at:at + n, h] = (2 * u + 2.0 ** -14) * (w @ x.abs()) + 2.0 ** -25 * small + 1e-30
        at += n
    return out, bound


def check(got, out, bound):
    assert bool(torch.isfinite(got).all())
    over = ((got.double() - out).abs() / bound.clamp_min(1e-30))
    assert float(over.max()) <= 1.0, f"{float(over.max())} of the bound at {np.unravel_index(int(over.argmax()), over.shape)}"


def vectors(rng_seed, dev, dtype, *shape):
    g = torch.Generator(device=dev).manual_seed(rng_seed)
    x = torch.randn(shape, device=dev, generator=g)
    return (x * torch.exp(0.5 * torch.randn(shape[:-1], device=dev, generator=g))[..., None]).to(dtype)


def run_dense(b, d, heads, kv, dtype, dev, seed, window=0, fill=math.nan, **more):
    q, kc, vc = (vectors(seed + i, dev, dtype, *s) for i, s in enumerate(((b.tokens, heads, d), (b.blocks, b.block, kv, d), (b.blocks, b.block, kv, d))))
    b.unused(fill, kc, vc)
    got = akv.paged_chunk_attention(q, kc, vc, b.tables, b.ctx, b.starts, window=window, **more)
    out, bound = dense_reference(b, q, kc, vc, 1 / math.sqrt(d), window)
    check(got, out, bound)
    return q, kc, vc, got


# lengths (new, context with them) around the edges of tiles: 32 rows, 64 and 128 keys, blocks of 16
FEW = [(1, 1), (2, 2), (1, 31), (3, 33), (1, 64), (4, 65), (2, 127), (1, 128), (8, 129), (5, 700), (1, 0), (0, 40), (3, 2)]
MANY = [(40, 40), (130, 130), (65, 300), (64, 64), (257, 500), (33, 1000), (100, 90)]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens", [FEW, MANY, MANY + FEW], ids=["few", "many", "both"])
def test_dense_lengths(dev, d, dtype, lens):
    run_dense(Batch(lens, 16, dev, d), d, 8, 2, dtype, dev, 11)


@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (5, 1), (14, 2), (32, 4), (33, 1), (66, 2), (130, 1)])
@pytest.mark.parametrize("lens", [[(1, 90), (2, 260)], [(70, 200), (3, 30)]], ids=["few", "many"])
def test_dense_heads(dev, heads, kv, lens):
    run_dense(Batch(lens, 16, dev, heads), 64, heads, kv, BF, dev, 12)


@pytest.mark.parametrize("block", [1, 5, 32, 48, 256])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_dense_blocks_and_index_types(dev, block, index):
    run_dense(Batch([(3, 200), (90, 333)], block, dev, block, index), 128, 8, 2, FP, dev, 13)


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 200, 1 << 30])
@pytest.mark.parametrize("lens", [[(1, 500), (7, 300)], [(150, 500), (150, 150), (2, 500), (60, 30)]], ids=["few", "many"])
def test_dense_windows(dev, window, lens):
    run_dense(Batch(lens, 16, dev, window % 97), 128, 8, 2, BF, dev, 14, window=window)


def test_dense_long_contexts_are_split(dev):
    run_dense(Batch([(2, 30000), (1, 17)], 16, dev, 1), 128, 4, 1, BF, dev, 15)
    run_dense(Batch([(200, 20000)], 16, dev, 2), 64, 4, 1, FP, dev, 16)


@pytest.mark.parametrize("hint", [None, 1, 9, 4096])
def test_dense_hint_does_not_matter(dev, hint):
    """Results are the same whatever the hint says, also where it is wrong."""
    b = Batch([(9, 300), (80, 200), (1, 77)], 16, dev, 3)
    run_dense(b, 128, 16, 4, BF, dev, 17, max_query_len=hint)


def test_dense_views_and_padding(dev):
    """Queries as a slice of a fused projection, caches as halves of one tensor, rows behind the last sequence."""
    b = Batch([(5, 90), (70, 100)], 16, dev, 4)
    heads, kv, d = 8, 2, 128
    fused = vectors(18, dev, BF, b.tokens + 3, heads + 2 * kv, d)
    cache = vectors(19, dev, BF, b.blocks, 2, b.block, kv, d)
    q, kc, vc = fused[:, :heads], cache[:, 0], cache[:, 1]
    out, bound = dense_reference(b, q[:b.tokens], kc, vc, 0.11, 0)
    got = akv.paged_chunk_attention(q, kc, vc, b.tables, b.ctx, b.starts, scale=0.11)
    check(got[:b.tokens], out, bound)
    assert not bool(got[b.tokens:].any())
    mine = torch.full((b.tokens + 3, heads + 1, d), 7.0, dtype=BF, device=dev)
    assert akv.paged_chunk_attention(q, kc, vc, b.tables, b.ctx, b.starts, scale=0.11, out=mine[:, :heads]).data_ptr() == mine.data_ptr()
    assert torch.equal(mine[:b.tokens, :heads], got[:b.tokens]) and bool((mine[b.tokens:] == 7).all()) and bool((mine[:, heads:] == 7).all())
    odd = vectors(20, dev, BF, b.tokens, heads, d + 1)[..., 1:]           # rows at odd places are copied
    a, c = (akv.paged_chunk_attention(x, kc, vc, b.tables, b.ctx, b.starts) for x in (odd, odd.contiguous()))
    assert torch.equal(a, c)


def test_dense_empty_batches(dev):
    kc = torch.ones(2, 16, 2, 64, dtype=FP, device=dev)
    none = torch.empty(0, 8, 64, dtype=FP, device=dev)
    zero = torch.zeros(1, dtype=torch.int32, device=dev)
    t = torch.zeros(0, 1, dtype=torch.int32, device=dev)
    assert akv.paged_chunk_attention(none, kc, kc, t, zero[:0], zero).shape == (0, 8, 64)
    q = torch.ones(3, 8, 64, dtype=FP, device=dev)
    assert not bool(akv.paged_chunk_attention(q, kc, kc, t, zero[:0], zero).any())                    # no sequences: rows of nobody
    assert not bool(akv.paged_chunk_attention(q, kc[:0], kc[:0], zero[None], zero + 5, torch.tensor([0, 3], device=dev)).any())     # no blocks


def test_dense_large_scores(dev):
    """Scores of some thousands, where weights are 0 or 1 and a maximum that is not carried overflows."""
    b = Batch([(4, 300), (90, 300)], 16, dev, 5)
    q, kc, vc = vectors(21, dev, BF, b.tokens, 4, 128) * 30, vectors(22, dev, BF, b.blocks, 16, 2, 128) * 30, vectors(23, dev, BF, b.blocks, 16, 2, 128)
    got = akv.paged_chunk_attention(q, kc, vc, b.tables, b.ctx, b.starts)
    out, _ = dense_reference(b, q, kc, vc, 1 / math.sqrt(128), 0)
    # a score of up to s is off by 128 products' roundings, 2^-17 of sum |q k| scale at most
    at, worst = 0, torch.zeros(b.tokens, device=dev, dtype=torch.float64)
    for i, (n, c) in enumerate(b.lens):
        k = b.rows(kc, i).double().abs().amax(1)
        worst[at:at + n] = (q[at:at + n].double().abs().amax(1) @ k.T.contiguous()).amax(1) / math.sqrt(128) * 2.0 ** -17
        at += n
    bound = (2 * HALF[BF] + 2.0 ** -14 + 2 * torch.expm1(2 * worst))[:, None, None] * vc.double().abs().amax()
    check(got, out, bound.expand_as(out))


# ---- packed ------------------------------------------------------------------------------------------------------------

def unpack(rows, bits, d):
    w = torch.from_numpy(np.unpackbits(rows[..., :d * bits // 8].cpu().numpy(), axis=-1)).view(*rows.shape[:-1], d, bits)
    return (w.long() * (1 << torch.arange(bits - 1, -1, -1))).sum(-1).to(rows.device)


class Packed:
    def __init__(self, b, d, bits, heads, kv, dtype, dev, seed, primary=False, scale_norms=1.0, centroids=None):
        self.tq = akv.TurboQuant(head_dim=d, bits=bits, device=str(dev), seed=seed)
        if centroids is not None:
            self.tq.centroids = centroids.to(dev)
        self.attn = akv.TQPagedAttention(self.tq, heads)
        g = torch.Generator(device=dev).manual_seed(seed)
        row = d * bits // 8
        if primary:
            kv_cache = torch.randint(0, 256, (b.blocks, 2, b.block, kv, row + 4), dtype=torch.uint8, device=dev, generator=g)
            self.k, self.v = kv_cache[:, 0, :, :, :row], kv_cache[:, 1, :, :, :row]
        else:
            self.k, self.v = (torch.randint(0, 256, (b.blocks, b.block, kv, row), dtype=torch.uint8, device=dev, generator=g) for _ in range(2))
        self.kn, self.vn = (math.sqrt(d) / 2 * scale_norms * torch.exp(0.5 * torch.randn(b.blocks, b.block, kv, device=dev, generator=g)) for _ in range(2))
        b.unused(math.nan, self.kn, self.vn)
        self.q = torch.randn(b.tokens, heads, d, device=dev, generator=g).to(dtype)
        self.b, self.d, self.bits = b, d, bits

    def run(self, **more):
        b = self.b
        return self.attn.forward_chunk(self.q, self.k, self.kn, self.v, self.vn, b.tables, b.ctx, b.starts, block_size=b.block, **more)

    def reference(self):
        b, q, d = self.b, self.q, self.d
        pi, cen, scale = self.tq.rotation.double(), self.tq.centroids.double(), self.attn.scale
        u, out, bound = HALF[q.dtype], torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        group, at = q.shape[1] // self.k.shape[2], 0
        for i, (n, c) in enumerate(b.lens):
            if c and n:
                ck, cv = (cen[unpack(b.rows(x, i), self.bits, d)] for x in (self.k, self.v))
                kn, vn = b.rows(self.kn, i).double(), b.rows(self.vn, i).double()
                hidden = hidden_of(n, c, 0, q.device)
                for h in range(q.shape[1]):
                    j = h // group
                    turned = q[at:at + n, h].double() @ pi.T.contiguous()
                    k, v = ck[:, j].contiguous(), cv[:, j] * vn[:, j, None]
                    w = softmax_rows(turned @ k.T.contiguous() * kn[:, j] * scale, hidden)
                    out[at:at + n, h] = w @ v @ pi
                    e = ((turned.abs() @ k.abs().T.contiguous()) * kn[:, j] * scale).masked_fill(hidden, 0.0).amax(1, keepdim=True) * 2.0 ** -10
                    a, sum_v = (w @ v.abs()), (~hidden).double() @ v.abs()
                    in_turned = (torch.expm1(2 * e) + 2.0 ** -11 + 2.0 ** -11 + 2.0 ** -13) * a * (1 + torch.expm1(2 * e)) + 2.0 ** -25 * sum_v
                    bound[at:at + n, h] = in_turned @ pi.abs() + u * out[at:at + n, h].abs() + 1e-30
            at += n
        return out, bound


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bits", [4, 3, 2])
@pytest.mark.parametrize("lens", [FEW, MANY, MANY[:3] + FEW[-6:]], ids=["few", "many", "both"])
def test_packed_lengths(dev, d, bits, lens):
    p = Packed(Batch(lens, 16, dev, bits), d, bits, 8, 2, BF if d != 64 else FP, dev, 31, primary=bits != 3)
    check(p.run(), *p.reference())


@pytest.mark.parametrize("heads,kv", [(3, 3), (14, 2), (33, 1), (130, 1)])
@pytest.mark.parametrize("block,index", [(16, torch.int64), (7, torch.int32)])
def test_packed_heads_and_blocks(dev, heads, kv, block, index):
    p = Packed(Batch([(2, 90), (40, 150)], block, dev, heads, index), 64, 4, heads, kv, FP, dev, 32)
    check(p.run(), *p.reference())


def test_packed_long_context_is_split(dev):
    p = Packed(Batch([(3, 21000)], 16, dev, 6), 128, 4, 8, 1, FP, dev, 33)
    check(p.run(), *p.reference())


@pytest.mark.parametrize("d,bits", [(64, 4), (128, 4), (128, 3), (128, 2), (256, 4)])
def test_packed_many_keys_a_workgroup(dev, d, bits):
    """Ranges of some twenty units and several tiles."""
    p = Packed(Batch([(700, 2900), (333, 6001)], 16, dev, 7), d, bits, 16, 2, BF, dev, 38)
    check(p.run(), *p.reference())


@pytest.mark.parametrize("d", [64, 128, 256])
def test_dense_many_keys_a_workgroup(dev, d):
    run_dense(Batch([(900, 3100), (333, 6001)], 16, dev, 8), d, 32, 4, BF, dev, 24)


@pytest.mark.parametrize("lens", [[(3, 200)], [(90, 200)]], ids=["few", "many"])
def test_packed_norms_of_any_size(dev, lens):
    """Value norms from 0 over 2^-60 to 2^60 of each other: the largest weights times norms decide, and the others are not lost
    where those are far away."""
    b = Batch(lens, 16, dev, 7)
    p = Packed(b, 128, 4, 8, 2, BF, dev, 34)
    p.vn.mul_(2.0 ** torch.randint(-60, 60, p.vn.shape, device=dev, generator=torch.Generator(device=dev).manual_seed(1)))
    p.vn[:, 3] = 0.0
    p.kn.mul_(0.01)
    check(p.run(), *p.reference())
    p.vn.zero_()
    assert not bool(p.run().any())


@pytest.mark.parametrize("size", [1e-20, 1.0, 3e20])
def test_packed_codebooks_of_any_size(dev, size):
    """Levels in any order and of any size, without symmetry."""
    cen = torch.randn(16, generator=torch.Generator().manual_seed(3)) * size
    b = Batch([(2, 100), (50, 100)], 16, dev, 8)
    p = Packed(b, 64, 4, 4, 2, BF, dev, 35, scale_norms=1.0, centroids=cen)
    p.kn.mul_(0.05 / size)
    p.vn.mul_(min(1.0, 1e10 / size))
    check(p.run(), *p.reference())


def test_packed_one_token_is_forward(dev):
    """A chunk of one token a sequence is what forward() computes."""
    b = Batch([(1, 1), (1, 77), (1, 900), (1, 4000)], 16, dev, 9)
    p = Packed(b, 128, 4, 32, 8, FP, dev, 36, primary=True)
    want = p.attn.forward(p.q, p.k, p.kn, p.v, p.vn, b.tables, b.ctx, block_size=16)
    out, bound = p.reference()
    check(p.run(), out, bound)
    assert float((p.run().double() - want.double()).abs().max()) <= float((2 * bound).max())


def test_packed_padding_and_empty(dev):
    b = Batch([(3, 50), (40, 60)], 16, dev, 10)
    p = Packed(b, 128, 3, 8, 2, BF, dev, 37)
    want = p.run()
    q, p.q = p.q, torch.cat([p.q, torch.ones(2, 8, 128, dtype=BF, device=dev)])
    got = p.run()
    assert torch.equal(got[:-2], want) and not bool(got[-2:].any())
    mine = torch.full_like(got, 5.0)
    p.run(out=mine)
    assert torch.equal(mine[:-2], want) and bool((mine[-2:] == 5).all())
    b.ctx.zero_()
    assert not bool(p.run().any())


# ---- rotary positions and the append -----------------------------------------------------------------------------------

def rope_reference(x, pos, table, sections, interleaved):
    """Rows of float64 turned, and the bound of one rounding of each product and the sum in float32 (3 x 2^-24 of |x1 c| + |x2 s|)."""
    half = table.shape[1] // 2
    axis = np.repeat(np.arange(len(sections)), sections) if sections else np.zeros(half, dtype=int)
    p = torch.arange(half, device=x.device)
    at = (pos if sections else pos[None]).long().clamp(0, table.shape[0] - 1)[torch.from_numpy(axis).to(x.device)].T       # [tokens, half]
    c, s = table.double()[at, p][:, None], table.double()[at, half + p][:, None]
    i, j = (2 * p, 2 * p + 1) if interleaved else (p, half + p)
    out, bound = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    a, b = x.double()[..., i], x.double()[..., j]
    out[..., i], out[..., j] = a * c - b * s, b * c + a * s
    bound[..., i], bound[..., j] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return out, bound * 3 * 2.0 ** -24


def check_rope(got, out, bound):
    u = {torch.float32: 2.0 ** -24, **HALF}[got.dtype]
    tiny = {torch.float32: 0.0, BF: 0.0, FP: 2.0 ** -25}[got.dtype]
    assert bool(((got.double() - out).abs() <= bound * (1 + u) + u * out.abs() + tiny).all())


def table_of(rows, rotary, dev):
    a = torch.arange(rows, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    return torch.cat([a.cos(), a.sin()], 1).float().to(dev)


@pytest.mark.parametrize("tokens", [1, 2, 17, 300])
@pytest.mark.parametrize("d,rotary,sections,interleaved", [(128, 128, None, False), (128, 64, None, True), (64, 16, (3, 5), False), (256, 256, (50, 1, 77), True),
                                                           (128, 128, (16, 24, 24), False), (80, 48, (1, 2, 3, 18), False), (128, 128, (0, 64), True)])
@pytest.mark.parametrize("dtype,cache_dtype", [(BF, BF), (FP, BF), (torch.float32, FP), (FP, torch.float32), (torch.float32, torch.float32)])
def test_rope_append(dev, tokens, d, rotary, sections, interleaved, dtype, cache_dtype):
    heads, kv, block = 5, 2, 16
    q, k, v = (vectors(40 + i, dev, dtype, tokens, h, d) for i, h in enumerate((heads, kv, kv)))
    table = table_of(500, rotary, dev)
    g = torch.Generator(device=dev).manual_seed(tokens)
    pos = torch.randint(-3, 505, (len(sections), tokens) if sections else (tokens,), device=dev, generator=g)      # clamped
    blocks = -(-tokens // block) + 3
    slots = torch.randperm(blocks * block, device=dev, generator=g)[:tokens]
    if tokens > 2:
        slots[1], slots[2] = -1, blocks * block + 5
    kc, vc = torch.full((blocks, block, kv, d), 3.0, dtype=cache_dtype, device=dev), torch.full((blocks, block, kv, d), 4.0, dtype=cache_dtype, device=dev)
    keep = q.clone()
    got = akv.rope_append(q, k, v, pos, table, slots, kc, vc, sections=sections, interleaved=interleaved)
    assert torch.equal(q, keep)
    check_rope(got, *rope_reference(q, pos, table, sections, interleaved))
    ok = (slots >= 0) & (slots < blocks * block)
    out, bound = rope_reference(k, pos, table, sections, interleaved)
    check_rope(kc.flatten(0, 1)[slots[ok]], out[ok], bound[ok])
    assert torch.equal(vc.flatten(0, 1)[slots[ok]], v[ok].to(cache_dtype))
    rest = torch.ones(blocks * block, dtype=torch.bool, device=dev)
    rest[slots[ok]] = False
    assert bool((kc.flatten(0, 1)[rest] == 3).all()) and bool((vc.flatten(0, 1)[rest] == 4).all())


def test_rope_views_in_place_and_without(dev):
    """Slices of a fused projection rotated in place; halves of one cache; rows at odd places; no queries; no rotation."""
    heads, kv, d, tokens = 4, 2, 64, 33
    table, pos = table_of(64, 64, dev), torch.arange(tokens, device=dev, dtype=torch.int32)
    fused = vectors(50, dev, BF, tokens, heads + 2 * kv, d)
    q, k, v = fused[:, :heads], fused[:, heads:heads + kv], fused[:, heads + kv:]
    cache, odd = torch.zeros(4, 2, 16, kv, d, dtype=BF, device=dev), torch.zeros(4, 2, 16, kv, d + 1, dtype=BF, device=dev)
    slots = torch.randperm(64, device=dev)[:tokens].int()
    want = akv.rope_append(q, k, v, pos, table, slots, cache[:, 0], cache[:, 1])
    akv.rope_append(q, k, v, pos, table, slots, odd[:, 0, :, :, :d], odd[:, 1, :, :, :d])
    assert torch.equal(odd[..., :d], cache) and not bool(odd[..., d].any())
    other = torch.zeros_like(cache)
    assert akv.rope_append(None, k, v, pos, table, slots, other[:, 0], other[:, 1]) is None and torch.equal(other, cache)
    akv.rope_append(None, k, v, None, None, slots, other[:, 0], other[:, 1])
    assert torch.equal(other[:, 0].flatten(0, 1)[slots.long()], k) and torch.equal(other[:, 1], cache[:, 1])
    assert akv.rope_append(q, k, v, pos, table, slots, cache[:, 0], cache[:, 1], query_out=q) is q and torch.equal(q, want)
    empty = fused[:0]
    assert akv.rope_append(empty[:, :heads], empty[:, :kv], empty[:, :kv], pos[:0], table, slots[:0], cache[:, 0], cache[:, 1]).shape == (0, heads, d)
