"""The operators on a part of a long context as a program uses them: one after the other, through the binding and past it, captured and
replayed, on several streams at once, over caches of other layouts and past 32 bits of offset, and with values that are no finite numbers.
Tolerances as in test_gpu_partial.py."""
import math

import numpy as np
import pytest
import torch

import aitherkvcache_amd as akv
from aitherkvcache_amd.fused_kv_update import fused_kv_update_pair
from tests.test_gpu_chunk import BF, FP, HALF, Batch, Packed, table_of
from tests.test_gpu_chunk_use import binding, slots_of
from tests.test_gpu_partial import assert_attention, index_of, kept_reference, selection, some_columns, sparse_reference, vectors, weights_reference

pytestmark = pytest.mark.gpu


def inputs(gen, b, dtype, dev, heads, kvh, d):
    return [vectors(gen, dtype, dev, *s) for s in ((b.tokens, heads, d), (b.blocks, b.block, kvh, d), (b.blocks, b.block, kvh, d))]


@pytest.mark.parametrize("dtype,index", [(FP, torch.int32), (BF, torch.int64)])
def test_binding_and_long_way_give_the_same(dev, monkeypatch, dtype, index):
    b = Batch([(3, 70), (1, 900), (40, 190)], 16, dev, 1, index)
    q, k, v = inputs(torch.Generator().manual_seed(1), b, dtype, dev, 8, 2, 128)
    got = []
    for take in (True, False):
        with binding(monkeypatch, take) as c:
            ix = akv.BlockIndex(b.blocks, 2, 128, dev)
            assert ix.update(k, b.tables, b.ctx, b.starts) is None
            part = ix.codes.clone()
            assert ix.update(k, b.tables, b.ctx) is None
            sel = ix.select(q, b.tables, b.ctx, b.starts, 16, 6)
            into, out = torch.full_like(sel, 5), torch.full_like(q, 3.0)
            assert ix.select(q, b.tables, b.ctx, b.starts, 16, 6, 2, 1, out=into) is into
            assert akv.paged_sparse_attention(q, k, v, b.tables, b.ctx, b.starts, into, 0.2, out=out) is out
            acc = torch.full((3, 2, b.tables.shape[1] * 16 + 3), 2.0, device=dev)
            assert akv.paged_key_weights(q, k, b.tables, b.ctx, b.starts, accumulated=acc, scale=0.3) is acc
            p = Packed(b, 128, 4, 8, 2, dtype, dev, 41, primary=True)
            packed = p.attn.key_weights(p.q, p.k, p.kn, b.tables, b.ctx, b.starts)
            more = packed.clone()
            assert p.attn.key_weights(p.q, p.k, p.kn, b.tables, b.ctx, b.starts, num_kv_heads=2, accumulated=more) is more
            k2, v2, k3, v3 = k.clone(), v.clone(), torch.cat([k, k]), torch.cat([v, v])
            cuts = [*akv.evict_tokens(packed, b.tables, b.ctx, [k2, v2, p.k, p.kn], 60), *akv.evict_tokens(more, b.tables, b.ctx, (k3, v3), 60, 3, 4, b.tables[:, :4] + b.blocks)]
            got.append([packed, more, k2, v2, k3, v3, *cuts, part, ix.codes, ix.scales, sel, into, out, acc, akv.paged_sparse_attention(q, k, v, b.tables, b.ctx, b.starts, sel),
                        akv.paged_key_weights(q, k, b.tables, b.ctx, b.starts)])
            assert c.taken == (12 if take else 0)
    for x, y in zip(*got):
        assert torch.equal(x, y)


def test_a_prompt_cut_and_decoded(dev):
    """A prompt in two chunks that read selected blocks, cut by the weights of its last tokens, then tokens of a decode step."""
    heads, kv, d, block, keep = 8, 2, 128, 16, 120
    lens = [400, 333, 90]
    b = Batch([(0, n + 40) for n in lens], block, dev, seed=3, pad_cols=0)
    gen = torch.Generator().manual_seed(2)
    table = table_of(600, d, dev)
    kc, vc = (torch.full((b.blocks, block, kv, d), math.nan, dtype=BF, device=dev) for _ in range(2))
    index = akv.BlockIndex(b.blocks, kv, d, dev)

    def step(new, positions):
        """`new` (new, context) a sequence, the tokens' rotary positions: append, take means, select, attend; all against the plain forms."""
        b.lens = new
        b.tokens = sum(n for n, _ in new)
        ctx = torch.tensor([c for _, c in new], dtype=torch.int32, device=dev)
        starts = torch.tensor(np.cumsum([0] + [n for n, _ in new]), dtype=torch.int32, device=dev)
        x = vectors(gen, BF, dev, b.tokens, heads + 2 * kv, d)
        q = akv.rope_append(x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], torch.tensor(positions, device=dev), table, slots_of(b), kc, vc)
        index.update(kc, b.tables, ctx, starts)
        touched = [(i, col) for i, (n, c) in enumerate(new) for col in range((c - n) // block, -(-c // block)) if n]
        for blk, (codes, scales) in index_of(kc, b, touched).items():
            assert torch.equal(index.codes[blk].cpu().float(), codes) and torch.equal(index.scales[blk].cpu(), scales)
        sel = index.select(q, b.tables, ctx, starts, block, 6)
        assert torch.equal(sel.cpu(), selection(b, index, q, kv, 6, 1, 2))
        assert_attention(akv.paged_sparse_attention(q, kc, vc, b.tables, ctx, starts, sel), b, q, kc, vc, sel)
        return q, ctx, starts

    half = [n // 2 + 5 for n in lens]
    step([(n, n) for n in half], [p for n in half for p in range(n)])
    q, ctx, starts = step([(n - m, n) for n, m in zip(lens, half)], [p for n, m in zip(lens, half) for p in range(m, n)])
    # the last 30 tokens say what stays
    rows = torch.cat([torch.arange(30, device=dev) + starts[i + 1] - 30 for i in range(3)])
    ends = torch.tensor([0, 30, 60, 90], dtype=torch.int32, device=dev)
    w = akv.paged_key_weights(q[rows].contiguous(), kc, b.tables, ctx, ends)
    b.lens, b.kvh = [(30, n) for n in lens], kv
    want, _ = weights_reference(b, q[rows], lambda i: b.rows(kc, i), 1 / math.sqrt(d))
    assert ((w.cpu().double() - want).square().sum() / want.square().sum()).sqrt() < 2e-6
    before = [[b.rows(c, i).clone() for i in range(3)] for c in (kc, vc)]
    kept, now, left = akv.evict_tokens(w, b.tables, ctx, [kc, vc], keep, num_sink=4, num_recent=30)
    assert now.tolist() == [min(n, keep) for n in lens]
    b.lens = [(0, min(n, keep)) for n in lens]
    for i, n in enumerate(lens):
        for h in range(kv):
            ref = kept_reference(w[i, h].cpu().numpy(), n, keep, 4, 30)
            assert np.array_equal(kept[i, h, :len(ref)].cpu().numpy(), ref)
            for c, old in zip((kc, vc), before):
                assert torch.equal(b.rows(c, i)[:, h], old[i][torch.from_numpy(ref).to(dev), h])
    index.update(kc, b.tables, now)
    held = now.tolist()
    for t in range(3):
        q, ctx, starts = step([(1, c + t + 1) for c in held], [n + t for n in lens])
        # weights go on being added up at the tokens' new places
        more = left.clone()
        akv.paged_key_weights(q, kc, b.tables, ctx, starts, accumulated=left)
        b.kvh = kv
        want, _ = weights_reference(b, q, lambda i: b.rows(kc, i), 1 / math.sqrt(d))
        assert (left.cpu().double() - more.cpu().double() - want[..., :left.shape[2]]).abs().max() < 1e-5
    akv.evict_tokens(left, b.tables, ctx, [kc, vc], keep)
    assert bool(torch.isfinite(b.rows(kc, 0)[:keep].float()).all())


@pytest.mark.parametrize("bits", [4, 3, 2])
def test_packed_rows_weighed_and_cut(dev, bits):
    """A packed cache: encoded, weighed, cut in place, read again: what attention reads is what was kept."""
    heads, kv, d, keep = 8, 2, 128, 40
    b = Batch([(16, 130), (16, 30)], 16, dev, 4)
    p = Packed(b, d, bits, heads, kv, BF, dev, 51, primary=True)
    gen = torch.Generator().manual_seed(bits)
    x = vectors(gen, BF, dev, 160, 2 * kv, d)
    p.kn.fill_(math.nan), p.vn.fill_(math.nan)
    fused_kv_update_pair(x[:, :kv], x[:, kv:], slots_of(b, [(0, c) for _, c in b.lens]), p.k, p.kn, p.v, p.vn, p.tq.rotation, p.tq.boundaries_inner, bits, block_size=16)
    w = p.attn.key_weights(p.q, p.k, p.kn, b.tables, b.ctx, b.starts)
    assert (w.double().sum(2) - 16 * heads / kv).abs().max() < 1e-3
    before = [[b.rows(c, i).clone() for i in range(2)] for c in (p.k, p.kn, p.v, p.vn)]
    kept, now, _ = akv.evict_tokens(w, b.tables, b.ctx, [p.k, p.kn, p.v, p.vn], keep, 2, 16)
    assert now.tolist() == [40, 30]
    b.lens = [(16, 40), (16, 30)]
    b.ctx = now
    for i, (_, n) in enumerate(b.lens):
        for h in range(kv):
            at = kept[i, h, :n].long()
            for c, old in zip((p.k, p.kn, p.v, p.vn), before):
                assert torch.equal(b.rows(c, i)[:, h], old[i][at, h])
    out, bound = p.reference()
    assert ((p.run().double() - out).abs() <= bound).all()


def whole_layer(b, index, q, k, v, ctx, p, tables_to, acc):
    """Every operator once."""
    index.update(k, b.tables, ctx, b.starts)
    sel = index.select(q, b.tables, ctx, b.starts, b.block, 5)
    out = akv.paged_sparse_attention(q, k, v, b.tables, ctx, b.starts, sel)
    w = akv.paged_key_weights(q, k, b.tables, ctx, b.starts)
    akv.paged_key_weights(q, k, b.tables, ctx, b.starts, accumulated=acc)
    pw = p.attn.key_weights(p.q, p.k, p.kn, b.tables, ctx, b.starts, block_size=b.block)
    kept = akv.evict_tokens(w, b.tables, ctx, [k, v, p.k, p.kn], 50, 3, 7, out_tables=tables_to)
    return (index.codes, index.scales, sel, out, w, acc, pw, *kept)


def spare_tables(b, S, columns, dev):
    """Blocks behind those of the batch."""
    to = torch.arange(b.blocks, b.blocks + S * columns, dtype=torch.int32, device=dev).view(S, columns)
    b.blocks += S * columns
    return to


def test_captured_and_replayed(dev):
    """One graph of all operators; lengths and inputs change between replays, other work runs too."""
    steps = [[(9, 200), (1, 33), (60, 77)], [(9, 209), (1, 500), (60, 60)], [(9, 9), (1, 1), (60, 900)]]
    b = [Batch([(n, 1000) for n, _ in s], 16, dev, 5) for s in steps][0]
    to = spare_tables(b, 3, 4, dev)
    gen = torch.Generator().manual_seed(3)
    p = Packed(b, 128, 4, 8, 2, BF, dev, 60)
    p.kn.copy_(p.kn.nan_to_num(1.0))
    q, k, v = inputs(gen, b, BF, dev, 8, 2, 128)
    ctx = torch.ones_like(b.ctx)
    acc = torch.zeros(3, 2, b.tables.shape[1] * 16, device=dev)
    index, other = akv.BlockIndex(b.blocks, 2, 128, dev), akv.BlockIndex(b.blocks, 2, 128, dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        whole_layer(b, index, q, k, v, ctx, p, to, acc)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = whole_layer(b, index, q, k, v, ctx, p, to, acc)
    index.codes.zero_(), index.scales.zero_(), acc.zero_()
    caches = (k, v, p.k, p.kn)
    for r in range(6):
        ctx.copy_(torch.tensor([c for _, c in steps[r % 3]], device=dev))
        q.copy_(vectors(gen, BF, dev, *q.shape))
        k.copy_(vectors(gen, BF, dev, *k.shape))
        other.codes.copy_(index.codes), other.scales.copy_(index.scales)
        acc2, old = acc.clone(), [c.clone() for c in caches]
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        after = [c.clone() for c in caches]
        for c, o in zip(caches, old):
            c.copy_(o)
        want = whole_layer(b, other, q, k, v, ctx, p, to, acc2)
        for i, (x, y) in enumerate(zip(kept, want)):
            assert torch.equal(x, y), (r, i)
        for c, a in zip(caches, after):
            assert torch.equal(c.view(torch.uint8), a.view(torch.uint8))


def test_two_graphs_and_eager_work_at_once(dev):
    """Two captured graphs and eager calls on streams of their own: nobody's scratch is another's."""
    b = Batch([(60, 3000), (2, 5000), (1, 8000)], 16, dev, 6)
    to = [spare_tables(b, 3, 4, dev) for _ in range(3)]
    gen = torch.Generator().manual_seed(4)
    ps = [Packed(b, 128, 4, 16, 4, BF, dev, 80 + i) for i in range(3)]
    dense = [inputs(gen, b, BF, dev, 16, 4, 128) for _ in range(3)]
    index = [akv.BlockIndex(b.blocks, 4, 128, dev) for _ in range(3)]
    acc = [torch.zeros(3, 4, b.tables.shape[1] * 16, device=dev) for _ in range(3)]

    def layer(i):
        acc[i].zero_()
        return [t.clone() for t in whole_layer(b, index[i], *dense[i], b.ctx, ps[i], to[i], acc[i])]

    want = [layer(i) for i in range(3)]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[i]):
            outs.append(layer(i))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(4):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        with torch.cuda.stream(streams[2]):
            eager = [layer(2) for _ in range(2)]
        torch.cuda.synchronize()
        for got, w in [(outs[0], want[0]), (outs[1], want[1])] + [(e, want[2]) for e in eager]:
            for i, (x, y) in enumerate(zip(got, w)):
                assert torch.equal(x, y), i


# ---- values that are no finite numbers ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d,heads,kvh,block", [(128, 8, 2, 16), (64, 28, 4, 32), (256, 4, 4, 7), (64, 1, 1, 16)])
def test_odd_values_reach_only_tokens_that_see_them(dev, d, heads, kvh, block, dtype):
    """NaN and infinities among the values of keys that some tokens of a tile see and others do not, by selection and by position."""
    gen = torch.Generator().manual_seed(d)
    b = Batch([(50, 400), (1, 90), (33, 33), (9, 700)], block, dev, seed=7)
    q, k, v = inputs(gen, b, dtype, dev, heads, kvh, d)
    sel = some_columns(gen, b, kvh, 6)
    clean = v.clone()
    odd = [(0, 380, math.nan), (0, 100, math.inf), (2, 20, -math.inf), (3, 650, math.nan), (3, 695, math.inf), (0, 399, math.nan)]
    for i, pos, value in odd:
        v[b.host[i, pos // block], pos % block, :, 3] = value
    k[b.host[0, 200 // block], 200 % block, 0, 5] = math.nan
    sel = sel.to(dev)
    got = akv.paged_sparse_attention(q, k, v, b.tables, b.ctx, b.starts, sel).cpu().double()
    want, size, total = sparse_reference(b, q, k, v, sel, 1 / math.sqrt(d))
    fine = torch.isfinite(want)
    # where nothing odd is seen the result is that over clean values (an odd value is one coordinate of a row: rows are counted)
    row_fine = fine.all(-1)
    assert 0 < row_fine.sum() < row_fine.numel() and (torch.isfinite(got) == fine).all()
    u = HALF[dtype]
    bound = (2 * u + 2.0 ** -14) * size + 2.0 ** -25 * total + 2.0 ** -25
    assert ((got - want).abs() <= bound)[row_fine].all()
    plain = akv.paged_sparse_attention(q, k.nan_to_num(0.0), clean, b.tables, b.ctx, b.starts, sel).cpu().double()
    assert ((plain - want).abs() <= bound)[row_fine].all()


def test_odd_keys(dev):
    """A key that is no finite number, in a block that some tokens of a tile select: the others do not meet it."""
    b = Batch([(32, 300)], 16, dev, seed=8)
    gen = torch.Generator().manual_seed(5)
    q, k, v = inputs(gen, b, BF, dev, 4, 1, 128)
    for pos, value in ((40, math.inf), (70, -math.inf), (100, math.nan)):
        k[b.host[0, pos // 16], pos % 16] = value
    sel = torch.tensor([0, 5, 9, 16, 17, 18], dtype=torch.int32).expand(32, 1, -1).clone()
    sel[::4, :, 1], sel[1::8, :, 2], sel[3::8, :, 0] = 2, 4, 6
    got = akv.paged_sparse_attention(q, k, v, b.tables, b.ctx, b.starts, sel.to(dev)).cpu().double()
    want, size, total = sparse_reference(b, q, k, v, sel, 1 / math.sqrt(128))
    fine = torch.isfinite(want).all(-1)
    assert 0 < fine.sum() < fine.numel() and torch.isfinite(got[fine]).all()
    assert ((got - want).abs() <= (2 * HALF[BF] + 2.0 ** -14) * size + 1e-30)[fine].all()


# ---- sizes, layouts, offsets ----------------------------------------------------------------------------------------------------
def test_nothing_to_do(dev):
    """No token, no sequence, no context, tables of no column, no block: zeros, -1 or nothing."""
    b = Batch([(0, 0), (0, 40)], 16, dev, seed=9)
    gen = torch.Generator().manual_seed(6)
    k, v = (vectors(gen, BF, dev, b.blocks, 16, 2, 64) for _ in range(2))
    index = akv.BlockIndex(b.blocks, 2, 64, dev)
    none = torch.empty(0, 4, 64, dtype=BF, device=dev)
    index.update(k, b.tables, b.ctx, b.starts)
    assert (index.codes == 0).all()
    sel = index.select(none, b.tables, b.ctx, b.starts, 16, 4)
    assert sel.shape == (0, 2, 4) and akv.paged_sparse_attention(none, k, v, b.tables, b.ctx, b.starts, sel).shape == none.shape
    assert (akv.paged_key_weights(none, k, b.tables, b.ctx, b.starts) == 0).all()
    # no sequence: every row is of none
    q = vectors(gen, BF, dev, 3, 4, 64)
    nobody = dict(block_tables=b.tables[:0], context_lens=b.ctx[:0], query_start_loc=b.starts[:1])
    sel = index.select(q, block_size=16, num_selected=4, **nobody)
    assert (sel == -1).all() and (akv.paged_sparse_attention(q, k, v, selected=sel, **nobody) == 0).all()
    assert akv.paged_key_weights(q, k, **nobody).shape == (0, 2, b.tables.shape[1] * 16)
    kept, now, left = akv.evict_tokens(torch.empty(0, 2, b.tables.shape[1] * 16, device=dev), b.tables[:0], b.ctx[:0], [k], 5, 0, 0)
    assert kept.shape == (0, 2, 5) and now.shape == (0,) and left.shape == (0, 2, b.tables.shape[1] * 16)
    # tokens before the first key, and tables without a column
    ctx, starts = torch.tensor([1], device=dev), torch.tensor([0, 3], device=dev)
    sel = index.select(q, b.tables[1:], ctx, starts, 16, 4)
    assert sel[2, 0].tolist() == [0, -1, -1, -1] and (sel[:2] == -1).all()
    out = akv.paged_sparse_attention(q, k, v, b.tables[1:], ctx, starts, sel)
    assert (out[:2] == 0).all() and torch.equal(out[2], v[b.host[1, 0], 0].repeat_interleave(2, 0))
    w = akv.paged_key_weights(q, k, b.tables[1:], ctx, starts)
    assert (w[0, :, 0] == 2).all() and (w[0, :, 1:] == 0).all()
    assert (akv.paged_sparse_attention(q, k, v, b.tables[1:, :0], ctx, starts, sel) == 0).all()
    assert (akv.paged_sparse_attention(q, k, v, b.tables[1:], ctx, starts, sel[..., :0]) == 0).all()
    assert (index.select(q, b.tables[1:, :0], ctx, starts, 16, 4) == -1).all() and akv.paged_key_weights(q, k, b.tables[1:, :0], ctx, starts).shape == (1, 2, 0)


def test_other_layouts(dev):
    """Queries out of a fused product, caches with heads before positions or side by side, selections as a view: the same as plain ones."""
    b = Batch([(5, 300), (40, 90), (1, 1000)], 16, dev, seed=10, index=torch.int64)
    gen = torch.Generator().manual_seed(7)
    q, k, v = inputs(gen, b, FP, dev, 12, 4, 64)
    index, other = akv.BlockIndex(b.blocks, 4, 64, dev), akv.BlockIndex(b.blocks, 4, 64, dev)
    index.update(k, b.tables, b.ctx, b.starts)
    sel = index.select(q, b.tables, b.ctx, b.starts, 16, 6)
    want = [akv.paged_sparse_attention(q, k, v, b.tables, b.ctx, b.starts, sel), akv.paged_key_weights(q, k, b.tables, b.ctx, b.starts)]
    fused = torch.randn(b.tokens, 20, 64, device=dev).to(FP)
    fused[:, 3:15] = q
    both = torch.full((b.blocks, 2, 4, 16, 64), math.nan, dtype=FP, device=dev)
    both[:, 0], both[:, 1] = k.transpose(1, 2), v.transpose(1, 2)
    k2, v2, q2 = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2), fused[:, 3:15]
    tables = torch.full((3, 2 * b.tables.shape[1]), -3, device=dev)
    tables[:, ::2] = b.tables
    tables = tables[:, ::2]
    starts, ctx = b.starts.repeat_interleave(2)[::2], b.ctx.int()
    other.update(k2, tables, ctx, starts)
    assert torch.equal(other.codes, index.codes) and torch.equal(other.scales, index.scales)
    assert torch.equal(other.select(q2, tables, ctx, starts, 16, 6), sel)
    wide = torch.full((4, b.tokens, 9), -1, dtype=torch.int32, device=dev)
    wide[..., :6] = sel.transpose(0, 1)
    into = torch.zeros(b.tokens, 30, 64, dtype=FP, device=dev)
    for s in (wide.transpose(0, 1), sel.flip(2).repeat(1, 1, 2)[..., ::2], torch.cat([sel, sel], 2)):
        if s.shape[2] == 6:
            s = torch.cat([s, sel], 2)
        akv.paged_sparse_attention(q2, k2, v2, tables, ctx, starts, s, out=into[:, 9:21])
        assert torch.equal(into[:, 9:21], want[0]) and (into[:, :9] == 0).all() and (into[:, 21:] == 0).all()
    acc = torch.zeros(4, 3, want[1].shape[2], device=dev).transpose(0, 1)
    akv.paged_key_weights(q2, k2, tables, ctx, starts, accumulated=acc)
    assert torch.equal(acc, want[1])
    # one position a block, wherever the strides of a dimension of one entry point
    one = Batch([(4, 50)], 1, dev, seed=11)
    q, k, v = inputs(gen, one, FP, dev, 4, 2, 64)
    sel = torch.arange(50, dtype=torch.int32, device=dev).expand(4, 2, -1)
    a = akv.paged_sparse_attention(q, k, v, one.tables, one.ctx, one.starts, sel)
    strange = [t.as_strided(t.shape, (t.stride(0), 1 << 33, t.stride(2), 1)) for t in (k, v)]
    assert torch.equal(a, akv.paged_sparse_attention(q, *strange, one.tables, one.ctx, one.starts, sel))


def test_offsets_past_32_bits(dev):
    """The same rows in blocks at the end of caches of more than 4 GB: the same results."""
    b = Batch([(20, 500), (1, 1500)], 16, dev, seed=13, spare=0)
    gen = torch.Generator().manual_seed(9)
    q, k, v = inputs(gen, b, BF, dev, 16, 8, 128)
    far = (5 << 30) // (16 * 8 * 128 * 2)
    k2, v2 = (torch.empty(far + b.blocks, 16, 8, 128, dtype=BF, device=dev) for _ in range(2))
    k2[far:], v2[far:] = k, v
    got = []
    for keys, values, shift in ((k, v, 0), (k2, v2, far)):
        tables = b.tables + shift
        index = akv.BlockIndex(keys.shape[0], 8, 128, dev)
        index.update(keys, tables, b.ctx)
        sel = index.select(q, tables, b.ctx, b.starts, 16, 7)
        w = akv.paged_key_weights(q, keys, tables, b.ctx, b.starts)
        out = akv.paged_sparse_attention(q, keys, values, tables, b.ctx, b.starts, sel)
        kept, now, _ = akv.evict_tokens(w, tables, b.ctx, [keys, values], 300)
        got.append((index.codes[shift:], index.scales[shift:], sel, w, out, kept, now, keys[shift:], values[shift:]))
    for i, (x, y) in enumerate(zip(*got)):
        assert torch.equal(x, y), i


@pytest.mark.parametrize("packed", [False, True])
def test_weights_in_slabs(dev, packed):
    """Tables so wide that scratch holds some of the tokens at a time: of few rows a head, and of many."""
    for lens, heads, kvh, columns in (([(30, 200), (40, 90), (3, 3), (50, 700)], 32, 32, 8500), ([(1500, 1600), (20, 900)], 32, 8, 17000)):
        b = Batch(lens, 16, dev, seed=14, pad_cols=columns)
        gen = torch.Generator().manual_seed(10)
        size = akv._lib.lib().akv_packed_key_weights_workspace_bytes if packed else akv._lib.lib().akv_key_weights_workspace_bytes
        length = b.tables.shape[1] * 16
        if heads == kvh:
            # (more tokens of more sequences need no more scratch: it is held to a slab)
            assert size(b.tokens, len(lens), heads, kvh, 64, length) == size(4 * b.tokens, 4 * len(lens), heads, kvh, 64, length)
        b.kvh = kvh
        if packed:
            p = Packed(b, 64, 4, heads, kvh, BF, dev, 90)
            got = p.attn.key_weights(p.q, p.k, p.kn, b.tables, b.ctx, b.starts)
            short = p.attn.key_weights(p.q, p.k, p.kn, b.tables[:, :-columns].contiguous(), b.ctx, b.starts)
        else:
            q, k, _ = inputs(gen, b, BF, dev, heads, kvh, 64)
            got = akv.paged_key_weights(q, k, b.tables, b.ctx, b.starts)
            short = akv.paged_key_weights(q, k, b.tables[:, :-columns].contiguous(), b.ctx, b.starts)
        assert (got[..., short.shape[2]:] == 0).all()
        off = (got[..., :short.shape[2]] - short).double()
        assert (off.square().sum() / short.double().square().sum()).sqrt() < 1e-6 and (off.abs() <= 1e-5 * short + 1e-12).all()
        rows = torch.tensor([sum(c - n + j >= 0 for j in range(n)) * heads // kvh for n, c in lens], dtype=torch.float64)
        assert (got.double().sum(2).cpu() - rows[:, None]).abs().max() <= 2.0 ** -17 * rows.max()


def test_shared_blocks_are_cut_to_blocks_of_their_own(dev):
    """Two sequences with the same beginning (and one sequence twice): each gets its own rows, the shared ones stay."""
    b = Batch([(0, 160), (0, 100)], 16, dev, seed=15, pad_cols=0)
    tables = b.tables.clone()
    tables[1, :3] = tables[0, :3]
    tables = torch.cat([tables, tables[:1]])
    ctx = torch.tensor([160, 100, 160], dtype=torch.int32, device=dev)
    to = spare_tables(b, 3, 3, dev)
    cache = torch.arange(b.blocks * 16 * 2, device=dev).view(b.blocks, 16, 2).clone()
    before = cache.clone()
    w = torch.rand(3, 2, 160, device=dev)
    kept, now, _ = akv.evict_tokens(w, tables, ctx, [cache], 40, 1, 5, out_tables=to)
    for i in range(3):
        for h in range(2):
            at = kept[i, h].long()
            want = before[tables[i].long()[at // 16], at % 16, h]
            assert torch.equal(cache[to[i].long()].flatten(0, 1)[:40, h], want)
            assert torch.equal(kept[i, h].cpu(), torch.from_numpy(kept_reference(w[i, h].cpu().numpy(), int(ctx[i]), 40, 1, 5)).int())
    assert torch.equal(cache[:int(to.min())], before[:int(to.min())])


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d,heads,kvh,block", [(128, 32, 8, 16), (64, 6, 1, 32), (256, 8, 2, 7), (128, 64, 1, 16), (64, 16, 16, 1)])
def test_few_tokens(dev, d, heads, kvh, block, dtype):
    """About one token a sequence, so that workgroups share the keys of a token: with gaps, two tokens at once, odd values, rows of no sequence."""
    gen = torch.Generator().manual_seed(d + heads)
    b = Batch([(1, 700), (0, 30), (1, 5), (2, 900), (0, 0), (1, 64), (0, 3), (1, 2000), (1, 1)], block, dev, seed=16)
    q, k, v = inputs(gen, b, dtype, dev, heads, kvh, d)
    b.unused(math.nan, k, v)
    sel = some_columns(gen, b, kvh, 64)
    sel[3] = -1
    sel = sel.to(dev)
    got = akv.paged_sparse_attention(q, k, v, b.tables, b.ctx, b.starts, sel)
    assert_attention(got, b, q, k, v, sel)
    for _ in range(3):
        assert torch.equal(got, akv.paged_sparse_attention(q, k, v, b.tables, b.ctx, b.starts, sel))
    into = torch.full_like(q, 3.0)
    akv.paged_sparse_attention(q, k, v, b.tables[2:6], b.ctx[2:6], b.starts[2:7], sel, out=into)
    few = akv.paged_sparse_attention(q, k, v, b.tables[2:6], b.ctx[2:6], b.starts[2:7], sel)
    assert (into[:1] == 3).all() and (into[5:] == 3).all() and (few[:1] == 0).all() and (few[5:] == 0).all() and torch.equal(few[1:5], into[1:5])
    assert_attention(torch.cat([got[:1], few[1:5], got[5:]]), b, q, k, v, sel)
    # the first of two tokens does not see what the second does
    v[b.host[3, 899 // block], 899 % block] = math.inf
    sel[2:4, :, 0] = 899 // block
    got = akv.paged_sparse_attention(q, k, v, b.tables, b.ctx, b.starts, sel)
    assert torch.isfinite(got[2]).all() and not torch.isfinite(got[3]).any()
    v[b.host[3, 899 // block], 899 % block] = 0
    sel[3] = -1
    got[3] = 0
    assert_attention(got, b, q, k, v, sel)


def test_few_tokens_captured(dev):
    """A decode step in a graph, with the second launch that joins what workgroups share; lengths and selections change between replays."""
    b = Batch([(1, 1500), (1, 900), (1, 700)], 16, dev, seed=17)
    gen = torch.Generator().manual_seed(11)
    q, k, v = inputs(gen, b, BF, dev, 16, 4, 128)
    index = akv.BlockIndex(b.blocks, 4, 128, dev)
    index.update(k, b.tables, b.ctx)
    ctx = b.ctx.clone()

    def step():
        sel = index.select(q, b.tables, ctx, b.starts, 16, 80)
        return sel, akv.paged_sparse_attention(q, k, v, b.tables, ctx, b.starts, sel)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for lens in ((1500, 900, 700), (17, 1, 0), (1400, 16, 699), (0, 900, 300)):
        ctx.copy_(torch.tensor(lens, device=dev))
        q.copy_(vectors(gen, BF, dev, *q.shape))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        for x, y in zip(kept, step()):
            assert torch.equal(x, y)
        b.lens = [(1, c) for c in lens]
        assert_attention(kept[1], b, q, k, v, kept[0])


def test_starts_that_go_back_and_lengths_out_of_range(dev):
    """Starts that go back, lengths below zero or past the tables: rows of such sequences are undefined, the others' are right, and nothing else is touched."""
    b = Batch([(4, 100), (6, 80), (5, 300)], 16, dev, seed=18)
    gen = torch.Generator().manual_seed(12)
    q, k, v = inputs(gen, b, BF, dev, 8, 2, 64)
    index = akv.BlockIndex(b.blocks, 2, 64, dev)
    index.update(k, b.tables, b.ctx)
    sel = index.select(q, b.tables, b.ctx, b.starts, 16, 5)
    want = akv.paged_sparse_attention(q, k, v, b.tables, b.ctx, b.starts, sel)
    w = akv.paged_key_weights(q, k, b.tables, b.ctx, b.starts)
    for starts in ([0, 4, 4, 0], [9, 4, 10, 15], [0, -5, 10, 99], [7, 3, 2, 1]):
        s = torch.tensor(starts, dtype=torch.int32, device=dev)
        index.select(q, b.tables, b.ctx, s, 16, 5)
        akv.paged_sparse_attention(q, k, v, b.tables, b.ctx, s, sel)
        akv.paged_key_weights(q, k, b.tables, b.ctx, s)
        index.update(k, b.tables, b.ctx, s)
    ctx = b.ctx.clone()
    ctx[0], ctx[2] = -7, 1 << 30
    tables = b.tables.clamp(0, b.blocks - 1)
    s2 = index.select(q, tables, ctx, b.starts, 16, 5)
    assert (s2[:4] == -1).all() and torch.equal(s2[4:10], sel[4:10])
    out = akv.paged_sparse_attention(q, k, v, tables, ctx, b.starts, s2)
    assert (out[:4] == 0).all() and torch.equal(out[4:10], want[4:10])
    w2 = akv.paged_key_weights(q, k, tables, ctx, b.starts)
    assert (w2[0] == 0).all() and torch.equal(w2[1], w[1])
    kept, now, _ = akv.evict_tokens(w, tables[:2], ctx[:2], [k, v], 40, 2, 8)
    assert now.tolist() == [0, 40] and (kept[0] == -1).all()
