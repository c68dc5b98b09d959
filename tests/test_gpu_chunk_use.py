"""The operators on a chunk of new tokens as a program uses them: one after the other, through the binding and past it, captured and
replayed, on two streams at once, with many sequences, with offsets past 32 bits.  Tolerances as in test_gpu_chunk.py."""
import contextlib
import math

import pytest
import torch

import aitherkvcache_amd as akv
from aitherkvcache_amd import _lib
from aitherkvcache_amd.fused_kv_update import fused_kv_update_pair
from tests.test_gpu_chunk import BF, FP, Batch, Packed, check, check_rope, dense_reference, rope_reference, table_of, vectors

pytestmark = pytest.mark.gpu


class Counting:
    """The binding with a count of the calls it took; take=False: it takes none."""

    def __init__(self, real, take):
        self.real, self.take, self.taken = real, take, 0

    def __getattr__(self, name):
        def call(*args):
            res = getattr(self.real, name)(*args) if self.take else None
            self.taken += res is not None
            return res
        return call


@contextlib.contextmanager
def binding(monkeypatch, take):
    c = Counting(_lib.calls(), take)
    with monkeypatch.context() as m:
        m.setattr(_lib, "_calls", c)
        yield c


def slots_of(b, which=None):
    """Slots of every sequence's newest tokens (or of `which` = (first, last) positions), in the order of the queries."""
    out = []
    for i, (n, c) in enumerate(b.lens):
        lo, hi = (c - n, c) if which is None else which[i]
        out += [int(b.host[i, p // b.block]) * b.block + p % b.block for p in range(lo, hi)]
    return torch.tensor(out, device=b.tables.device)


# ---- the binding and the long way -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,index", [(FP, torch.int32), (BF, torch.int64)])
@pytest.mark.parametrize("own_out", [False, True])
def test_binding_and_long_way_give_the_same(dev, monkeypatch, dtype, index, own_out):
    b = Batch([(3, 70), (1, 200), (40, 90)], 16, dev, 1, index)
    p = Packed(b, 128, 4, 8, 2, dtype, dev, 41, primary=True)
    kc, vc = (vectors(42 + i, dev, dtype, b.blocks, 16, 2, 128) for i in range(2))
    fused = vectors(44, dev, dtype, b.tokens, 12, 128)
    table, slots = table_of(256, 96, dev), slots_of(b).to(index)
    pos = torch.arange(b.tokens, device=dev, dtype=index)
    three = torch.stack([pos, pos // 2, pos // 3])
    got = []
    for take in (True, False):
        with binding(monkeypatch, take) as c:
            k2, v2 = kc.clone(), vc.clone()
            new = lambda: torch.full_like(p.q, 3.0) if own_out else None
            res = [akv.rope_append(fused[:, :8], fused[:, 8:10], fused[:, 10:], pos, table, slots, k2, v2, query_out=new())]
            res += [akv.rope_append(fused[:, :8], fused[:, 8:10], fused[:, 10:], three, table, slots, k2, v2, (24, 12, 12), True, new())]
            assert akv.rope_append(None, fused[:, 8:10], fused[:, 10:], None, None, slots, k2, v2) is None
            res += [k2.clone(), v2.clone(), akv.paged_chunk_attention(p.q, k2, v2, b.tables, b.ctx, b.starts, out=new()),
                    akv.paged_chunk_attention(p.q, k2, v2, b.tables, b.ctx, b.starts, 0.05, 33, max_query_len=40, out=new()),
                    p.run(out=new()), p.run(max_query_len=40, out=new())]
            assert c.taken == (7 if take else 0)
            got.append(res)
    for x, y in zip(*got):
        assert torch.equal(x, y)


def test_binding_refuses_what_the_long_way_refuses(dev):
    b = Batch([(3, 70)], 16, dev, 2)
    q = vectors(45, dev, FP, 3, 8, 128)
    kc = vectors(46, dev, FP, b.blocks, 16, 2, 128)
    ok = dict(query=q, key_cache=kc, value_cache=kc, block_tables=b.tables, context_lens=b.ctx, query_start_loc=b.starts)
    assert akv.paged_chunk_attention(**ok).shape == q.shape
    for error, change in ((ValueError, dict(window=-1)), (ValueError, dict(scale=0.0)), (ValueError, dict(scale=math.nan)), (ValueError, dict(query=q[:, :7])),
                          (ValueError, dict(value_cache=kc[:, :8])), (ValueError, dict(key_cache=kc.bfloat16())), (NotImplementedError, dict(query=q.float())),
                          (ValueError, dict(out=q.float())), (ValueError, dict(block_tables=b.tables[:0])), (ValueError, dict(context_lens=b.ctx[:0])),
                          (NotImplementedError, dict(key_cache=kc.flatten()[1:1 + 32 * 256].view(2, 16, 2, 128), value_cache=kc[:2]))):
        with pytest.raises(error):
            akv.paged_chunk_attention(**{**ok, **change})
    slots = slots_of(b)
    table, pos = table_of(64, 96, dev), torch.arange(3, device=dev)
    good = dict(query=q, key=q[:, :2], value=q[:, 2:4], positions=pos, cos_sin=table, slot_mapping=slots, key_cache=kc.clone(), value_cache=kc.clone())
    assert akv.rope_append(**good).shape == q.shape
    for error, change in ((ValueError, dict(key=q[:, :3])), (ValueError, dict(value=q[:, 2:4].bfloat16())), (ValueError, dict(positions=pos[:2])), (ValueError, dict(positions=None)),
                          (ValueError, dict(slot_mapping=slots[:2])), (ValueError, dict(cos_sin=table.half())), (ValueError, dict(sections=(24, 24))), (ValueError, dict(sections=(47,), positions=pos[None])),
                          (ValueError, dict(value_cache=kc[:, :8]))):
        with pytest.raises(error):
            akv.rope_append(**{**good, **change})


# ---- together ----------------------------------------------------------------------------------------------------------------

def test_a_prompt_in_chunks_over_the_plain_cache(dev):
    """Append and attention of two chunks, one after the other, are those of the prompt at once."""
    lens = [(90, 90), (33, 33), (200, 200)]
    heads, kv, d = 8, 2, 128
    whole = Batch(lens, 16, dev, 3)
    fused = vectors(50, dev, BF, whole.tokens, heads + 2 * kv, d)
    table = table_of(256, d, dev)
    cuts = [(37, 37), (1, 1), (64, 64)]
    rows, at = [], 0
    for n, _ in lens:
        rows.append(range(at, at + n))
        at += n
    kc, vc = (torch.full((whole.blocks, 16, kv, d), math.nan, dtype=BF, device=dev) for _ in range(2))
    got = torch.empty(whole.tokens, heads, d, dtype=BF, device=dev)
    turned = torch.empty_like(got)
    for part in range(2):
        span = [(0, cuts[i][0]) if part == 0 else (cuts[i][0], lens[i][0]) for i in range(3)]
        pick = torch.tensor([rows[i][p] for i in range(3) for p in range(*span[i])], device=dev)
        pos = torch.tensor([p for s in span for p in range(*s)], device=dev)
        x = fused[pick]
        q = akv.rope_append(x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], pos, table, slots_of(whole, span), kc, vc)
        ctx = torch.tensor([s[1] for s in span], device=dev)
        starts = torch.tensor([0] + [sum(s[1] - s[0] for s in span[:i + 1]) for i in range(3)], device=dev)
        got[pick], turned[pick] = akv.paged_chunk_attention(q, kc, vc, whole.tables, ctx, starts), q
    pos = torch.cat([torch.arange(n, device=dev) for n, _ in lens])
    want_q, q_bound = rope_reference(fused[:, :heads], pos[None], table, [d // 2], False)
    check_rope(turned, want_q, q_bound)
    check(got, *dense_reference(whole, turned, kc, vc, 1 / math.sqrt(d), 0))


@pytest.mark.parametrize("bits", [4, 3, 2])
def test_encode_then_chunk_then_one_token(dev, bits):
    """Keys and values encoded into the packed cache, a chunk over them, then a token of forward(): one cache, one codebook."""
    heads, kv, d = 8, 2, 128
    b = Batch([(40, 70), (5, 20)], 16, dev, 4)
    p = Packed(b, d, bits, heads, kv, BF, dev, 51)
    all_slots = slots_of(b, [(0, c) for _, c in b.lens])
    x = vectors(52, dev, BF, len(all_slots), 2 * kv, d)
    p.kn.fill_(math.nan), p.vn.fill_(math.nan)
    fused_kv_update_pair(x[:, :kv], x[:, kv:], all_slots, p.k, p.kn, p.v, p.vn, p.tq.rotation, p.tq.boundaries_inner, bits, block_size=16)
    out, bound = p.reference()
    got = p.run()
    check(got, out, bound)
    last = torch.tensor([39, 44], device=dev)
    want = p.attn.forward(p.q[last].contiguous(), p.k, p.kn, p.v, p.vn, b.tables, b.ctx, block_size=16)
    assert bool(((got[last].double() - want.double()).abs() <= 2 * bound[last]).all())


# ---- captured and replayed ---------------------------------------------------------------------------------------------------

def test_captured_and_replayed(dev):
    """One graph of append, plain and packed attention; lengths, positions and inputs change between replays, other work runs too."""
    heads, kv, d, block = 8, 2, 128, 16
    steps = [[(9, 200), (1, 33), (60, 77)], [(9, 209), (1, 500), (60, 60)], [(9, 9), (1, 1), (60, 900)]]
    batches = [Batch([(n, 1000) for n, _ in s], block, dev, 5) for s in steps]        # (one pool: the same tables)
    b = batches[0]
    p = Packed(b, d, 4, heads, kv, BF, dev, 60)
    p.kn.copy_(p.kn.nan_to_num(1.0)), p.vn.copy_(p.vn.nan_to_num(1.0))
    table = table_of(1024, d, dev)
    kc, vc = (vectors(61 + i, dev, BF, b.blocks, block, kv, d) for i in range(2))
    x, ctx = torch.empty(b.tokens, heads + 2 * kv, d, dtype=BF, device=dev), torch.ones_like(b.ctx)
    pos, slots = torch.zeros(b.tokens, dtype=torch.int64, device=dev), torch.full((b.tokens,), -1, device=dev)

    def layer(k, v):
        q = akv.rope_append(x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], pos, table, slots, k, v)
        return (q, akv.paged_chunk_attention(q, k, v, b.tables, ctx, b.starts), akv.paged_chunk_attention(q, k, v, b.tables, ctx, b.starts, window=50, max_query_len=60),
                p.attn.forward_chunk(q, p.k, p.kn, p.v, p.vn, b.tables, ctx, b.starts, block_size=block))

    x.copy_(vectors(70, dev, BF, *x.shape))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(kc.clone(), vc.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(kc, vc)
    for r in range(5):
        s = steps[r % 3]
        x.copy_(vectors(71 + r, dev, BF, *x.shape))
        ctx.copy_(torch.tensor([c for _, c in s], device=dev))
        b.lens = s
        pos.copy_(torch.cat([torch.arange(c - n, c, device=dev) for n, c in s]))
        slots.copy_(slots_of(b))
        k2, v2 = kc.clone(), vc.clone()
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        for y, z in zip(kept, layer(k2, v2)):
            assert torch.equal(y, z), r
        assert torch.equal(k2, kc) and torch.equal(v2, vc)
        check(kept[1], *dense_reference(b, kept[0], kc, vc, 1 / math.sqrt(d), 0))


def test_two_graphs_and_eager_work_at_once(dev):
    """Two captured graphs and eager calls of the same operators on streams of their own: nobody's scratch is another's."""
    b = Batch([(60, 3000), (2, 5000), (1, 8000)], 16, dev, 6)
    ps = [Packed(b, 128, 4, 16, 4, BF, dev, 80 + i) for i in range(3)]
    dense = [[vectors(90 + 3 * i + j, dev, BF, b.blocks, 16, 4, 128) for j in range(2)] for i in range(3)]

    def layer(i):
        return ps[i].run(), akv.paged_chunk_attention(ps[i].q, *dense[i], b.tables, b.ctx, b.starts)

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
            assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])


# ---- sizes -----------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("seqs", [255, 256, 257, 600])
def test_many_sequences(dev, seqs):
    """More sequences than lengths held at a time, with and without tokens, of both classes."""
    lens = [((0, 1, 3, 1)[i % 4] if i % 97 else 40, 20 + i % 90 + 40 * (i % 97 == 0)) for i in range(seqs)]
    b = Batch(lens, 16, dev, 7)
    q, kc, vc = (vectors(100 + i, dev, FP, *s) for i, s in enumerate(((b.tokens, 4, 64), (b.blocks, 16, 2, 64), (b.blocks, 16, 2, 64))))
    check(akv.paged_chunk_attention(q, kc, vc, b.tables, b.ctx, b.starts), *dense_reference(b, q, kc, vc, 1 / 8, 0))
    p = Packed(b, 64, 4, 4, 2, FP, dev, 101)
    check(p.run(), *p.reference())


@pytest.mark.parametrize("lens", [[(2, 60)], [(80, 90)]], ids=["few", "many"])
@pytest.mark.parametrize("where", ["block", "place"])
def test_offsets_past_32_bits(dev, lens, where):
    """Caches of more than 2^32 elements from the first row to the last: the stride of a block or of a place in it."""
    b = Batch(lens, 32, dev, 8, spare=0)
    shape, n = (b.blocks, 32, 2, 64), b.blocks * 32 - 1
    big = (3 << 30) // (b.blocks - 1) * 2 // 8 * 8 if where == "block" else (5 << 30) // n // 8 * 8
    strides = (big, 128, 64, 1) if where == "block" else (32 * big, big, 64, 1)
    span = sum((s - 1) * t for s, t in zip(shape, strides)) + 1
    assert span > 1 << 32
    q = vectors(110, dev, FP, b.tokens, 4, 64)
    raw = torch.empty(span, dtype=FP, device=dev)
    kc = raw.as_strided(shape, strides)
    kc.copy_(vectors(111, dev, FP, *shape))
    small = kc.contiguous()
    check(akv.paged_chunk_attention(q, kc, kc, b.tables, b.ctx, b.starts), *dense_reference(b, q, small, small, 1 / 8, 0))
    slots = slots_of(b)
    x = vectors(112, dev, FP, b.tokens, 2, 64)
    akv.rope_append(None, x, x, None, None, slots, kc, kc)
    assert torch.equal(kc.flatten(0, 1)[slots] if where == "place" else torch.stack([kc[int(s) // 32, int(s) % 32] for s in slots]), x)
    p = Packed(b, 64, 4, 4, 2, FP, dev, 113)
    rows = raw.view(torch.uint8).as_strided((*shape[:3], 32), strides)
    rows.copy_(p.k)
    p.k = rows
    check(p.run(), *p.reference())


def test_a_row_of_nan_stays_its_own(dev):
    """NaN and infinities in a query, or in rows behind the last sequence: the other rows do not see them."""
    b = Batch([(4, 100), (70, 150)], 16, dev, 9)
    p = Packed(b, 128, 4, 8, 2, BF, dev, 120)
    kc, vc = (vectors(121 + i, dev, BF, b.blocks, 16, 2, 128) for i in range(2))
    (o1, b1), (o2, b2) = dense_reference(b, p.q, kc, vc, 1 / math.sqrt(128), 0), p.reference()
    p.q = torch.cat([p.q, torch.full_like(p.q[:3], math.nan)])
    p.q[1, 3] = math.nan
    p.q[20, 5, 7] = math.inf
    p.q[60, 0] = -math.inf
    clean = torch.ones(b.tokens, 8, dtype=torch.bool, device=dev)
    clean[1, 3] = clean[20, 5] = clean[60, 0] = False
    for got, o, bound in ((akv.paged_chunk_attention(p.q, kc, vc, b.tables, b.ctx, b.starts), o1, b1), (p.run(), o2, b2)):
        assert not bool(got[b.tokens:].any())
        check(got[:b.tokens][clean], o[clean], bound[clean])


@pytest.mark.parametrize("dtype,cache_dtype", [(BF, BF), (torch.float32, FP), (FP, torch.float32)])
@pytest.mark.parametrize("sections", [None, (16, 24, 24), (15, 25, 24)])
def test_rope_append_of_many_tokens(dev, dtype, cache_dtype, sections):
    """More rows than the second-level caches hold; axes that take whole units of eight pairs, and others."""
    tokens, heads, kv, d = 3001, 32, 8, 128
    x = vectors(130, dev, dtype, tokens, heads + 2 * kv, d)
    table = table_of(4000, d, dev)
    g = torch.Generator(device=dev).manual_seed(1)
    pos = torch.randint(0, 4000, (3, tokens) if sections else (tokens,), device=dev, generator=g)
    slots = torch.randperm(200 * 16, device=dev, generator=g)[:tokens]
    kc, vc = (torch.zeros(200, 16, kv, d, dtype=cache_dtype, device=dev) for _ in range(2))
    got = akv.rope_append(x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], pos, table, slots, kc, vc, sections=sections)
    check_rope(got, *rope_reference(x[:, :heads], pos, table, sections, False))
    check_rope(kc.flatten(0, 1)[slots], *rope_reference(x[:, heads:heads + kv], pos, table, sections, False))
    assert torch.equal(vc.flatten(0, 1)[slots], x[:, heads + kv:].to(cache_dtype))


@pytest.mark.parametrize("d,heads,kv", [(256, 130, 130), (64, 300, 300), (128, 129, 129)])
def test_mixed_batch_of_many_heads(dev, d, heads, kv):
    """More kv heads than half the workgroups: few and many rows are not divided over one launch."""
    b = Batch([(66, 100), (1, 70), (3, 40)], 16, dev, 11)
    q, kc, vc = (vectors(140 + i, dev, BF, *s) for i, s in enumerate(((b.tokens, heads, d), (b.blocks, 16, kv, d), (b.blocks, 16, kv, d))))
    check(akv.paged_chunk_attention(q, kc, vc, b.tables, b.ctx, b.starts), *dense_reference(b, q, kc, vc, 1 / math.sqrt(d), 0))
    if d > 64:
        p = Packed(b, d, 4, heads, kv, BF, dev, 141)
        check(p.run(), *p.reference())


@pytest.mark.parametrize("few,many", [(1, 40), (40, 1), (12, 12)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_shares_of_a_mixed_batch(dev, few, many, d):
    """Workgroups divided between few and many rows, whichever has more to do."""
    b = Batch([(1 + i % 3, 100 + 177 * i) for i in range(few)] + [(70 + 9 * i, 200 + 50 * i) for i in range(many)], 16, dev, 12)
    q, kc, vc = (vectors(150 + i, dev, FP, *s) for i, s in enumerate(((b.tokens, 8, d), (b.blocks, 16, 2, d), (b.blocks, 16, 2, d))))
    check(akv.paged_chunk_attention(q, kc, vc, b.tables, b.ctx, b.starts), *dense_reference(b, q, kc, vc, 1 / math.sqrt(d), 0))
    for bits in (4, 3, 2):
        p = Packed(b, d, bits, 8, 2, FP, dev, 151)
        check(p.run(), *p.reference())
