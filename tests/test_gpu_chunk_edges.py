"""Attention of a chunk where its batch or its cache is out of the ordinary.  Tolerances as in test_gpu_chunk.py, but that a
16-bit weight is off by at most 2^-30 of its row's largest beside its own rounding (float16 has steps of 2^-24 at its lower end, half of one
may be lost, and the largest weight is at least 2^5)."""
import math

import pytest
import torch

import aitherkvcache_amd as akv
from tests.test_gpu_chunk import BF, FP, HALF, Batch, Packed, check, dense_reference, hidden_of, run_dense, softmax_rows, unpack, vectors

pytestmark = pytest.mark.gpu


def dense_inputs(b, heads, kv, d, dtype, dev, seed):
    return [vectors(seed + i, dev, dtype, *s) for i, s in enumerate(((b.tokens, heads, d), (b.blocks, b.block, kv, d), (b.blocks, b.block, kv, d)))]


# ---- more work than 32 bits count ---------------------------------------------------------------------------------------------

def repeated(dev, seqs, n, ctx, seed):
    """A call whose sequences all hold the same 8192 keys over and over, and its result with bound: what they attend to is those keys
    once (`ctx` a multiple of 8192; up to n - 1 of its keys at the end are hidden from a row, 2^-20 of them at most here)."""
    d, heads, keys = 64, 8, 8192
    q, kc, vc = (vectors(seed + i, dev, BF, *s) for i, s in enumerate(((seqs * n, heads, d), (2, keys // 2, 1, d), (2, keys // 2, 1, d))))
    q *= 3
    tables = torch.tensor([0, 1], dtype=torch.int32, device=dev).repeat(ctx // keys).expand(seqs, -1)
    got = akv.paged_chunk_attention(q, kc, vc, tables, torch.full((seqs,), ctx, device=dev), torch.arange(seqs + 1, device=dev) * n, max_query_len=n)
    k, v = kc.view(keys, d).double().T.contiguous(), vc.view(keys, d).double()
    out, size = (torch.empty(seqs * n * heads, d, dtype=torch.float64, device=dev) for _ in range(2))
    for i in range(0, len(out), 8192):
        w = torch.softmax(q.view(-1, d)[i:i + 8192].double() @ k / math.sqrt(d), 1)
        out[i:i + 8192], size[i:i + 8192] = w @ v, w @ v.abs()
    # (sums of ctx / 64 steps or fewer, each rounded: 2^-24 of the sum so far)
    return got, out.view(got.shape), ((2 * HALF[BF] + 2.0 ** -14 + ctx / 64 * 2.0 ** -24) * size).view(got.shape)


@pytest.mark.parametrize("n,ctx", [(1, 1 << 25), (9, 1 << 24)], ids=["few", "many"])
def test_axis_past_32_bits(dev, n, ctx):
    """8192 sequences of 2^18 units each: the axis that is cut among the workgroups is longer than 2^31.  Takes seconds: so much
    work is what it takes to get there."""
    check(*repeated(dev, 8192, n, ctx, 300))


# ---- starts that go back -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("seqs", [7, 300])
@pytest.mark.parametrize("longest", [None, 3])
@pytest.mark.parametrize("d", [64, 128])
def test_starts_out_of_order(dev, seqs, longest, d):
    """Starts that decrease, or lie outside of the call: every workgroup ends, rows that are not the call's stay as they were, and the
    next call is right."""
    b = Batch([(9, 60 + 40 * (i % 9)) for i in range(seqs)], 16, dev, 17)
    p = Packed(b, d, 4, 8, 2, BF, dev, 310)
    kc, vc = (vectors(311 + i, dev, BF, b.blocks, 16, 2, d) for i in range(2))
    want = [p.reference(), dense_reference(b, p.q, kc, vc, 1 / math.sqrt(d), 0)]
    good, n = b.starts.clone(), b.tokens
    room = torch.full((n + 64, 8, d), 7.0, dtype=BF, device=dev)
    calls = (lambda **more: p.run(max_query_len=longest, **more),
             lambda **more: akv.paged_chunk_attention(p.q, kc, vc, b.tables, b.ctx, b.starts, max_query_len=longest, **more))
    g = torch.Generator(device=dev).manual_seed(seqs)
    for bad in (good.flip(0), good[torch.randperm(seqs + 1, device=dev, generator=g)], torch.randint(-50, n + 50, good.shape, device=dev, generator=g),
                torch.where(torch.arange(seqs + 1, device=dev) % 2 == 0, n, 0), torch.full_like(good, n + 1000)):
        b.starts = bad.to(torch.int32)
        for call in calls:
            call(out=room[32:-32])
            call()
    assert bool((room[:32] == 7).all()) and bool((room[-32:] == 7).all())
    b.starts = good
    for call, w in zip(calls, want):
        check(call(), *w)


# ---- windows ---------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("lens", [[(3, 2), (9, 1), (5, 30)], [(100, 10), (300, 290), (90, 33)], [(100, 10), (3, 2)]], ids=["few", "many", "both"])
@pytest.mark.parametrize("window", [(1 << 31) - 1, (1 << 31) - 40, 1 << 40, 7])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_windows_of_any_length_and_rows_before_the_first_key(dev, lens, window, d):
    run_dense(Batch(lens, 16, dev, 18), d, 8, 2, BF, dev, 320, window=window)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("fill", [math.nan, math.inf])
@pytest.mark.parametrize("lens", [[(3, 700), (1, 450), (7, 1201)], [(150, 700), (90, 333), (3, 900)]], ids=["few", "many"])
def test_what_lies_before_every_window_is_not_read(dev, d, dtype, fill, lens):
    """Blocks behind a sliding window have been given back: another request's numbers, or none, and entries of the table to match."""
    for window in (1, 5, 63, 64, 100, 200):
        b = Batch(lens, 16, dev, window, spare=3)
        q, kc, vc = dense_inputs(b, 8, 2, d, dtype, dev, 200)
        b.unused(fill, kc, vc)
        want = dense_reference(b, q, kc, vc, 1 / math.sqrt(d), window)
        spare = (set(range(b.blocks)) - {int(b.host[i, j]) for i, (_, c) in enumerate(lens) for j in range(-(-c // 16))}).pop()
        for i, (n, c) in enumerate(lens):
            old = max(0, c - n - window + 1)          # the first key that any of the sequence's tokens sees
            for x in (kc, vc):
                x[b.host[i, old // 16], :old % 16] = fill
            for j in range(old // 16):
                kc[b.host[i, j]] = vc[b.host[i, j]] = fill
                b.host[i, j] = (spare, -1, int(b.host[i, j]))[j % 3]
        tables = torch.from_numpy(b.host).to(dev, torch.int32)
        check(akv.paged_chunk_attention(q, kc, vc, tables, b.ctx, b.starts, window=window), *want)


# ---- weights far below the largest ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("n", [2, 70], ids=["few", "many"])
@pytest.mark.parametrize("gap", [18.4, 20.0])
def test_small_weights_of_large_values(dev, d, dtype, n, gap):
    """One key of 32 outweighs the others by a factor of exp(gap); their values make up for it."""
    b = Batch([(n, 2600)], 16, dev, 13)
    q, kc, vc = dense_inputs(b, 4, 2, d, dtype, dev, 210)
    q.zero_(), kc.zero_()
    q[..., 3] = 8.0
    heavy = torch.from_numpy(b.host[0, 0:2600 // 16:2]).to(dev)
    kc[heavy, 7, :, 3] = gap / 8 * math.sqrt(d)
    vc.fill_(60000.0)
    vc[heavy, 7] = 1.0
    got = akv.paged_chunk_attention(q, kc, vc, b.tables, b.ctx, b.starts)
    u, c = HALF[dtype], b.lens[0][1]
    k, v = b.rows(kc, 0).double()[:, 0], b.rows(vc, 0).double()[:, 0]
    w = softmax_rows(q[:, 0].double() @ k.T.contiguous() / math.sqrt(d), hidden_of(n, c, 0, dev))
    out = (w @ v)[:, None].expand(n, 4, d)
    check(got, out, (2 * u + 2.0 ** -14) * out + 2.0 ** -30 * w.amax(1)[:, None, None] * float(v.sum(0)[0]))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [2, 70], ids=["few", "many"])
def test_large_bfloat16_values(dev, d, n):
    """Values of up to 2^119 under equal scores: with weights of 1 their sum over 100 keys is a float32 number."""
    b = Batch([(n, 100)], 16, dev, 25)
    q, kc, vc = dense_inputs(b, 4, 2, d, BF, dev, 215)
    q.zero_()
    vc = (vc.float().abs().clamp(0.5, 2.0) * 2.0 ** 118).bfloat16()
    got = akv.paged_chunk_attention(q, kc, vc, b.tables, b.ctx, b.starts)
    check(got, *dense_reference(b, q, kc, vc, 1 / math.sqrt(d), 0))


# ---- norms of zero -------------------------------------------------------------------------------------------------------------------

def packed_reference(p):
    """(out, bound): as Packed.reference, the loss of small weights by what weight times norm is at most."""
    b, q, d = p.b, p.q, p.d
    pi, cen, scale = p.tq.rotation.double(), p.tq.centroids.double(), p.attn.scale
    out, bound = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    group, at = q.shape[1] // p.k.shape[2], 0
    for i, (n, c) in enumerate(b.lens):
        ck, cv = (cen[unpack(b.rows(x, i), p.bits, d)] for x in (p.k, p.v))
        kn, vn = b.rows(p.kn, i).double(), b.rows(p.vn, i).double()
        hidden = hidden_of(n, c, 0, q.device)
        for h in range(q.shape[1]):
            j = h // group
            turned = q[at:at + n, h].double() @ pi.T.contiguous()
            k = ck[:, j] * kn[:, j, None]
            a = softmax_rows(turned @ k.T.contiguous() * scale, hidden) * vn[:, j]          # weight times norm
            out[at:at + n, h] = a @ cv[:, j] @ pi
            e = ((turned.abs() @ k.abs().T.contiguous()) * scale).masked_fill(hidden, 0.0).amax(1, keepdim=True) * 2.0 ** -10
            grown = torch.expm1(2 * e)
            lost = 2.0 ** -30 * a.amax(1, keepdim=True) * cv[:, j].abs().sum(0)
            bound[at:at + n, h] = ((grown + 2.0 ** -10 + 2.0 ** -13) * (1 + grown) * (a @ cv[:, j].abs()) + lost) @ pi.abs() + HALF[q.dtype] * out[at:at + n, h].abs() + 1e-38
        at += n
    return out, bound


@pytest.mark.parametrize("d,bits", [(64, 3), (128, 4), (256, 2)])
@pytest.mark.parametrize("lens", [[(3, 200), (1, 64)], [(90, 200), (70, 71)]], ids=["few", "many"])
@pytest.mark.parametrize("size", [2.0 ** -50, 2.0 ** -26, 1.0, 2.0 ** 40])
def test_zero_norms_beside_norms_of_any_size(dev, d, bits, lens, size):
    """A value of zero has weight and no size: how large the others are does not change by it."""
    b = Batch(lens, 16, dev, 14)
    p = Packed(b, d, bits, 8, 2, BF, dev, 220)
    p.kn.mul_(0.02)
    p.vn.mul_(size)
    for i, (_, c) in enumerate(lens):
        p.vn[b.host[i, 0], 5] = 0.0
        p.vn[b.host[i, c // 32], 2, 1] = 0.0
    check(p.run(), *packed_reference(p))


@pytest.mark.parametrize("d,bits", [(64, 3), (128, 4), (256, 2)])
@pytest.mark.parametrize("lens", [[(3, 200)], [(90, 200)]], ids=["few", "many"])
@pytest.mark.parametrize("score", [10.0, 24.0])
def test_a_zero_value_may_outweigh_all_others(dev, d, bits, lens, score):
    """Attention rests on keys whose values are zero, one of 32 (by exp(score)): what the others leave is small, and right."""
    b = Batch(lens, 16, dev, 15)
    p = Packed(b, d, bits, 8, 2, BF, dev, 221)
    p.kn.mul_(0.02)
    at = (int(b.host[0, 0]), 9)
    heavy = torch.from_numpy(b.host[0, 0:lens[0][1] // 16:2]).to(dev)
    p.k[heavy, 9] = p.k[at]
    p.v.copy_(p.v[at].clone())                 # (values alike: nothing of the result cancels)
    p.vn[heavy, 9] = 0.0
    p.kn[heavy, 9] = score
    code = p.tq.centroids.double()[unpack(p.k[at], bits, d)]                                # [kv heads, d]
    row = code @ p.tq.rotation.double() * math.sqrt(d)
    p.q = (row / (code * code).sum(-1, keepdim=True)).repeat_interleave(4, 0).expand(b.tokens, 8, d).to(BF).contiguous()
    check(p.run(), *packed_reference(p))


# ---- codebooks ---------------------------------------------------------------------------------------------------------------------

def test_codebooks_in_other_forms(dev):
    """Levels as float64 or a strided view are what they are as float32; on the host, or too few, they are refused."""
    p = Packed(Batch([(3, 90), (40, 77)], 16, dev, 19), 128, 4, 8, 2, BF, dev, 330)
    want, levels = p.run(), p.tq.centroids
    for same in (levels.double(), torch.stack([levels, -levels], 1)[:, 0]):
        p.attn.centroids = same
        assert torch.equal(p.run(), want)
    for error, other in ((RuntimeError, levels.cpu()), (ValueError, levels[:8])):
        p.attn.centroids = other
        with pytest.raises(error):
            p.run()


# ---- rows of no sequence ------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("lens", [[(3, 50)], [(90, 90)], [(3, 50), (90, 90)]], ids=["few", "many", "both"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_before_the_first_sequence(dev, lens, d):
    """Starts that begin past row 0 (a part of a batch): rows of nobody are zero in a new tensor and left alone in a given one."""
    b = Batch(lens, 16, dev, 16)
    p = Packed(b, d, 4, 8, 2, BF, dev, 230)
    _, kc, vc = dense_inputs(b, 8, 2, d, BF, dev, 231)
    want = [p.reference(), dense_reference(b, p.q, kc, vc, 1 / math.sqrt(d), 0)]
    p.q = torch.cat([torch.ones(37, 8, d, dtype=BF, device=dev), p.q, torch.ones(5, 8, d, dtype=BF, device=dev)])
    b.starts = b.starts + 37
    for call, w in zip((p.run, lambda **more: akv.paged_chunk_attention(p.q, kc, vc, b.tables, b.ctx, b.starts, **more)), want):
        for _ in range(2):
            torch.full_like(p.q, 7.0)                       # (what the next tensor of this size finds in memory)
            got = call()
            check(got[37:-5], *w)
            assert not bool(got[:37].any()) and not bool(got[-5:].any())
        mine = torch.full_like(p.q, 7.0)
        call(out=mine)
        check(mine[37:-5], *w)
        assert bool((mine[:37] == 7).all()) and bool((mine[-5:] == 7).all())


def test_rows_of_no_sequence_at_all(dev):
    """No sequences: every row is nobody's, wherever the one start stands."""
    kc = torch.ones(2, 16, 2, 64, dtype=FP, device=dev)
    none = torch.zeros(0, 1, dtype=torch.int32, device=dev)
    q = torch.ones(37, 8, 64, dtype=FP, device=dev)
    for start in (0, 20, 37):
        torch.full_like(q, 7.0)
        assert not bool(akv.paged_chunk_attention(q, kc, kc, none, none[:, 0], torch.tensor([start], device=dev)).any())


# ---- caches laid out otherwise -----------------------------------------------------------------------------------------------------

def relaid(x, order):
    """The same cache with its dimensions in `order` in memory, rows 16 bytes apart and more."""
    room = torch.zeros(*[x.shape[i] for i in order], x.shape[3] + (16 if x.dtype == torch.uint8 else 8), dtype=x.dtype, device=x.device)
    back = [order.index(i) for i in range(3)]
    y = room[..., :x.shape[3]].permute(*back, 3)
    return y.copy_(x)


@pytest.mark.parametrize("lens", [[(3, 150), (1, 40)], [(90, 200), (70, 70)], [(3, 150), (90, 200)]], ids=["few", "many", "both"])
@pytest.mark.parametrize("orders", [((0, 2, 1), (0, 1, 2)), ((2, 0, 1), (1, 0, 2)), ((0, 2, 1), (0, 2, 1))])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_keys_and_values_laid_out_otherwise(dev, lens, orders, d):
    """Heads before places, heads before blocks, places before blocks; keys and values each their own."""
    b = Batch(lens, 16, dev, 26)
    q, kc, vc = dense_inputs(b, 8, 2, d, BF, dev, 340)
    b.unused(math.nan, kc, vc)
    want = akv.paged_chunk_attention(q, kc, vc, b.tables, b.ctx, b.starts)
    check(want, *dense_reference(b, q, kc, vc, 1 / math.sqrt(d), 0))
    assert torch.equal(akv.paged_chunk_attention(q, relaid(kc, orders[0]), relaid(vc, orders[1]), b.tables, b.ctx, b.starts), want)
    p = Packed(b, d, 3, 8, 2, BF, dev, 341)
    want = p.run()
    check(want, *p.reference())
    p.k, p.v = relaid(p.k, orders[0]), relaid(p.v, orders[1])
    assert torch.equal(p.run(), want)
    p.kn, p.vn = (relaid(x[..., None], o)[..., 0] for x, o in ((p.kn, orders[1]), (p.vn, orders[0])))
    assert torch.equal(p.run(), want)
    slots = torch.randperm(b.blocks * 16, device=dev)[:b.tokens]
    plain, other = [torch.zeros_like(kc) for _ in range(2)], [relaid(torch.zeros_like(kc), o) for o in orders]
    for caches in (plain, other):
        akv.rope_append(None, q[:, :2], q[:, 2:4], None, None, slots, *caches)
    assert torch.equal(other[0], plain[0]) and torch.equal(other[1], plain[1])
