"""evict_tokens over caches that lie inside one tensor: beside each other they are moved like separate ones, over each other they are refused
and left as they were, through the binding and past it."""
import pytest
import torch

import aitherkvcache_amd as akv
from tests.test_gpu_chunk import BF, Batch
from tests.test_gpu_chunk_use import binding

pytestmark = pytest.mark.gpu

BLOCK, HEADS = 16, 2


def rows_in_engine_tensor(pool):
    """Rows of 32 bytes with a norm behind each, keys and values of a block one after the other."""
    t = pool[:, :2 * BLOCK * HEADS * 36].unflatten(1, (2, BLOCK, HEADS, 36))
    f = pool.view(torch.float32)[:, :2 * BLOCK * HEADS * 9].unflatten(1, (2, BLOCK, HEADS, 9))
    return [t[:, 0, ..., :32], t[:, 1, ..., :32], f[:, 0, ..., 8], f[:, 1, ..., 8]]


def pages(pool):
    """Codes of keys, codes of values, norms of both, one after the other."""
    codes = pool[:, :2048].unflatten(1, (2, BLOCK, HEADS, 32))
    norms = pool.view(torch.float32)[:, 512:512 + 64].unflatten(1, (2, BLOCK, HEADS))
    return [codes[:, 0], codes[:, 1], norms[:, 0], norms[:, 1]]


def heads_first_and_positions_first(pool):
    half = pool.view(BF)
    return [half[:, :512].unflatten(1, (HEADS, BLOCK, 16)).transpose(1, 2), half[:, 512:1024].unflatten(1, (BLOCK, HEADS, 16))]


@pytest.mark.parametrize("take", [True, False])
@pytest.mark.parametrize("to_others", [True, False])
@pytest.mark.parametrize("layout", [rows_in_engine_tensor, pages, heads_first_and_positions_first])
def test_caches_beside_each_other(dev, monkeypatch, layout, to_others, take):
    b = Batch([(0, 200), (0, 90), (0, 17)], BLOCK, dev, seed=31, spare=12)
    pool = torch.randint(1, 100, (b.blocks, 2560), dtype=torch.uint8, generator=torch.Generator().manual_seed(1)).to(dev)
    caches = layout(pool)
    apart = [c.clone() for c in caches]
    w = torch.rand(3, HEADS, b.tables.shape[1] * BLOCK, device=dev)
    spare = torch.tensor(sorted(set(range(b.blocks)) - {int(b.host[i, j]) for i, (_, c) in enumerate(b.lens) for j in range(-(-c // BLOCK))}), dtype=torch.int32, device=dev)
    to = spare[:12].view(3, 4) if to_others else None
    with binding(monkeypatch, take) as c:
        got = akv.evict_tokens(w, b.tables, b.ctx, caches, 60, 2, 8, out_tables=to)
        assert c.taken == (1 if take else 0)
    want = akv.evict_tokens(w, b.tables, b.ctx, apart, 60, 2, 8, out_tables=to)
    for x, y in zip([*got, *caches], [*want, *apart]):
        assert torch.equal(x, y)


@pytest.mark.parametrize("take", [True, False])
@pytest.mark.parametrize("view", [lambda c: c, lambda c: c[1:], lambda c: c[:, :, 1:].expand(-1, -1, HEADS, -1), lambda c: c.flatten(0, 1)[4:-12].unflatten(0, (-1, BLOCK)),
                                  lambda c: c[..., 3:], lambda c: c[::2]])
def test_caches_over_each_other(dev, monkeypatch, view, take):
    b = Batch([(0, 200), (0, 90)], BLOCK, dev, seed=32, spare=3)
    cache = torch.randn(b.blocks, BLOCK, HEADS, 8, device=dev)
    before = cache.clone()
    w = torch.rand(2, HEADS, b.tables.shape[1] * BLOCK, device=dev)
    with binding(monkeypatch, take):
        with pytest.raises(ValueError, match="share"):
            akv.evict_tokens(w, b.tables, b.ctx, [cache, view(cache)], 60, 2, 8)
    assert torch.equal(cache, before)


@pytest.mark.parametrize("take", [True, False])
@pytest.mark.parametrize("strides,fine", [((64, 32, 1), True), ((32, 96, 1), True), ((200, 40, 1), True), ((64, 31, 1), False), ((33, 33, 1), False), ((0, 32, 1), False)])
def test_accumulated_weights_apart_and_over_each_other(dev, monkeypatch, strides, fine, take):
    b = Batch([(3, 20), (1, 30)], BLOCK, dev, seed=35, pad_cols=0)
    q, k = torch.randn(4, 4, 64, device=dev).to(BF), torch.randn(b.blocks, BLOCK, HEADS, 64, device=dev).to(BF)
    want = akv.paged_key_weights(q, k, b.tables, b.ctx, b.starts)
    acc = torch.zeros(1024, device=dev).as_strided((2, HEADS, 32), strides)
    with binding(monkeypatch, take) as c:
        if fine:
            akv.paged_key_weights(q, k, b.tables, b.ctx, b.starts, accumulated=acc)
            assert torch.equal(acc, want) and c.taken == (1 if take else 0)
        else:
            with pytest.raises(ValueError, match="share memory"):
                akv.paged_key_weights(q, k, b.tables, b.ctx, b.starts, accumulated=acc)
            assert not acc.any()


def test_chosen_and_moved_by_two_calls(dev):
    """akv_evict_select, then akv_evict_move: what akv_evict does."""
    from aitherkvcache_amd import _lib
    b = Batch([(0, 200), (0, 90), (0, 17)], BLOCK, dev, seed=36)
    w = torch.rand(3, HEADS, b.tables.shape[1] * BLOCK, device=dev)
    cache, other = torch.randn(b.blocks, BLOCK, HEADS, 5, device=dev), torch.randn(b.blocks, BLOCK, HEADS, device=dev).half()
    mine = [cache.clone(), other.clone()]
    want = akv.evict_tokens(w, b.tables, b.ctx, [cache, other], 60, 2, 8)
    kept, left, now = torch.empty(3, HEADS, 60, dtype=torch.int32, device=dev), torch.empty_like(w), torch.empty(3, dtype=torch.int32, device=dev)
    L, stream = _lib.lib(), _lib.stream_ptr(dev)
    held = (_lib.EvictCache * 2)(*(_lib.EvictCache(c.data_ptr(), *(s * c.element_size() for s in c.stride()[:3]), c[0, 0, 0].numel() * c.element_size()) for c in mine))
    _lib.check(L.akv_evict_select(w.data_ptr(), w.stride(0), w.stride(1), w.shape[2], b.ctx.data_ptr(), 0, 3, HEADS, 60, 2, 8, kept.data_ptr(), kept.stride(0), kept.stride(1), left.data_ptr(),
                                  left.stride(0), left.stride(1), now.data_ptr(), stream))
    _lib.check(L.akv_evict_move(kept.data_ptr(), kept.stride(0), kept.stride(1), now.data_ptr(), 0, 60, b.tables.data_ptr(), 0, b.tables.stride(0), b.tables.shape[1], None, 0, 0, 0, held, 2, 3,
                                HEADS, BLOCK, b.blocks, stream))
    for x, y in zip([kept, now, left, *mine], [*want, cache, other]):
        assert torch.equal(x, y)


def test_rows_of_nothing(dev):
    """A cache whose rows hold nothing does not keep the others from being moved."""
    b = Batch([(0, 200), (0, 90)], BLOCK, dev, seed=37)
    w = torch.rand(2, HEADS, b.tables.shape[1] * BLOCK, device=dev)
    cache = torch.randn(b.blocks, BLOCK, HEADS, 4, device=dev)
    alone = cache.clone()
    empty = torch.zeros(b.blocks, BLOCK, HEADS, 0, device=dev)
    got, want = akv.evict_tokens(w, b.tables, b.ctx, [empty, cache], 60, 2, 8), akv.evict_tokens(w, b.tables, b.ctx, [alone], 60, 2, 8)
    for x, y in zip([*got, cache], [*want, alone]):
        assert torch.equal(x, y)
    got = akv.evict_tokens(w, b.tables, b.ctx, [empty], 60, 2, 8)
    for x, y in zip(got, want):
        assert torch.equal(x, y)
