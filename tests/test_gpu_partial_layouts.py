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
