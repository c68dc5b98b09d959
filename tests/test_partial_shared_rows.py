"""Caches of evict_tokens that share rows with each other, or with themselves, are refused before anything runs: no GPU needed."""
import random

import pytest

from aitherkvcache_amd import _lib

pytestmark = pytest.mark.skipif(not _lib.available(), reason="library not built")

P = 1 << 16          # an address that is aligned and never read
# blocks of sixteen tokens of two heads, rows of 128 bytes
BLK, POS, HEAD, ROW = 4096, 256, 128, 128
ONE = (P, BLK, POS, HEAD, ROW)


def held(caches):
    return (_lib.EvictCache * len(caches))(*(_lib.EvictCache(*c) for c in caches))


def move(caches, blocks):
    return _lib.lib().akv_evict_move(P, 20, 10, P, 0, 10, P, 0, 2, 2, None, 0, 2, 2, held(caches), len(caches), 2, 2, 16, blocks, None)


def evict(caches, blocks):
    return _lib.lib().akv_evict(P, 64, 32, 32, P, 0, 2, 2, 10, 2, 4, P, 20, 10, P, 64, 32, P, P, 0, 2, 2, None, 0, 2, 2, held(caches), len(caches), 16, blocks, None)


@pytest.mark.parametrize("call", [move, evict])
@pytest.mark.parametrize("blocks,caches", [
    (3, [ONE, ONE]),
    # a view of the same storage, further by a head, a position, a block, by some of each, and back
    (3, [ONE, (P + HEAD, BLK, POS, HEAD, ROW)]),
    (3, [ONE, (P + POS, BLK, POS, HEAD, ROW)]),
    (3, [ONE, (P + BLK, BLK, POS, HEAD, ROW)]),
    (3, [ONE, (P + 2 * BLK + 5 * POS - HEAD, BLK, POS, HEAD, ROW)]),
    (3, [ONE, (P - BLK, BLK, POS, HEAD, ROW)]),
    (3, [ONE, (P - POS - HEAD, BLK, POS, HEAD, ROW)]),
    # by a part of a row
    (3, [ONE, (P + 4, BLK, POS, HEAD, 64)]),
    (3, [ONE, (P + 2 * BLK + POS + 64, BLK, POS, HEAD, ROW)]),
    (3, [(P, BLK, POS, HEAD, 64), (P + BLK + 60, BLK, POS, HEAD, 8)]),
    # far apart in the call: the last of three with the first
    (3, [ONE, (P + (1 << 20), BLK, POS, HEAD, ROW), (P + BLK, BLK, POS, HEAD, ROW)]),
    # strides that differ: heads before positions, blocks of another size, every other block
    (3, [ONE, (P, BLK, HEAD, 16 * HEAD, ROW)]),
    (3, [ONE, (P + 64, BLK, HEAD, 16 * HEAD, 32)]),
    (3, [ONE, (P + BLK, 2 * BLK, POS, HEAD, ROW)]),
    (3, [(P, 2 * BLK, POS, HEAD, ROW), (P + BLK, 3 * BLK, POS, HEAD, ROW)]),
    # pages of codes and norms whose norms begin too early, or run into the next page
    (3, [(P, 8192, POS, HEAD, ROW), (P + 4096 - 8, 8192, 8, 4, 4)]),
    (3, [(P, 4224, POS, HEAD, ROW), (P + 4096 + 64, 4224, 8, 4, 4)]),
    # rows of one cache that share memory: an expanded dimension, rows that overlap, blocks that do
    (3, [(P, BLK, POS, 0, ROW)]),
    (3, [(P, BLK, 0, HEAD, ROW)]),
    (3, [(P, 0, POS, HEAD, ROW)]),
    (3, [(P, BLK, POS, 64, ROW)]),
    (3, [(P, BLK, POS - 4, HEAD, ROW)]),
    (3, [(P, 2048, POS, HEAD, ROW)]),
    (1 << 30, [ONE, (P + (BLK << 29), BLK, POS, HEAD, ROW)]),
])
def test_rows_in_two_places_are_refused(call, blocks, caches):
    assert call(caches, blocks) == _lib.AKV_ERR_INVALID
    assert b"share" in _lib.lib().akv_last_error()
    if len(caches) == 2:
        assert call(caches[::-1], blocks) == _lib.AKV_ERR_INVALID


def places(cache, blocks, block, heads):
    p, *strides, row = cache
    return [p + b * strides[0] + t * strides[1] + h * strides[2] for b in range(blocks) for t in range(block) for h in range(heads)], row


def meet(x, y, shape):
    """Whether a row of x and one of y (of one cache: two of its rows) have a byte in common."""
    (xs, xr), (ys, yr) = places(x, *shape), places(y, *shape)
    return any(a < b + yr and b < a + xr for i, a in enumerate(xs) for j, b in enumerate(ys) if x is not y or i != j)


def checked(caches, shape):
    """The refusal alone: blocks to move to that have room for nothing."""
    blocks, block, heads = shape
    return _lib.lib().akv_evict_move(P, 20, 10, P, 0, 10, P, 0, 2, 2, P, 0, 2, 0, held(caches), len(caches), 2, heads, block, blocks, None)


def test_what_is_refused_is_what_meets():
    rng = random.Random(5)
    outcomes = [0, 0]
    for _ in range(4000):
        shape = rng.choice([(3, 4, 2), (1, 3, 2), (4, 1, 3), (2, 2, 1), (3, 2, 2)])
        row = rng.choice([4, 8, 12])
        # a layout of rows side by side, its dimensions in any order, with gaps or without, or (at times) one that is none
        strides, at = [0, 0, 0], row + rng.choice([0, 0, 4, 16])
        for i in rng.sample(range(3), 3):
            strides[i] = at
            at = at * shape[i] + rng.choice([0, 0, 8, 40])
        if rng.random() < 0.15:
            strides[rng.randrange(3)] = rng.choice([0, 4, 8, 20])
        x = (P, *strides, row)
        y = (P + 4 * rng.randrange(-at // 2, at // 2), *strides, rng.choice([4, 8, 12]))
        want = meet(x, x, shape) or meet(y, y, shape) or meet(x, y, shape)
        outcomes[want] += 1
        assert checked([x, y], shape) == (_lib.AKV_ERR_INVALID if want else 0), (x, y, shape)
        # other strides: what meets is refused, what lies apart is not
        z = (y[0], *rng.sample(strides, 3), y[4])
        if meet(x, z, shape):
            assert checked([x, z], shape) == _lib.AKV_ERR_INVALID, (x, z, shape)
        elif not meet(x, x, shape) and not meet(z, z, shape):
            far = (max(places(x, *shape)[0]) + row, *z[1:])
            assert checked([x, far], shape) == 0, (x, far, shape)
    assert min(outcomes) > 500


@pytest.mark.parametrize("caches", [
    # keys and values of a block one after the other, norms in the ends of rows
    [(P, 9216, 288, 144, 128), (P + 4608, 9216, 288, 144, 128), (P + 128, 9216, 288, 144, 4), (P + 4608 + 128, 9216, 288, 144, 4)],
    # pages: codes of keys, codes of values, norms of both
    [(P, 8448, POS, HEAD, ROW), (P + 4096, 8448, POS, HEAD, ROW), (P + 8192, 8448, 8, 4, 4), (P + 8192 + 128, 8448, 8, 4, 4)],
    # keys heads first, values positions first
    [(P, 8192, HEAD, 16 * HEAD, ROW), (P + 4096, 8192, POS, HEAD, ROW)],
    # every other block of a pool
    [(P, 2 * BLK, POS, HEAD, ROW), (P + BLK, 2 * BLK, POS, HEAD, ROW)],
    # halves of a pool; halves of rows
    [ONE, (P + 3 * BLK, BLK, POS, HEAD, ROW)],
    [(P, BLK, POS, HEAD, 64), (P + 64, BLK, POS, HEAD, 64)],
])
def test_layouts_side_by_side_are_taken(caches):
    for order in (caches, caches[::-1]):
        assert checked(order, (3, 16, 2)) == 0
    assert checked([ONE, (P + BLK, BLK, POS, HEAD, ROW)], (1, 16, 2)) == 0      # (of pools of one block: another block)
