"""Scratch of key weights is held to 256 MB (and 2 MB of sums) however wide the tables are, as long as that holds one token: no GPU needed."""
import pytest

from aitherkvcache_amd import _lib

pytestmark = pytest.mark.skipif(not _lib.available(), reason="library not built")

LIMIT = (256 << 20) + (2 << 20) + 8 * 256


@pytest.mark.parametrize("name", ["akv_key_weights_workspace_bytes", "akv_packed_key_weights_workspace_bytes"])
@pytest.mark.parametrize("places", [1 << 12, 1 << 17, 1 << 18, 1 << 20, 1 << 22])
@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (64, 8), (64, 1), (16, 16)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_scratch_is_held(name, places, heads, kv_heads, d):
    size = getattr(_lib.lib(), name)
    for seqs in (1, 4, 16, 64, 1000):
        for tokens in (1, seqs, 3 * seqs, 40 * seqs, 1 << 17):
            assert 0 < size(tokens, seqs, heads, kv_heads, d, places) <= LIMIT, (seqs, tokens)


@pytest.mark.parametrize("name", ["akv_key_weights_workspace_bytes", "akv_packed_key_weights_workspace_bytes"])
def test_scratch_of_the_longest_tables(name):
    """Where one token needs more: eight bytes for each of its heads and 128 keys or more."""
    for seqs, tokens in ((1, 1), (64, 64), (2, 5000)):
        assert 0 < getattr(_lib.lib(), name)(tokens, seqs, 64, 8, 128, 1 << 30) <= LIMIT + 64 * (8 * (1 << 30) // 128 + 4096)
