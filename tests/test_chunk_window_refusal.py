"""Windows of paged_chunk_attention that the host decides on: no GPU needed."""
import pytest

from aitherkvcache_amd import _lib
from tests.test_chunk_refusals import c_dense


@pytest.mark.parametrize("window", [(1 << 30) + 1, 0x7ffe0000])
def test_a_window_past_30_bits_over_a_longer_table_is_refused(window):
    """A position may lie 2^30 below 0 (a chunk longer than its context): the two together would not fit 32 bits."""
    assert c_dense(window=window, block=1 << 20, width=1 << 12) == _lib.AKV_ERR_UNSUPPORTED
