"""Host side of PagedKVCache: limits of its book-keeping."""
import numpy as np
import pytest

from tscale_b200 import abi, ops


def test_positions_end_with_int32():
    """A cache that is cut may see any number of tokens; their positions are 32-bit numbers."""
    cache = ops.PagedKVCache(2, 12, 2, 64, "cpu", page_size=16, evict=True)
    cache.extend([3, 5])
    cache.seen[:] = [10, 2 ** 31 - 3]
    cache.extend([4, 2])
    assert cache.tokens.tolist() == [14, 2 ** 31 - 1]
    before = cache._host.copy()
    for counts in (1, [0, 1], [1, 20]):
        with pytest.raises(abi.TsaError, match="positions"):
            cache.extend(counts)
        assert np.array_equal(cache._host, before) and len(cache.free) == 10
    cache.extend([1, 0])
    cache.release(1)
    cache.extend()
    assert cache.tokens.tolist() == [16, 1]
