"""Host side of the paged KV cache: refusals of memory that a call must not be given (fake addresses are never dereferenced)."""
import ctypes

import pytest

from tscale_b200 import abi

CTX, TOKENS, FAR = 1 << 20, 1 << 21, 1 << 24


OF_LENGTHS = [("new", CTX), ("new", CTX + 8), ("new", CTX - 8), ("counts", CTX), ("counts", CTX - 20), ("moves", CTX - 8), ("moves", CTX - 3 * 2 * 50 * 8 + 8)]
OF_TOKENS = [("new", TOKENS), ("counts", TOKENS + 8), ("moves", TOKENS + 8)]


@pytest.mark.parametrize("name,at,positions", [x + (p,) for x in OF_LENGTHS for p in (True, False)] + [x + (True,) for x in OF_TOKENS])
def test_outputs_of_the_choice_that_overlap_its_lengths(name, at, positions):
    """Three sequences of two key heads: lengths of 12 bytes, 24 of counts, 2400 of moves."""
    out = dict(moves=FAR, counts=2 * FAR, new=3 * FAR)
    out[name] = at
    plane = abi.Ptr2D(4 * FAR, 16, 4, 3)
    kv = abi.PagedKv(FAR, FAR, FAR, FAR, FAR if positions else None, FAR, 10, 64, 2)
    rc = abi.lib().tsa_paged_evict_select(ctypes.byref(kv), plane, CTX, TOKENS if positions else None, 3, 200, 50, 4, out["moves"], 50, out["counts"], out["new"], None, None)
    assert rc == abi.TSA_BAD_ARG and b"overlap" in abi.lib().tsa_last_error()
