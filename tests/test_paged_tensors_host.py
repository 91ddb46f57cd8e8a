"""Host side of the paged functions: tensors that they must not take (on the CPU: a call that gets past these checks ends at the check for a GPU)."""
import pytest
import torch

from tscale_b200 import ops

PLANE = (10, 2, 64)
KV = ops.PagedKV(torch.zeros(PLANE + (64,), dtype=torch.int8), torch.zeros(PLANE + (64,), dtype=torch.int8), torch.ones(PLANE, dtype=torch.float16),
                 torch.ones(PLANE, dtype=torch.float16), torch.zeros(PLANE, dtype=torch.int32), torch.zeros(PLANE))
TABLE, CTX = torch.zeros((3, 4), dtype=torch.int32), torch.ones(3, dtype=torch.int32)
ROW, SCALE = torch.zeros((3, 128), dtype=torch.int8), torch.ones((2, 3))
MOVES, COUNTS = torch.zeros((3, 2, 5, 2), dtype=torch.int32), torch.zeros((3, 2), dtype=torch.int32)
CALLS = [lambda **kw: ops.paged_append(KV, TABLE, CTX, ROW, SCALE, ROW, SCALE, tokens=CTX, **kw),
         lambda **kw: ops.paged_decode(KV, TABLE, CTX, torch.zeros((3, 256), dtype=torch.int8), None, 5, 0.0, tokens=CTX, **kw),
         lambda **kw: ops.paged_evict_select(KV, TABLE, CTX, 5, 1, tokens=CTX, **kw), lambda **kw: ops.paged_evict_move(KV, TABLE, MOVES, COUNTS, **kw)]


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("status,text", [(torch.zeros(1, dtype=torch.int16), "status"), (torch.zeros(1, dtype=torch.uint8), "status"), (torch.zeros(1), "status"),
                                         (torch.zeros(0, dtype=torch.int32), "status"), (torch.zeros(1, dtype=torch.int32), "one GPU"), (None, "one GPU")])
def test_status_words(call, status, text):
    with pytest.raises(AssertionError, match=text):
        call(status=status)


@pytest.mark.parametrize("workspace,text", [(torch.zeros(1, dtype=torch.uint8).expand(1 << 20), "contiguous"), (torch.zeros(1 << 12, dtype=torch.uint8)[::2], "contiguous"),
                                            (torch.zeros((64, 64)).t(), "contiguous"), (torch.zeros(1 << 12, dtype=torch.uint8), "one GPU")])
def test_workspaces(workspace, text):
    """Memory that a tensor only seems to have, or that lies between its elements."""
    with pytest.raises(AssertionError, match=text):
        CALLS[1](workspace=workspace)
