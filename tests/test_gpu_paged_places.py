"""GPU tests of paged_append where rows have no place: they are left out, and all others are stored."""
import pytest
import torch

from tests.test_gpu_paged import DEV, Cache, _codes, _gen, _same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv,scale,kvh,d,track", [("i8", torch.float16, 2, 64, True), ("e4m3", torch.float32, 12, 128, True), ("i8", torch.float32, 1, 128, False)])
@pytest.mark.parametrize("ctx,pages", [([20, 1, 20], {}), ([20, 20, 40], {}), ([0, -3, 33], {}), ([20, 20, 2 ** 31 - 1], {}), ([20, 20, 20], {(1, 1): -1}),
                                       ([20, 20, 20], {(1, 1): 1 << 20, (2, 0): -2 ** 31}), ([17, 17, 17], {(0, 0): -1, (2, 1): 2 ** 31 - 1})])
def test_rows_without_a_place(kv, scale, kvh, d, track, ctx, pages):
    from tscale_b200 import ops
    c = Cache(40, [20, 20, 20], kvh, d, 16, kv, scale, track)
    gen, starts, rows = _gen(40), [0, 2, 4, 7], 7
    k, v = _codes((rows, kvh * d), kv, gen), _codes((rows, kvh * d), kv, gen)
    ks, vs = torch.rand((kvh, rows), generator=gen, device=DEV), torch.rand((kvh, rows), generator=gen, device=DEV)
    table = c.host_table.clone()
    for at, page in pages.items():
        table[at] = page
    planes = [None if x is None else (x.view(torch.int8) if x.element_size() == 1 else x) for x in c.kv]
    want, lost = [None if x is None else x.clone() for x in planes], 0
    for s in range(3):
        for row in range(starts[s], starts[s + 1]):
            back = starts[s + 1] - row
            slot = ctx[s] - back
            page = int(table[s, slot // 16]) if 0 <= slot < 16 * table.shape[1] else -1
            if not 0 <= page < c.k.shape[0]:
                lost += 1
                continue
            at = (page, slice(None), slot % 16)
            want[0][at], want[1][at] = k.view(torch.int8)[row].view(kvh, d), v.view(torch.int8)[row].view(kvh, d)
            want[2][at], want[3][at] = ks[:, row].to(scale), vs[:, row].to(scale)
            if track:
                want[4][at], want[5][at] = int(c.tokens[s]) - back, 0.0
    assert 0 < lost < rows
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.paged_append(c.kv, table.to(DEV), torch.tensor(ctx, dtype=torch.int32, device=DEV), k, ks, v, vs, torch.tensor(starts, dtype=torch.int32, device=DEV), c.tokens, status)
    assert int(status) != 0 and all(_same(a, b) for a, b in zip(planes, want))


@pytest.mark.parametrize("kvh,d,rows", [(2, 64, 3000), (16, 128, 500)])
def test_rows_that_the_kernel_before_writes(kvh, d, rows):
    """The quantiser lets the next kernel start while it still writes; replayed, it writes other rows over those of the replay before."""
    from tscale_b200 import ops
    c = Cache(41, [rows], kvh, d, 64, "i8", torch.float32, False)
    gen = _gen(41)
    x, starts = torch.zeros((rows, kvh * d), device=DEV), torch.tensor([0, rows], dtype=torch.int32, device=DEV)
    p, o = c.place(0)

    def step():
        k, ks = ops.quant_rows(x, "rms", "i8", d, vec_scale=1 / 24.0)
        ops.paged_append(c.kv, c.table, c.ctx, k.view(torch.int8), ks, k.view(torch.int8), ks, starts)
        return k, ks

    x.copy_(torch.randn(x.shape, generator=gen, device=DEV))
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        k, ks = step()
    for _ in range(20):
        x.copy_(torch.randn(x.shape, generator=gen, device=DEV))
        graph.replay()
        for plane in (c.k, c.v):
            assert torch.equal(plane[p, :, o].reshape(rows, -1), k.view(torch.int8))
        assert torch.equal(c.ks[p, :, o], ks.t()) and torch.equal(c.vs[p, :, o], ks.t()) and k.any()
