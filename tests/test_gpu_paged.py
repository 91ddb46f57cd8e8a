"""GPU tests of the paged KV cache (append, decode, eviction) against plain implementations in 64 bits.

Tolerances.  A logit is three float32 roundings of a value below 32 (the inputs are made so): its weight is off by at most
3 * 2^-24 * 32 * ln 2 plus 2^-22 of the exponential, 5e-6 of itself.  The weights are multiplied in two f16 parts (2^-22) and summed in
float32 with at most 64 roundings per partial sum (2^-24 each, 4e-6; twice that if an instruction truncates).  Together below 2^-16 of the
sum of weights times the largest value.  Results in 16 bits may be half a step off on top.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ERR = 2.0 ** -16
WHOLE = 1 << 30
CODES = {"i8": torch.int8, "e4m3": torch.float8_e4m3fn}
DOT = 0.5 / 0.693147


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _codes(shape, kv, gen):
    x = torch.randn(shape, generator=gen, device=DEV)
    return (x * 40).round().clamp(-128, 127).to(torch.int8) if kv == "i8" else (x * 1.5).to(CODES[kv])


def _unit(kv):
    return 1 / 40.0 if kv == "i8" else 1 / 1.5


class Cache:
    """Pools whose unused slots hold NaN (e4m3 codes, scales) or nonsense, with the tokens of `lens` in shuffled pages."""

    def __init__(self, seed, lens, kvh, d, page, kv, scale, track, spare=2, max_pages=None):
        from tscale_b200 import ops
        gen = _gen(seed)
        self.lens, self.kvh, self.d, self.page, self.kv_type = list(lens), kvh, d, page, kv
        used = [-(-n // page) for n in lens]
        cols = max_pages or max(max(used), 1)
        pages = sum(used) + spare
        order = torch.randperm(pages, generator=gen, device=DEV).tolist()
        table = torch.full((len(lens), cols), -1, dtype=torch.int32)
        for s, n in enumerate(used):
            for i in range(n):
                table[s, i] = order.pop()
        self.host_table = table
        self.table = table.to(DEV)
        plane = (pages, kvh, page)
        live = torch.zeros((pages, page), dtype=torch.bool)
        for s, n in enumerate(lens):
            for t in range(0, n, page):
                live[table[s, t // page], :min(page, n - t)] = True
        self.live = live[:, None].expand(plane).to(DEV)
        self.k, self.v = _codes(plane + (d,), kv, gen), _codes(plane + (d,), kv, gen)
        self.ks, self.vs = (((torch.rand(plane, generator=gen, device=DEV) + 0.5) * _unit(kv)).to(scale) for _ in range(2))
        for x in (self.ks, self.vs):
            x[~self.live] = float("nan")
        if kv == "e4m3":
            for x in (self.k, self.v):
                x.view(torch.uint8)[~self.live] = 0x7f
        self.pos = self.weight = self.tokens = None
        if track:
            self.pos = torch.full(plane, 1 << 20, dtype=torch.int32, device=DEV)
            self.weight = torch.full(plane, float("nan"), device=DEV)
            seen = [n + (7 * s) % 50 for s, n in enumerate(lens)]
            self.tokens = torch.tensor(seen, dtype=torch.int32, device=DEV)
            for s, n in enumerate(lens):
                for h in range(kvh):
                    if n:
                        keep = torch.randperm(seen[s] - 1, generator=gen, device=DEV)[:n - 1]
                        self.write(self.pos, s, h, torch.cat([keep, torch.tensor([seen[s] - 1], device=DEV)]).to(torch.int32))
                        self.write(self.weight, s, h, torch.rand(n, generator=gen, device=DEV))
        self.kv = ops.PagedKV(self.k, self.v, self.ks, self.vs, self.pos, self.weight)
        self.ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)

    def place(self, s, n=None):
        t = torch.arange(self.lens[s] if n is None else n, device=DEV)
        return self.table[s].long()[t // self.page], t % self.page

    def write(self, plane, s, h, values):
        p, o = self.place(s, len(values))
        plane[p, h, o] = values

    def read(self, plane, s, h):
        p, o = self.place(s)
        return (plane.view(torch.int8)[p, h, o].view(plane.dtype) if plane.element_size() == 1 else plane[p, h, o]).double()


def _decode_ref(c, q, qs, heads, window, slope):
    """(out [n][H * D], {(s, h): weights}) in 64 bits."""
    d, group = c.d, heads // c.kvh
    out = torch.zeros((len(c.lens), heads, d), dtype=torch.float64, device=DEV)
    added = {}
    for s, n in enumerate(c.lens):
        if n == 0:
            continue
        for h in range(c.kvh):
            pos = torch.arange(n, device=DEV, dtype=torch.float64) if c.pos is None else c.read(c.pos, s, h)
            cur = (n if c.tokens is None else int(c.tokens[s])) - 1
            far = cur - pos
            sel = far == 0 if window == 0 else (far >= 1) & (far <= window)
            k = c.read(c.k, s, h)[sel] * c.read(c.ks, s, h)[sel][:, None]
            v = c.read(c.v, s, h)[sel] * c.read(c.vs, s, h)[sel][:, None]
            qh = q[s].view(heads, d)[h * group:(h + 1) * group].double() * qs[s, h * group:(h + 1) * group].double()[:, None]
            z = qh @ k.T * (DOT / d ** 0.5) - slope * far[sel]
            assert not z.numel() or float(z[torch.isfinite(z)].abs().max()) < 32 + slope * 1000
            w = torch.exp2(z)
            w = w / (1 + w.sum(1, keepdim=True))
            out[s, h * group:(h + 1) * group] = w @ v
            full = torch.zeros(n, dtype=torch.float64, device=DEV)
            full[sel] = w.sum(0)
            added[s, h] = full
    return out.view(len(c.lens), -1), added


def _query(seed, n, heads, d, kv):
    gen = _gen(seed + 1000)
    return _codes((n, heads * d), kv, gen), (torch.rand((n, heads), generator=gen, device=DEV) + 0.5) * _unit(kv)


def _check_out(got, want, c):
    big = max([1e-6] + [float((c.read(c.v, s, h) * c.read(c.vs, s, h)[:, None]).abs().max()) for s, n in enumerate(c.lens) if n for h in range(c.kvh)])
    tol = ERR * big + (0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2) * want.abs()
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), float((got.double() - want).abs().max()), big)


LENS = [0, 1, 2, 16, 17, 33, 130, 700, 255]


@pytest.mark.parametrize("kv,scale,d,heads,kvh,page,window,slope,out,track", [
    ("i8", torch.float16, 128, 4, 4, 64, WHOLE, 0.0, torch.float32, False),
    ("e4m3", torch.float16, 128, 8, 2, 16, WHOLE, 0.0, torch.bfloat16, False),
    ("i8", torch.float32, 64, 12, 12, 32, WHOLE, 0.01, torch.float32, False),
    ("e4m3", torch.float32, 64, 7, 1, 128, WHOLE, 0.0, torch.float16, False),
    ("i8", torch.float16, 128, 16, 1, 256, 100, 0.0, torch.float32, False),   # sixteen heads share a key head
    ("e4m3", torch.float16, 64, 24, 2, 16, 200, 0.02, torch.float32, True),    # twelve
    ("i8", torch.float32, 128, 40, 1, 64, WHOLE, 0.0, torch.float32, True),   # more than a unit's sixteen
    ("i8", torch.float16, 64, 8, 8, 16, 64, 0.5, torch.float32, False),       # short window: one CTA per unit
    ("e4m3", torch.float32, 128, 6, 3, 32, 64, 0.5, torch.bfloat16, True),
    ("i8", torch.float16, 128, 4, 2, 32, 0, 0.0, torch.float32, False),       # the new token itself
    ("i8", torch.float16, 64, 9, 1, 64, 0, 0.0, torch.float32, True),
    ("i8", torch.float16, 128, 32, 8, 64, 1, 0.0, torch.float16, True),
])
def test_decode(kv, scale, d, heads, kvh, page, window, slope, out, track):
    _decode_of(LENS, kv, scale, d, heads, kvh, page, window, slope, out, track)


def _decode_of(lens, kv, scale, d, heads, kvh, page, window, slope, out, track):
    from tscale_b200 import ops
    c = Cache(1, lens, kvh, d, page, kv, scale, track)
    q, qs = _query(1, len(lens), heads, d, kv)
    before = None if c.weight is None else c.weight.clone()
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    want, added = _decode_ref(c, q, qs, heads, window, slope)
    got = ops.paged_decode(c.kv, c.table, c.ctx, q, qs, window, slope, max_ctx=max(lens), out_dtype=out, tokens=c.tokens, status=status)
    assert int(status) == 0
    _check_out(got, want, c)
    assert not got[0].any()
    if not track:
        assert not got[1].any() or window == 0
    if track:
        for (s, h), w in added.items():
            p, o = c.place(s)
            diff = c.weight[p, h, o].double() - before[p, h, o].double() - w
            assert float(diff.abs().max()) <= ERR * (heads // kvh) + 2.0 ** -23
            assert (c.weight[p, h, o][w == 0] == before[p, h, o][w == 0]).all()
        assert torch.equal(c.weight[~c.live].isnan(), torch.ones_like(c.weight[~c.live], dtype=torch.bool))
    # the bound may be larger than the longest sequence, and absent
    if not track:
        assert torch.equal(got, ops.paged_decode(c.kv, c.table, c.ctx, q, qs, window, slope, max_ctx=max(lens), out_dtype=out, tokens=c.tokens))
        _check_out(ops.paged_decode(c.kv, c.table, c.ctx, q, qs, window, slope, out_dtype=out), want, c)


MANY = [0, 1, 700, 129, 128, 127, 2, 1000, 383, 16, 257, 640]  # with eight or more key heads: more units than clusters would have room for


@pytest.mark.parametrize("kv,scale,d,heads,kvh,page,window,slope,out,track", [
    ("i8", torch.float16, 128, 8, 8, 64, WHOLE, 0.0, torch.float32, False),
    ("e4m3", torch.float16, 128, 8, 8, 16, WHOLE, 0.0, torch.float32, False),
    ("i8", torch.float32, 64, 40, 8, 32, WHOLE, 0.01, torch.float32, True),    # five query heads per key head
    ("e4m3", torch.float32, 64, 64, 8, 256, WHOLE, 0.0, torch.bfloat16, False),
    ("i8", torch.float16, 128, 128, 8, 16, 300, 0.0, torch.float32, False),    # sixteen
    ("e4m3", torch.float16, 128, 104, 8, 128, 300, 0.02, torch.float32, True),  # thirteen
    ("i8", torch.float32, 64, 144, 8, 64, WHOLE, 0.0, torch.float32, True),    # eighteen: two units
    ("e4m3", torch.float32, 64, 72, 4, 32, WHOLE, 0.0, torch.float16, True),
    ("i8", torch.float16, 64, 96, 8, 64, WHOLE, 0.0, torch.float16, False),    # twelve
])
def test_decode_in_ranges(kv, scale, d, heads, kvh, page, window, slope, out, track):
    _decode_of(MANY, kv, scale, d, heads, kvh, page, window, slope, out, track)


@pytest.mark.parametrize("kv,scale,d,heads,kvh,page,window,slope,out,track", [
    ("i8", torch.float16, 128, 16, 8, 32, WHOLE, 0.0, torch.float32, False), ("e4m3", torch.float32, 64, 96, 8, 16, WHOLE, 0.02, torch.bfloat16, True),
    ("e4m3", torch.float16, 128, 128, 8, 64, 40, 0.0, torch.float16, False), ("i8", torch.float32, 64, 8, 8, 16, 0, 0.0, torch.float32, True)])
def test_decode_many_short_sequences(kv, scale, d, heads, kvh, page, window, slope, out, track):
    """More units of a few tiles than CTAs of four warps would have room for."""
    _decode_of([0, 1, 2, 15, 16, 17, 97, 111] + [(s * 37) % 60 for s in range(76)], kv, scale, d, heads, kvh, page, window, slope, out, track)


@pytest.mark.parametrize("heads,kvh,lens", [(4, 2, [700, 300]), (16, 8, MANY), (12, 1, [513]), (128, 8, MANY)])
@pytest.mark.parametrize("kv", ["i8", "e4m3"])
def test_decode_logits_that_rise(heads, kvh, lens, kv):
    """Logits that rise along the cache by about 60 powers of two: the reference moves again and again, and what was summed before fades."""
    from tscale_b200 import ops
    c = Cache(20, lens, kvh, 128, 32, kv, torch.float32, False)
    q, qs = _query(20, len(lens), heads, 128, kv)
    c.k.view(torch.int8).copy_((torch.ones_like(c.k, dtype=torch.float32) * (40 if kv == "i8" else 1)).to(c.k.dtype).view(torch.int8))
    q = (torch.ones_like(q, dtype=torch.float32) * (40 if kv == "i8" else 1)).to(q.dtype)
    unit = (1600 if kv == "i8" else 1) * 128 * DOT / 128 ** 0.5
    for s, n in enumerate(lens):
        for h in range(kvh):
            c.write(c.ks, s, h, torch.linspace(-30, 30, max(n, 2), device=DEV)[:n] / unit)
    qs.fill_(1.0)
    want, _ = _decode_ref(c, q, qs, heads, WHOLE, 0.0)
    _check_out(ops.paged_decode(c.kv, c.table, c.ctx, q, qs, WHOLE, 0.0), want, c)


def test_decode_nan_and_bad_pages_in_ranges():
    from tscale_b200 import ops
    for kv in ("i8", "e4m3"):
        c = Cache(21, [300, 290], 40, 64, 16, kv, torch.float16, False)
        q, qs = _query(21, 2, 80, 64, kv)
        clean = ops.paged_decode(c.kv, c.table, c.ctx, q, qs, WHOLE, 0.0)
        p, o = c.place(0)
        for plane in (c.ks, c.vs):
            keep = plane[p[150], 7, o[150]].clone()
            for x in (float("nan"), float("inf")):
                plane[p[150], 7, o[150]] = x
                got = ops.paged_decode(c.kv, c.table, c.ctx, q, qs, WHOLE, 0.0)
                assert got[0, 14 * 64:16 * 64].isnan().any(), (kv, x)
                got[0, 14 * 64:16 * 64] = clean[0, 14 * 64:16 * 64]
                assert torch.equal(got, clean)
                assert not ops.paged_decode(c.kv, c.table, c.ctx, q, qs, 100, 0.0).isnan().any()  # in front of the window
            plane[p[150], 7, o[150]] = keep
        if kv == "e4m3":
            c.v.view(torch.uint8)[p[150], 7, o[150]] = 0x7f
            got = ops.paged_decode(c.kv, c.table, c.ctx, q, qs, WHOLE, 0.0)
            assert got[0, 14 * 64:16 * 64].isnan().all() and torch.equal(got[1], clean[1])
            assert not ops.paged_decode(c.kv, c.table, c.ctx, q, qs, 100, 0.0).isnan().any()
            c.v.view(torch.uint8)[p[150], 7, o[150]] = 0
            clean = ops.paged_decode(c.kv, c.table, c.ctx, q, qs, WHOLE, 0.0)
        for bad in (-1, c.k.shape[0], 0x7fffffff, -0x80000000):
            table = c.table.clone()
            table[1, 3] = bad
            status = torch.zeros(1, dtype=torch.int32, device=DEV)
            got = ops.paged_decode(c.kv, table, c.ctx, q, qs, WHOLE, 0.0, status=status)
            assert int(status) != 0 and got.isfinite().all() and torch.equal(got[0], clean[0])
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        got = ops.paged_decode(c.kv, c.table, c.ctx, q, qs, WHOLE, 0.0, max_ctx=295, status=status)
        assert int(status) != 0 and not got[0].any() and float((got[1] - clean[1]).abs().max()) <= 2 * ERR * 128 * 1.5 * _unit(kv)


def test_decode_sums_of_a_very_long_cache():
    """Some 60 million equal keys, 1050 tiles of 128 a range, all digits of the weights and all codes at their largest: int32 sums that
    have to be emptied on the way."""
    from tscale_b200 import ops
    n = 444 * 1050 * 128
    pages = n // 256 + 1
    shape = (pages, 1, 256)
    k, v = torch.zeros(shape + (64,), dtype=torch.int8, device=DEV), torch.full(shape + (64,), 127, dtype=torch.int8, device=DEV)
    scale = 0x7f7f7f / 2.0 ** 22
    kv = ops.PagedKV(k, v, torch.ones(shape, device=DEV), torch.full(shape, scale, device=DEV))
    ctx = torch.tensor([n + 1], dtype=torch.int32, device=DEV)
    q = torch.ones((1, 128), dtype=torch.int8, device=DEV)
    got = ops.paged_decode(kv, torch.arange(pages, dtype=torch.int32, device=DEV)[None], ctx, q, None, WHOLE, 0.0)
    want = scale * 127 * n / (n + 1)
    # a range's sums are integers below 2^24 or one rounding off; the join adds 444 records: fewer than 512 roundings of 2^-24
    assert float((got.double() - want).abs().max()) <= 2.0 ** -15 * want


@pytest.mark.parametrize("kv,lens,heads,kvh,d,page,track", [("i8", [20011, 3, 9999], 8, 2, 128, 64, False), ("e4m3", [30000], 3, 1, 64, 16, True),
                                                            ("i8", [5000] + [40] * 30, 4, 4, 64, 32, False)])
def test_decode_split_over_long_caches(kv, lens, heads, kvh, d, page, track):
    from tscale_b200 import ops
    c = Cache(2, lens, kvh, d, page, kv, torch.float16, track)
    q, qs = _query(2, len(lens), heads, d, kv)
    before = None if c.weight is None else c.weight.clone()
    want, added = _decode_ref(c, q, qs, heads, WHOLE, 0.0)
    got = ops.paged_decode(c.kv, c.table, c.ctx, q, qs, WHOLE, 0.0, max_ctx=max(lens), tokens=c.tokens)
    _check_out(got, want, c)
    if track:
        p, o = c.place(0)
        for h in range(kvh):
            assert float((c.weight[p, h, o].double() - before[p, h, o].double() - added[0, h]).abs().max()) <= ERR * (heads // kvh) + 2.0 ** -23


@pytest.mark.parametrize("kv,scale,d,heads,kvh,page", [("i8", torch.float16, 64, 4, 2, 32), ("e4m3", torch.float32, 128, 6, 1, 128), ("i8", torch.float32, 128, 24, 2, 16),
                                                       ("e4m3", torch.float16, 64, 40, 2, 256), ("i8", torch.float16, 64, 16, 1, 64)])
@pytest.mark.parametrize("window,ordered,slope", [(30, False, 0.0), (0, False, 0.0), (1000, True, 0.02), (5000, False, 0.0), (30, True, 0.5), (700, False, 0.01)])
def test_decode_windows_of_long_caches_with_positions(kv, scale, d, heads, kvh, page, window, ordered, slope):
    """Most tiles have no key inside the window, some key heads none at all."""
    from tscale_b200 import ops
    lens = [6000, 1, 9000, 0, 140, 20000]
    c = Cache(21, lens, kvh, d, page, kv, scale, True)
    for s, n in enumerate(lens):
        for h in range(kvh):
            if ordered and n:
                c.write(c.pos, s, h, c.read(c.pos, s, h).sort().values.to(torch.int32))
    p, o = c.place(2)
    c.pos[p, kvh - 1, o] = 0  # nothing in the window of the last key head
    q, qs = _query(21, len(lens), heads, d, kv)
    before = c.weight.clone()
    want, added = _decode_ref(c, q, qs, heads, window, slope)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = ops.paged_decode(c.kv, c.table, c.ctx, q, qs, window, slope, max_ctx=max(lens), tokens=c.tokens, status=status)
    assert int(status) == 0
    _check_out(got, want, c)
    # without the weights, into another type, and the same again
    plain = c.kv._replace(weight=None)
    runs = [ops.paged_decode(plain, c.table, c.ctx, q, qs, window, slope, max_ctx=max(lens), tokens=c.tokens, out_dtype=torch.bfloat16) for _ in range(2)]
    assert torch.equal(*runs)
    _check_out(runs[0], want, c)
    for (s, h), w in added.items():
        p, o = c.place(s)
        assert float((c.weight[p, h, o].double() - before[p, h, o].double() - w).abs().max()) <= ERR * (heads // kvh) + 2.0 ** -23
    # a page outside the pool is reported from a tile that nobody needs, too
    c.table[5, 3] = 1 << 20
    ops.paged_decode(c.kv, c.table, c.ctx, q, qs, 30, 0.0, max_ctx=max(lens), tokens=c.tokens, status=status)
    assert int(status) != 0


def test_decode_positions_that_repeat():
    """More keys inside the window than it has positions: reported, and the others of the batch are right."""
    from tscale_b200 import ops
    c = Cache(22, [5000, 3000], 1, 64, 64, "i8", torch.float16, True)
    q, qs = _query(22, 2, 4, 64, "i8")
    want, added = _decode_ref(c, q, qs, 4, 100, 0.0)
    p, o = c.place(0)
    c.pos[p, 0, o] = int(c.tokens[0]) - 5
    before = c.weight.clone()
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = ops.paged_decode(c.kv, c.table, c.ctx, q, qs, 100, 0.0, max_ctx=5000, tokens=c.tokens, status=status)
    assert int(status) != 0
    c.lens[0] = 0
    _check_out(got[1:], want[1:], c)
    p, o = c.place(1)
    assert float((c.weight[p, 0, o].double() - before[p, 0, o].double() - added[1, 0]).abs().max()) <= 4 * ERR + 2.0 ** -23


def test_decode_no_key_inside_the_window_and_no_query_scale():
    from tscale_b200 import ops
    c = Cache(3, [300, 40], 2, 64, 32, "e4m3", torch.float16, True)
    q, _ = _query(3, 2, 4, 64, "e4m3")
    c.pos.fill_(5)
    assert not ops.paged_decode(c.kv, c.table, c.ctx, q, None, 10, 0.0, tokens=c.tokens).any()
    c = Cache(3, [300, 40], 2, 64, 32, "i8", torch.float16, False)
    q, qs = _query(3, 2, 4, 64, "i8")
    want, _ = _decode_ref(c, q, torch.full_like(qs, 0.025), 4, WHOLE, 0.0)
    _check_out(ops.paged_decode(c.kv, c.table, c.ctx, q, None, WHOLE, 0.0, vec_scale=0.025), want, c)


def test_decode_scales_of_any_size():
    """Value scales over many powers of two, zero and negative ones; logits far from zero on both sides."""
    from tscale_b200 import ops
    c = Cache(4, [400, 37, 64], 2, 128, 16, "i8", torch.float32, False)
    q, qs = _query(4, 3, 4, 128, "i8")
    gen = _gen(4)
    c.vs.copy_(torch.exp2(torch.rand(c.vs.shape, generator=gen, device=DEV) * 60 - 50) * torch.where(torch.rand(c.vs.shape, generator=gen, device=DEV) < 0.3, -1.0, 1.0))
    c.vs[torch.rand(c.vs.shape, generator=gen, device=DEV) < 0.2] = 0.0
    want, _ = _decode_ref(c, q, qs, 4, WHOLE, 0.0)
    _check_out(ops.paged_decode(c.kv, c.table, c.ctx, q, qs, WHOLE, 0.0), want, c)
    c.vs.fill_(2.0 ** -70)  # all small: nothing is lost
    want, _ = _decode_ref(c, q, qs, 4, WHOLE, 0.0)
    _check_out(ops.paged_decode(c.kv, c.table, c.ctx, q, qs, WHOLE, 0.0), want, c)


@pytest.mark.parametrize("kv", ["i8", "e4m3"])
def test_decode_values_that_are_all_zero(kv):
    """Four million keys of value scale zero, the logits of every other tile higher by 7.9: nothing to add up, but their weights count."""
    from tscale_b200 import ops
    n = 444 * 80 * 128
    shape = (n // 256 + 1, 1, 256)
    codes = [torch.ones(shape + (64,), device=DEV).to(CODES[kv]) for _ in range(2)]
    ks = torch.full(shape, 50.0 / 8 / DOT, device=DEV)
    ks[:, :, 128:] = 57.9 / 8 / DOT
    cache = ops.PagedKV(*codes, ks, torch.zeros(shape, device=DEV), None, torch.zeros(shape, device=DEV))
    table, ctx = torch.arange(shape[0], dtype=torch.int32, device=DEV)[None], torch.tensor([n + 1], dtype=torch.int32, device=DEV)
    got = ops.paged_decode(cache, table, ctx, torch.ones((1, 128), device=DEV).to(CODES[kv]), None, WHOLE, 0.0)
    assert not got.any()
    # The heavier half has weight 2 / (n / 2 * (1 + 2^-7.9)) for two heads; the sink, 2^-57, is below all roundings.  Exponents: z - reference
    # and the logarithm of the sum are below 129, each half a step of 2^-16 off, the results of three more additions less than that again; times
    # ln 2 that is below 2^-15.  Sums: 80 + 8 + 444 additions of 2^-24.  The lighter half's own logits count 2^-7.9 times
    w = cache.weight.view(-1)[:n].view(-1, 256)
    assert float((w[:, 128:].double() * (n / 4 * (1 + 2 ** -7.9)) - 1).abs().max()) <= 2.0 ** -14 + 2.0 ** -15
    assert float((w[:, :128].double() * (n / 4 * (1 + 2 ** 7.9)) - 1).abs().max()) <= 2.0 ** -13


def test_decode_nan_and_infinity_stay_where_they_are():
    from tscale_b200 import ops
    c = Cache(5, [200, 90], 2, 64, 16, "e4m3", torch.float16, False)
    q, qs = _query(5, 2, 4, 64, "e4m3")
    clean = ops.paged_decode(c.kv, c.table, c.ctx, q, qs, WHOLE, 0.0)
    p, o = c.place(0)
    c.ks[p[150], 1, o[150]] = float("nan")
    got = ops.paged_decode(c.kv, c.table, c.ctx, q, qs, WHOLE, 0.0)
    assert got[0, 128:].isnan().all() and torch.equal(got[0, :128], clean[0, :128]) and torch.equal(got[1], clean[1])
    c.ks[p[150], 1, o[150]] = 0.5
    for plane, x in ((c.ks, float("inf")), (c.vs, float("nan")), (c.vs, float("inf"))):
        keep = plane[p[10], 0, o[10]].clone()
        plane[p[10], 0, o[10]] = x  # in front of the window: not attended
        got = ops.paged_decode(c.kv, c.table, c.ctx, q, qs, 100, 0.0)
        assert not got.isnan().any()
        plane[p[10], 0, o[10]] = keep


def test_decode_pages_outside_the_pool_and_sequences_beyond_the_bound():
    from tscale_b200 import ops
    c = Cache(6, [100, 200, 300], 2, 64, 16, "i8", torch.float16, False)
    q, qs = _query(6, 3, 2, 64, "i8")
    clean = ops.paged_decode(c.kv, c.table, c.ctx, q, qs, WHOLE, 0.0)
    for bad in (-1, c.k.shape[0], 0x7fffffff, -0x80000000):
        table = c.table.clone()
        table[1, 3] = bad
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        got = ops.paged_decode(c.kv, table, c.ctx, q, qs, WHOLE, 0.0, status=status)
        assert int(status) != 0 and got.isfinite().all() and torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])
    for ctx, bound in (([100, 200, 300], 250), ([100, 200, 16 * c.table.shape[1] + 1], None)):
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        got = ops.paged_decode(c.kv, c.table, torch.tensor(ctx, dtype=torch.int32, device=DEV), q, qs, WHOLE, 0.0, max_ctx=bound, status=status)
        assert int(status) != 0 and not got[2].any()
        big = float((clean[:2] - got[:2]).abs().max())
        assert big <= 2 * ERR * 127 * 1.5 / 40


def test_decode_strided_rows_given_output_and_workspace():
    from tscale_b200 import ops
    c = Cache(7, [100, 50], 2, 64, 16, "i8", torch.float16, False, max_pages=20)
    q, qs = _query(7, 2, 4, 64, "i8")
    want = ops.paged_decode(c.kv, c.table, c.ctx, q, qs, WHOLE, 0.0)
    wide_q, wide_s, wide_t = torch.zeros((2, 512), dtype=torch.int8, device=DEV), torch.zeros((2, 9), device=DEV), torch.full((2, 31), 7, dtype=torch.int32, device=DEV)
    wide_q[:, 128:384], wide_s[:, 3:7], wide_t[:, 5:25] = q, qs, c.table
    out = torch.full((4, 300), 3.0, device=DEV)
    got = ops.paged_decode(c.kv, wide_t[:, 5:25], c.ctx, wide_q[:, 128:384], wide_s[:, 3:7], WHOLE, 0.0, out=out[1:3, 4:260],
                           workspace=torch.empty(1 << 22, dtype=torch.uint8, device=DEV))
    assert got.data_ptr() == out[1:3, 4:].data_ptr() and torch.equal(got, want)
    out[1:3, 4:260] = 3.0
    assert (out == 3.0).all()


def test_decode_equals_the_contiguous_cache():
    from tscale_b200 import ops
    lens, heads, d = [700, 1, 257], 4, 128
    c = Cache(8, lens, heads, d, 64, "i8", torch.float16, False)
    q, qs = _query(8, 3, heads, d, "i8")
    flat = ops.KVCache(3, 700, heads, d, DEV)
    for s, n in enumerate(lens):
        p, o = c.place(s)
        flat.k[s, :n], flat.v[s, :n] = c.k[p, :, o].reshape(n, -1), c.v[p, :, o].reshape(n, -1)
        flat.k_scale[s, :n], flat.v_scale[s, :n] = c.ks[p, :, o], c.vs[p, :, o]
    flat.ctx_lens.copy_(c.ctx)
    flat.max_ctx = 700
    for window, slope in ((WHOLE, 0.0), (64, 0.5), (0, 0.0)):
        a, b = flat.decode(q, qs, window, slope), ops.paged_decode(c.kv, c.table, c.ctx, q, qs, window, slope)
        assert float((a - b).abs().max()) <= 2 * ERR * 128 * 1.5 / 40


def _append_ref(c, counts, k, ks, v, vs, starts):
    planes = [x.clone() for x in (c.k.view(torch.int8), c.v.view(torch.int8), c.ks, c.vs)] + [None if x is None else x.clone() for x in (c.pos, c.weight)]
    for s, n in enumerate(counts):
        for i in range(n):
            slot, row = c.lens[s] - n + i, starts[s] + i
            p, o = int(c.table[s, slot // c.page]), slot % c.page
            planes[0][p, :, o] = k.view(torch.int8)[row].view(c.kvh, c.d)
            planes[1][p, :, o] = v.view(torch.int8)[row].view(c.kvh, c.d)
            planes[2][p, :, o], planes[3][p, :, o] = ks[:, row].to(c.ks.dtype), vs[:, row].to(c.vs.dtype)
            if c.pos is not None:
                planes[4][p, :, o] = int(c.tokens[s]) - n + i
                planes[5][p, :, o] = 0.0
    return planes


def _same(a, b):
    return a is None or torch.equal(a.view(torch.uint8) if a.dtype != torch.float8_e4m3fn else a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("kv,scale,kvh,d,page,counts,track", [
    ("i8", torch.float16, 4, 128, 64, [1] * 7, False), ("e4m3", torch.float32, 3, 64, 16, [0, 5, 0, 0, 33, 1, 100, 0], True),
    ("i8", torch.float32, 16, 128, 32, [17], True), ("e4m3", torch.float16, 1, 64, 256, [0, 0, 300, 0], False), ("i8", torch.float16, 40, 64, 16, [3, 2], True)])
@pytest.mark.parametrize("lead", [0, 5])
def test_append(kv, scale, kvh, d, page, counts, track, lead):
    from tscale_b200 import ops
    lens = [n + (13 * s) % 40 for s, n in enumerate(counts)]
    c = Cache(9, lens, kvh, d, page, kv, scale, track)
    gen = _gen(9)
    rows = lead + sum(counts) + (3 if lead else 0)  # rows of no sequence in front and behind
    k, v = (_codes((rows, kvh * d + 32), kv, gen)[:, 16:-16] for _ in range(2))
    ks, vs = (torch.rand((kvh, rows + 3), generator=gen, device=DEV)[:, :rows] for _ in range(2))
    starts = [lead]
    for n in counts:
        starts.append(starts[-1] + n)
    want = _append_ref(c, counts, k, ks, v, vs, starts)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ones = counts == [1] * len(counts) and not lead
    ops.paged_append(c.kv, c.table, c.ctx, k, ks, v, vs, None if ones else torch.tensor(starts, dtype=torch.int32, device=DEV), c.tokens, status)
    assert int(status) == 0
    assert all(_same(a, b) for a, b in zip((c.k.view(torch.int8), c.v.view(torch.int8), c.ks, c.vs, c.pos, c.weight), want))


@pytest.mark.parametrize("n,kvh,d", [(1500, 1, 64), (2500, 3, 64), (2500, 5, 128)])
def test_append_many_sequences(n, kvh, d):
    from tscale_b200 import ops
    counts = [(s * 7919) % 5 for s in range(n)]
    c = Cache(10, [m + s % 3 for s, m in enumerate(counts)], kvh, d, 16, "i8", torch.float16, False)
    gen, rows = _gen(10), sum(counts)
    k, v = _codes((rows, kvh * d), "i8", gen), _codes((rows, kvh * d), "i8", gen)
    ks, vs = torch.rand((kvh, rows), generator=gen, device=DEV), torch.rand((kvh, rows), generator=gen, device=DEV)
    starts = np.concatenate([[0], np.cumsum(counts)])
    slot = np.concatenate([np.arange(c.lens[s] - m, c.lens[s]) for s, m in enumerate(counts)])
    seq = np.repeat(np.arange(n), counts)
    ops.paged_append(c.kv, c.table, c.ctx, k, ks, v, vs, torch.tensor(starts, dtype=torch.int32, device=DEV))
    page = c.table[torch.from_numpy(seq).to(DEV), torch.from_numpy(slot // 16).to(DEV)].long()
    off = torch.from_numpy(slot % 16).to(DEV)
    for h in range(kvh):
        assert torch.equal(c.k[page, h, off], k[:, h * d:(h + 1) * d]) and torch.equal(c.v[page, h, off], v[:, h * d:(h + 1) * d])
        assert torch.equal(c.ks[page, h, off], ks[h].half()) and torch.equal(c.vs[page, h, off], vs[h].half())


def test_append_places_that_do_not_exist():
    from tscale_b200 import ops
    c = Cache(11, [20, 20, 20], 2, 64, 16, "i8", torch.float16, False)
    gen = _gen(11)
    k, ks = _codes((6, 128), "i8", gen), torch.rand((2, 6), generator=gen, device=DEV)
    for ctx, bad in (([20, 1, 20], None), ([20, 20, 40], None), ([20, 20, 20], -1), ([20, 20, 20], c.k.shape[0])):
        before = [x.clone() for x in c.kv[:4]]
        table = c.table.clone()
        if bad is not None:
            table[1, 1] = bad
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        ops.paged_append(c.kv, table, torch.tensor(ctx, dtype=torch.int32, device=DEV), k, ks, k, ks,
                         torch.tensor([0, 2, 4, 6], dtype=torch.int32, device=DEV), status=status)
        assert int(status) != 0
        changed = (c.k != before[0]).any(-1).any(1).sum()
        assert int(changed) <= 5
        for x, b in zip(c.kv[:4], before):
            x.copy_(b)


def _select_ref(w, pos, n, newest, keep, recent):
    if n <= keep:
        return [], n
    key = [(1, 0.0) if pos[i] > newest - recent else (0, float(w[i])) for i in range(n)]
    order = sorted(range(n), key=lambda i: (-key[i][0], 0 if key[i][0] or key[i][1] != key[i][1] else 1, 0.0 if key[i][1] != key[i][1] else -key[i][1], i))
    kept = set(order[:keep])
    holes = [i for i in range(keep) if i not in kept]
    movers = [i for i in range(keep, n) if i in kept]
    return list(zip(holes, movers)), keep


@pytest.mark.parametrize("lens,kvh,page,keep,recent,positions,values", [
    ([0, 1, 31, 32, 33, 500, 1500], 3, 16, 32, 4, True, "smooth"), ([700, 100], 2, 64, 99, 0, True, "few"), ([5000, 4097], 1, 256, 4096, 4096, True, "zeros"),
    ([3000, 900], 2, 32, 1000, 7, False, "special"), ([2049], 1, 16, 1, 1, True, "smooth"), ([1025, 1024], 1, 32, 1024, 100, True, "few"),
    ([40000], 1, 64, 5000, 64, True, "few"), ([30000, 100000], 1, 16, 70001, 0, True, "few"),
    ([60000] + [10] * 24, 12, 64, 5000, 8, True, "few"),
    ([400000, 260001], 1, 256, 9000, 100, True, "smooth"), ([750000], 1, 256, 5000, 8, False, "few")])  # the last: more than sixteen CTAs' shared memory holds
def test_select(lens, kvh, page, keep, recent, positions, values):
    from tscale_b200 import ops
    c = Cache(12, lens, kvh, 64, page, "i8", torch.float16, True)
    gen = _gen(12)
    if not positions:
        c.kv, c.tokens = c.kv._replace(pos=None), None
    if values == "few":
        c.weight.copy_(torch.randint(0, 4, c.weight.shape, generator=gen, device=DEV))
    elif values == "zeros":
        c.weight.zero_()
    elif values == "special":
        some = torch.tensor([0.0, -0.0, float("inf"), float("nan"), 1e-40, -1.0, 2.0, -float("inf")], device=DEV)
        c.weight.copy_(some[torch.randint(0, 8, c.weight.shape, generator=gen, device=DEV)])
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    moves, counts, new = ops.paged_evict_select(c.kv, c.table, c.ctx, keep, recent, max_ctx=max(lens), tokens=c.tokens, status=status)
    assert int(status) == 0 and moves.shape[2] == max(1, min(keep, max(lens) - keep))
    for s, n in enumerate(lens):
        newest = (n if c.tokens is None else int(c.tokens[s])) - 1
        for h in range(kvh):
            w = c.read(c.weight, s, h).tolist() if n else []
            pos = list(range(n)) if not positions else c.read(c.pos, s, h).tolist() if n else []
            want, length = _select_ref(w, pos, n, newest, keep, recent)
            assert int(counts[s, h]) == len(want) and int(new[s]) == length
            assert moves[s, h].tolist() == [list(m) for m in want] + [[-1, -1]] * (moves.shape[2] - len(want))


def test_select_in_two_threads():
    """Calls of different sizes at once: the launch of each finds the shared memory it asks for."""
    import threading
    from tscale_b200 import ops
    jobs, wrong = [], []
    for seed, (n, length) in enumerate([(200, 12000), (2, 5000), (1, 70000)]):
        pages = n * -(-length // 64)
        weight = torch.rand((pages, 1, 64), generator=_gen(seed), device=DEV)
        table = torch.arange(pages, dtype=torch.int32, device=DEV).view(n, -1)
        kv = ops.PagedKV(None, None, None, None, None, weight)
        call = lambda kv=kv, table=table, ctx=torch.full((n,), length, dtype=torch.int32, device=DEV): ops.paged_evict_select(kv, table, ctx, 900, 10)  # noqa: E731
        jobs.append((call, call()))

    def work(call, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(150):
                    got = call()
                torch.cuda.current_stream().synchronize()
                assert all(torch.equal(a, b) for a, b in zip(got, want))
        except Exception as e:
            wrong.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=jobs[i % 3]) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[0]


@pytest.mark.parametrize("kv,scale,kvh,d,page,track", [("i8", torch.float16, 3, 128, 16, True), ("e4m3", torch.float32, 2, 64, 64, True),
                                                       ("i8", torch.float32, 1, 128, 32, False)])
def test_move(kv, scale, kvh, d, page, track):
    from tscale_b200 import ops
    lens, keep = [300, 120, 90, 0], 100
    c = Cache(13, lens, kvh, d, page, kv, scale, track)
    cap = 150
    moves = torch.full((4, kvh, cap, 2), -1, dtype=torch.int32)
    counts = torch.zeros((4, kvh), dtype=torch.int32)
    rng = np.random.default_rng(13)
    for s in (0, 1):
        for h in range(kvh):
            n = rng.integers(1, min(keep, lens[s] - keep) + 1)
            counts[s, h] = int(n)
            moves[s, h, :n, 0] = torch.from_numpy(np.sort(rng.permutation(keep)[:n]))
            moves[s, h, :n, 1] = torch.from_numpy(np.sort(keep + rng.permutation(lens[s] - keep)[:n]))
    moves[2, 0, 0] = torch.tensor([5, 80])  # not counted: not moved
    planes = [None if x is None else (x.view(torch.int8) if x.element_size() == 1 else x) for x in c.kv]
    want = [None if x is None else x.clone() for x in planes]
    for s in (0, 1):
        for h in range(kvh):
            m = moves[s, h, :int(counts[s, h])].long().to(DEV)
            dp, do, sp, so = c.table[s].long()[m[:, 0] // page], m[:, 0] % page, c.table[s].long()[m[:, 1] // page], m[:, 1] % page
            for x, y in zip(planes, want):
                if x is not None:
                    y[dp, h, do] = x[sp, h, so]
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    for _ in range(2):  # a second time changes nothing
        ops.paged_evict_move(c.kv, c.table, moves.to(DEV), counts.to(DEV), status)
        assert int(status) == 0 and all(_same(a, b) for a, b in zip(planes, want))
    moves[0, 0, 0] = torch.tensor([-1, 200])
    moves[0, 0, 1] = torch.tensor([3, 1 << 30])
    ops.paged_evict_move(c.kv, c.table, moves.to(DEV), counts.to(DEV), status)
    assert int(status) != 0 and all(_same(a, b) for a, b in zip(planes, want))


def test_pools_beyond_four_gigabytes():
    """Pages whose bytes lie behind 2^32: append, decode and moves."""
    from tscale_b200 import ops
    kvh, d, page = 2, 128, 256
    pages = (1 << 32) // (kvh * d * page) + 8
    k, v = (torch.zeros((pages, kvh, page, d), dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.full((pages, kvh, page), 1 / 40.0, dtype=torch.float16, device=DEV) for _ in range(2))
    kv = ops.PagedKV(k, v, ks, vs, torch.zeros((pages, kvh, page), dtype=torch.int32, device=DEV), torch.zeros((pages, kvh, page), device=DEV))
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device=DEV)
    n, gen = 600, _gen(14)
    ctx = torch.tensor([n], dtype=torch.int32, device=DEV)
    kn, vn = _codes((n, kvh * d), "i8", gen), _codes((n, kvh * d), "i8", gen)
    sn = (torch.rand((kvh, n), generator=gen, device=DEV) + 0.5) / 40
    ops.paged_append(kv, table, ctx, kn, sn, vn, sn, torch.tensor([0, n], dtype=torch.int32, device=DEV), ctx)
    assert torch.equal(k[pages - 1].transpose(0, 1).reshape(page, -1), kn[:256]) and torch.equal(v[pages - 2, :, :88].transpose(0, 1).reshape(88, -1), vn[512:])
    assert not k[0].any() and not k[pages - 3].any()
    q, qs = _query(14, 1, 4, d, "i8")
    small = Cache(14, [n], kvh, d, page, "i8", torch.float16, True)
    for a, b in ((small.k, k), (small.v, v), (small.ks, ks), (small.vs, vs), (small.pos, kv.pos)):
        a[small.table[0].long()] = b[table[0].long()]
    small.tokens = ctx
    want, _ = _decode_ref(small, q, qs, 4, WHOLE, 0.0)
    _check_out(ops.paged_decode(kv, table, ctx, q, qs, WHOLE, 0.0, tokens=ctx), want, small)
    moves, counts, new = ops.paged_evict_select(kv, table, ctx, 256, 16, tokens=ctx)
    ops.paged_evict_move(kv, table, moves, counts)
    for h in range(kvh):
        m = moves[0, h, :int(counts[0, h])].long()
        assert int(counts[0, h]) > 10 and torch.equal(k[pages - 1, h, m[:, 0]], kn.view(n, kvh, d)[m[:, 1], h])


def test_captured_calls_replay_and_streams_do_not_share_scratch():
    from tscale_b200 import ops
    cache = ops.PagedKVCache(3, 60, 2, 64, DEV, page_size=16, max_pages=20)
    gen = _gen(15)
    new = lambda rows: (_codes((rows, 128), "i8", gen), (torch.rand((2, rows), generator=gen, device=DEV) + 0.5) / 40,  # noqa: E731
                        _codes((rows, 128), "i8", gen), (torch.rand((2, rows), generator=gen, device=DEV) + 0.5) / 40)
    cache.append(*new(330), row_starts=cache.extend([200, 100, 30]))
    q, qs = _query(15, 3, 4, 64, "i8")
    step = new(3)
    side = torch.cuda.Stream()
    graphs = []
    cache.extend()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):  # two graphs of the same calls
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                cache.append(*step)
                out = cache.decode(q, qs, WHOLE, 0.0, max_ctx=320)
            graphs.append((graph, out))
    torch.cuda.current_stream().wait_stream(side)
    for i in range(6):
        if i:
            cache.extend()
            for x in step:
                x.copy_(x.flip(0))
        graph, out = graphs[i % 2]
        graph.replay()
        got = out.clone()
        cache.append(*step)
        want = cache.decode(q, qs, WHOLE, 0.0, max_ctx=320)
        assert torch.equal(got, want), i
    # the same on two streams at once
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(cache.decode(q if i % 2 else q.neg(), qs, WHOLE, 0.0, max_ctx=320))
    torch.cuda.synchronize()
    assert all(torch.equal(o, outs[i % 2]) for i, o in enumerate(outs)) and not torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("kv,d,heads,kvh,page", [("i8", 128, 4, 2, 16), ("e4m3", 64, 6, 6, 32)])
def test_a_cache_that_is_filled_read_and_cut(kv, d, heads, kvh, page):
    """Prompts, single tokens, evictions, a sequence that ends and another in its place, against lists of tokens per key head."""
    from tscale_b200 import ops
    n_seq, group = 3, heads // kvh
    cache = ops.PagedKVCache(n_seq, 40, kvh, d, DEV, page_size=page, max_pages=24, kv_dtype=kv, scale_dtype=torch.float32, evict=True)
    gen = _gen(16)
    model = [[[] for _ in range(kvh)] for _ in range(n_seq)]  # of (position, k, v)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)

    def feed(counts):
        rows = sum(counts)
        k, v = _codes((rows, kvh * d), kv, gen), _codes((rows, kvh * d), kv, gen)
        ks, vs = ((torch.rand((kvh, rows), generator=gen, device=DEV) + 0.5) * _unit(kv) for _ in range(2))
        at = 0
        for s, n in enumerate(counts):
            for i in range(n):
                for h in range(kvh):
                    model[s][h].append((int(cache.seen[s]) + i, k[at + i, h * d:(h + 1) * d].double() * ks[h, at + i].double(),
                                        v[at + i, h * d:(h + 1) * d].double() * vs[h, at + i].double()))
            at += n
        cache.append(k, ks, v, vs, cache.extend(counts), status)

    def step(window, slope):
        q, qs = _query(int(cache.seen.sum()), n_seq, heads, d, kv)
        got = cache.decode(q, qs, window, slope, status=status)
        big, want = 1e-6, torch.zeros((n_seq, heads, d), dtype=torch.float64, device=DEV)
        for s in range(n_seq):
            for h in range(kvh):
                cur = int(cache.seen[s]) - 1
                seen = [x for x in model[s][h] if 1 <= cur - x[0] <= window]
                if seen:
                    k, v = torch.stack([x[1] for x in seen]), torch.stack([x[2] for x in seen])
                    far = torch.tensor([float(cur - x[0]) for x in seen], dtype=torch.float64, device=DEV)
                    qh = (q[s].view(heads, d).double() * qs[s].double()[:, None])[h * group:(h + 1) * group]
                    w = torch.exp2(qh @ k.T * (DOT / d ** 0.5) - slope * far)
                    want[s, h * group:(h + 1) * group] = w / (1 + w.sum(1, keepdim=True)) @ v
                    big = max(big, float(v.abs().max()))
        assert float((got.double() - want.view(n_seq, -1)).abs().max()) <= ERR * big

    def cut(keep, recent):
        old = []
        for s in range(n_seq):
            n = int(cache.lens[s])
            t = torch.arange(n, device=DEV)
            p = cache.page_table[s].long()[t // page]
            old.append([(cache.kv.weight[p, h, t % page].tolist(), cache.kv.pos[p, h, t % page].tolist()) for h in range(kvh)])
        cache.evict(keep, recent, status)
        for s in range(n_seq):
            for h in range(kvh):
                w, pos = old[s][h]
                n = len(w)
                assert sorted(pos) == sorted(x[0] for x in model[s][h])
                if n > keep:
                    moves, _ = _select_ref(w, pos, n, int(cache.seen[s]) - 1, keep, recent)
                    slots = list(range(keep))
                    for to, of in moves:
                        slots[to] = of
                    stay = {pos[i] for i in slots}
                    model[s][h] = [x for x in model[s][h] if x[0] in stay]
                    assert len(model[s][h]) == keep

    feed([100, 37, 0])
    step(WHOLE, 0.0)
    feed([1, 1, 1])
    step(WHOLE, 0.01)
    feed([50, 1, 3])
    step(64, 0.0)
    cut(60, 8)
    assert len(cache.free) == 40 - sum(-(-int(n) // page) for n in cache.lens)
    for _ in range(3):
        feed([1, 1, 1])
        step(WHOLE, 0.0)
    cut(33, 1)
    cut(33, 0)
    cache.release(1)
    for h in range(kvh):
        model[1][h] = []
    feed([20, 90, 1])
    step(1000, 0.0)
    cut(17, 17)
    step(WHOLE, 0.0)
    assert int(status) == 0 and sorted(cache.free + cache.page_table[cache.page_table >= 0].tolist()) == list(range(40))


def test_prompt_from_the_producers_into_pages():
    """The int8 producers' outputs go into the cache as they are: keys with their planes, queries of the newest token."""
    from tscale_b200 import ops
    heads, d, rows = 4, 64, 150
    gen = _gen(17)
    x = torch.randn((rows, 256), generator=gen, device=DEV)
    x8, _ = ops.quant_rows(x, "rms", "i8", 64, vec_scale=1 / 24.0)
    w = torch.randint(-127, 128, (3 * heads * d, 256), generator=gen, device=DEV, dtype=torch.int8)
    kk, ks = ops.matmul_norm_rope_quant(x8.view(torch.int8), w[:heads * d], None, "i8", heads, d, vec_scale=1 / 24.0)
    vv, vs = ops.matmul_norm_rope_quant(x8.view(torch.int8), w[heads * d:2 * heads * d], None, "i8", heads, d, vec_scale=1 / 24.0)
    qq, _ = ops.matmul_norm_rope_quant(x8.view(torch.int8), w[2 * heads * d:], None, "i8", heads, d, vec_scale=1 / 24.0)
    ks, vs = ks / ks.mean() / 24, vs / vs.mean() / 24
    cache = ops.PagedKVCache(2, 12, heads, d, DEV, page_size=16, max_pages=10, qk_vec_scale=1 / 24.0)
    k8, v8, q8 = (t.view(torch.int8) for t in (kk, vv, qq))
    cache.append(k8, ks, v8, vs, cache.extend([100, 50]))
    got = cache.decode(torch.stack([q8[99], q8[149]]), None, WHOLE, 0.0)
    for s, (a, b) in enumerate(((0, 100), (100, 150))):
        for h in range(heads):
            col = slice(h * d, (h + 1) * d)
            k = k8[a:b - 1, col].double() * ks[h, a:b - 1].half().double()[:, None]
            v = v8[a:b - 1, col].double() * vs[h, a:b - 1].half().double()[:, None]
            p = torch.exp2(k @ (q8[b - 1, col].double() / 24) * (DOT / d ** 0.5))
            want = p @ v / (1 + p.sum())
            assert float((got[s, col].double() - want).abs().max()) <= ERR * float(v.abs().max())
