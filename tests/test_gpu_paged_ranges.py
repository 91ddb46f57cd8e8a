"""GPU tests of the paged decode in ranges (long caches and many units), every call of which is checked to take that form.

Tolerances, beside those of test_gpu_paged: a range's weights are fixed numbers of four 8-bit digits.  int8: 2^-28 of 2^ref off at most, 2048 keys
to a reference and a key of 2^ref / 2 or more among them, so that all keys together are off by 2^-16 of the sum of the weights times the largest value.
e4m3: half of that, and 2^-16 of each weight itself.  Logits (5e-6 of a weight) and float32 sums (two roundings for 2048 keys of a range, one for each range
of a unit, 2^-24 of a weight each, 2^-17 for 128 of them) come on top: 2^-15 of the sum of weights times values.
"""
import ctypes

import pytest
import torch

from tests.test_gpu_paged import CODES, DEV, DOT, WHOLE, _gen

pytestmark = pytest.mark.gpu


def _needs_workspace(kv, n_seq, heads, max_ctx, window=WHOLE):
    """Bytes of scratch that the call asks for; the form in ranges is the one that asks for any."""
    from tscale_b200 import abi
    k, scale = kv[0], kv[2]
    cfg = abi.PagedCfg(k.shape[3], abi.TSA_I8 if k.dtype == torch.int8 else abi.TSA_E4M3, abi.TSA_F16 if scale.dtype == torch.float16 else abi.TSA_F32, abi.TSA_F32, 1.0)
    pools = abi.PagedKv(*(None if x is None else x.data_ptr() for x in kv), k.shape[0], k.shape[2], k.shape[1])
    size = abi.lib().tsa_paged_decode_workspace_bytes(ctypes.byref(cfg), ctypes.byref(pools), n_seq, heads, max_ctx, window)
    assert size > 0
    return size


@pytest.mark.parametrize("kv", ["i8", "e4m3"])
@pytest.mark.parametrize("d,group", [(64, 1), (64, 7), (64, 12), (128, 3), (128, 8), (128, 16)])
@pytest.mark.parametrize("logits", ["first", "middle", "last", "spread", "falls"])
def test_one_heavy_key_among_very_many_light_ones(kv, d, group, logits):
    """All sequences have the same pages, and a range holds a unit or more: keys of 2^-22 to 2^-33 of the heavy one, up to 70000 of them, together up to a
    fiftieth of it.  The heavy key's value is zero in half of the dimensions."""
    from tscale_b200 import ops
    n_seq, n, page = 460, 70001, 128
    pages, gen = -(-n // page), _gen(30)
    shape, one = (pages, 1, page), 40 if kv == "i8" else 1
    k = torch.full(shape + (d,), one, device=DEV).to(CODES[kv])
    v = torch.randint(20, 128, shape + (d,), generator=gen, device=DEV).to(torch.int8) if kv == "i8" else (torch.rand(shape + (d,), generator=gen, device=DEV) * 1.5 + 0.5).to(CODES[kv])
    unit = one * one * d * DOT / d ** 0.5
    z = torch.full((pages * page,), -16.3, device=DEV)
    heavy = {"first": 0, "middle": 35555, "last": n - 2, "spread": 3, "falls": 0}[logits]
    if logits == "spread":
        z = z + 1.5 * torch.randn(z.shape, generator=gen, device=DEV).clamp(-3, 3)
    if logits == "falls":
        z = torch.linspace(12, -20, z.shape[0], device=DEV)
    else:
        z[heavy] = 6.0
    rows = v.view(torch.int8).view(-1, d)
    rows[heavy, :d // 2] = 0
    ks, vs = (z / unit).view(shape).contiguous(), (torch.rand(shape, generator=gen, device=DEV) + 0.5) * (0.01 if kv == "i8" else 0.5)
    cache = ops.PagedKV(k, v, ks, vs)
    table = torch.arange(pages, dtype=torch.int32, device=DEV).expand(n_seq, pages).contiguous()
    ctx = torch.full((n_seq,), n, dtype=torch.int32, device=DEV)
    q = torch.full((n_seq, group * d), one, device=DEV).to(CODES[kv])
    qs = torch.linspace(1.0, 1.45, group, device=DEV).expand(n_seq, group).contiguous()
    _needs_workspace(cache, n_seq, group, n)
    got = ops.paged_decode(cache, table, ctx, q, qs, WHOLE, 0.0, max_ctx=n)
    zs = qs[0].double()[:, None] * ks.view(-1)[:n - 1].double() * unit
    values = v.view(-1, d)[:n - 1].double() * vs.view(-1)[:n - 1].double()[:, None]
    w = torch.exp2(zs)
    w = w / (1 + w.sum(1, keepdim=True))
    tol = 2.0 ** -16 * float(values.abs().max()) + 2.0 ** -15 * (w @ values.abs())
    off = (got.double().view(n_seq, group, d) - (w @ values)).abs()
    assert not (off > tol).any(), float((off / tol).max())
