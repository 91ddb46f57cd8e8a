"""Measured cases of the paged key-value cache: the calls a serving program makes, and the same operators in plain torch.

  append  rows of a ragged batch of prompts, or one row per sequence, into the pages (ops.paged_append)
  decode  attention of one new token per sequence over the pages (ops.paged_decode); with `track` it also adds each key's attention
          weight to the cache's accumulated weights
  select  which slots of each sequence and key head stay when a cache is cut to a budget (ops.paged_evict_select)
  move    the kept rows behind the budget move into the slots that became free (ops.paged_evict_move)

A cache is a tuple (k, v, k_scale, v_scale, pos, weight) of pools: k, v 8-bit [pages][key heads][page size][head size], the others
[pages][key heads][page size]; token t of sequence s is in slot t % page size of page table[s][t // page size].  pos (positions of the
tokens) and weight exist in caches that are evicted from.  A case is a dict of plain values; `listed` gives the fixed ones, `draw` more.
"""
import math
import random

import torch

own = False

DEV = torch.device("cuda:0")
WHOLE = 1 << 30  # a window longer than any context
VEC = 1.0 / 24   # scale of a unit vector's int8 codes
CODES = {"i8": torch.int8, "e4m3": torch.float8_e4m3fn}
FLOATS = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # a serving batch's new tokens: one row per sequence, the call's latency
        dict(name="append_token", kind="append", seqs=64, rows_lo=1, rows_hi=1, before=1500, kvh=8, d=128, page=64, kv="i8", scale="f16", track=False),
        # a batch of prompts of unequal length, written behind what their sequences hold, into a cache that is evicted from
        dict(name="append_prompts", kind="append", seqs=9, rows_lo=700, rows_hi=4096, before=333, kvh=16, d=128, page=64, kv="e4m3", scale="f16", track=True),
        # one user's conversation: the step's latency
        dict(name="decode_single", kind="decode", seqs=1, ctx_lo=1000, ctx_hi=1000, heads=12, kvh=12, d=64, page=64, kv="i8", scale="f32", out="f32",
             window=WHOLE, slope=0.0, track=False),
        # a serving batch, a key head for each query head: the stream of the caches
        dict(name="decode_batch", kind="decode", seqs=64, ctx_lo=1024, ctx_hi=8192, heads=16, kvh=16, d=128, page=64, kv="i8", scale="f16", out="bf16",
             window=WHOLE, slope=0.0, track=False),
        # the same with key heads shared by four query heads, in the prefill's type, small pages
        dict(name="decode_shared", kind="decode", seqs=48, ctx_lo=500, ctx_hi=9000, heads=32, kvh=8, d=128, page=16, kv="e4m3", scale="f16", out="bf16",
             window=WHOLE, slope=0.0, track=False),
        # few long contexts: the work has to be split over the cache's length
        dict(name="decode_long", kind="decode", seqs=2, ctx_lo=100000, ctx_hi=131072, heads=32, kvh=4, d=128, page=128, kv="i8", scale="f16", out="f16",
             window=WHOLE, slope=0.0, track=False),
        # one conversation, and a serving batch, over caches that are evicted from: attention that keeps the keys' weights
        dict(name="track_single", kind="decode", seqs=1, ctx_lo=2049, ctx_hi=2049, heads=16, kvh=4, d=64, page=32, kv="i8", scale="f16", out="f32",
             window=WHOLE, slope=0.0, track=True),
        dict(name="track_batch", kind="decode", seqs=40, ctx_lo=2048, ctx_hi=6144, heads=32, kvh=8, d=128, page=64, kv="i8", scale="f16", out="bf16",
             window=WHOLE, slope=0.0, track=True),
        # a batch of caches over their budget
        dict(name="select_batch", kind="select", seqs=40, ctx_lo=2000, ctx_hi=6144, kvh=8, page=64, keep=2048, recent=64),
        # two long conversations cut to an eighth
        dict(name="select_long", kind="select", seqs=2, ctx_lo=100000, ctx_hi=131072, kvh=4, page=128, keep=16384, recent=1000),
        # the rows of one small cache, and those of a batch, take their new places
        dict(name="move_single", kind="move", seqs=1, ctx_lo=1500, ctx_hi=1500, kvh=4, d=64, page=32, kv="i8", scale="f16", keep=1000),
        dict(name="move_batch", kind="move", seqs=40, ctx_lo=2500, ctx_hi=6144, kvh=8, d=128, page=64, kv="e4m3", scale="f16", keep=2048),
    ]


def _log(rng, lo, hi):
    """Log-uniform integer in [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("append", "decode", "decode", "decode", "select", "move"))
    seqs, page = _log(rng, 1, 96), rng.choice((16, 32, 64, 128, 256))
    if kind == "select":
        # at most 40 * 6144 * 8 slots
        kvh = rng.choice((1, 2, 4, 8, 12))
        hi = _log(rng, 40, max(41, min(131072, 40 * 6144 * 8 // (seqs * kvh))))
        keep = _log(rng, 8, hi)
        return dict(kind=kind, seqs=seqs, ctx_lo=rng.randrange(1, hi), ctx_hi=hi, kvh=kvh, page=page, keep=keep, recent=rng.randrange(0, keep // 4 + 1))
    d, kvh = rng.choice(((64, 4), (64, 12), (128, 1), (128, 5), (128, 8), (128, 16)))
    kv, scale = rng.choice(("i8", "e4m3")), rng.choice(("f16", "f32"))
    if kind == "append":
        # at most 9 * 4096 rows of 16 * 128
        hi = _log(rng, 1, 9 * 4096 * 16 * 128 // (seqs * kvh * d))
        return dict(kind=kind, seqs=seqs, rows_lo=rng.randrange(0, hi), rows_hi=hi, before=rng.randrange(0, 2000), kvh=kvh, d=d, page=page, kv=kv, scale=scale,
                    track=rng.random() < 0.5)
    if kind == "move":
        hi = _log(rng, 40, max(41, min(65536, 40 * 6144 * 8 * 128 // (seqs * kvh * d))))
        return dict(kind=kind, seqs=seqs, ctx_lo=rng.randrange(1, hi), ctx_hi=hi, kvh=kvh, d=d, page=page, kv=kv, scale=scale, keep=_log(rng, 8, hi - 1))
    # at most 64 * 8192 tokens of 16 * 128
    hi = _log(rng, 2, min(200000, 64 * 8192 * 16 * 128 // (seqs * kvh * d)))
    window, slope = rng.choice(((WHOLE, 0.0), (WHOLE, 0.0), (64, 0.5), (1000, 0.0), (WHOLE, 0.01)))
    return dict(kind=kind, seqs=seqs, ctx_lo=rng.randrange(1, hi), ctx_hi=hi, heads=kvh * rng.choice((1, 1, 2, 4, 7, 8, 16)), kvh=kvh, d=d, page=page, kv=kv,
                scale=scale, out=rng.choice(("f32", "bf16", "f16")), window=window, slope=slope, track=rng.random() < 0.4)


def _lengths(lo, hi, n, seed):
    """n lengths in [lo, hi], hi among them."""
    r = random.Random(seed)
    lens = [r.randint(lo, hi) for _ in range(n)]
    lens[r.randrange(n)] = hi
    return lens


def _vectors(shape, kv, gen):
    """Codes of unit-variance vectors: int8 with a step of 1 / 24, or e4m3."""
    x = torch.randn(shape, generator=gen, device=DEV, dtype=torch.float16)
    return (x * 24).clamp_(-127, 127).round_().to(torch.int8) if kv == "i8" else x.to(CODES[kv])


def _scales(shape, kv, dtype, gen):
    """Root mean squares of the vectors, times the step of their codes."""
    return ((torch.rand(shape, generator=gen, device=DEV) + 0.5) * (VEC if kv == "i8" else 1.0)).to(dtype)


def _pool(lens, most, case, gen, vectors=True):
    """Pools with room for `most` tokens of every sequence, and the table of the pages that `lens` tokens take, in random order; other entries are -1."""
    page, kvh = case["page"], case["kvh"]
    cols = torch.arange(-(-most // page), device=DEV)
    pages = len(lens) * cols.shape[0]
    order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    used = -(-torch.tensor(lens, device=DEV) // page)
    first = used.cumsum(0) - used
    table = torch.where(cols < used[:, None], order[(first[:, None] + cols).clamp(max=pages - 1)], -1).to(torch.int32).contiguous()
    k = v = ks = vs = None
    if vectors:
        k, v = (_vectors((pages, kvh, page, case["d"]), case["kv"], gen) for _ in range(2))
        ks, vs = (_scales((pages, kvh, page), case["kv"], FLOATS[case["scale"]], gen) for _ in range(2))
    return k, v, ks, vs, table, pages


def _tracked(table, lens, tokens, case, pages, gen):
    """pos and weight of caches that were evicted from before: each key head keeps other tokens, not in their order; the newest token is last."""
    page, kvh = case["page"], case["kvh"]
    pos = torch.zeros((pages, kvh, page), dtype=torch.int32, device=DEV)
    weight = torch.zeros((pages, kvh, page), dtype=torch.float32, device=DEV)
    top = max(lens)
    slot = torch.arange(top, device=DEV)
    n, seen = torch.tensor(lens, device=DEV)[:, None, None], torch.tensor(tokens, device=DEV)[:, None, None]
    mix = torch.rand((len(lens), kvh, top), generator=gen, device=DEV)
    mix = torch.where(slot < n - 1, mix, 2.0 + slot).argsort(-1)                       # a permutation of the slots before the newest
    where = (mix * (seen - 1) // (n - 1).clamp(min=1)).to(torch.int32)                 # spread over what the sequence has seen
    heavy = torch.rand((len(lens), kvh, top), generator=gen, device=DEV) ** 9 * 20
    heavy = torch.where(torch.rand(heavy.shape, generator=gen, device=DEV) < 0.05, 0.0, heavy)  # never attended
    live = (slot < n).expand_as(where)
    at, head = table.long()[:, slot // page][:, None].expand_as(where), torch.arange(kvh, device=DEV)[:, None].expand_as(where)
    off = (slot % page).expand_as(where)
    pos[at[live], head[live], off[live]] = where[live]
    weight[at[live], head[live], off[live]] = heavy[live]
    return pos, weight


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    kvh, page, kind = case["kvh"], case["page"], case["kind"]
    r = random.Random(seed)
    if kind == "append":
        counts = _lengths(case["rows_lo"], case["rows_hi"], case["seqs"], seed)
        lens, most = [n + r.randint(0, case["before"]) for n in counts], case["rows_hi"] + case["before"]
    else:
        lens, most = _lengths(case["ctx_lo"], case["ctx_hi"], case["seqs"], seed), case["ctx_hi"]
    k, v, ks, vs, table, pages = _pool(lens, most, case, gen, kind != "select")
    state = dict(case=case, table=table, lens=_int32(lens), pos=None, tokens=None, top=max(lens))
    pos = weight = None
    if case.get("track") or kind in ("select", "move"):
        tokens = [n + r.randint(0, n) for n in lens]
        pos, weight = _tracked(table, lens, tokens, case, pages, gen)
        state["tokens"] = _int32(tokens)
    state["kv"] = (k, v, ks, vs, pos, weight)
    if kind == "append":
        rows, d = sum(counts), case["d"]
        starts = [0]
        for n in counts:
            starts.append(starts[-1] + n)
        state["new"] = tuple(x for _ in range(2) for x in (_vectors((rows, kvh * d), case["kv"], gen), _scales((kvh, rows), case["kv"], torch.float32, gen)))
        state["starts"] = _int32(starts)
    elif kind == "decode":
        state["q"] = _vectors((case["seqs"], case["heads"] * case["d"]), case["kv"], gen)
        state["q_scale"] = _scales((case["seqs"], case["heads"]), case["kv"], torch.float32, gen)
    elif kind == "move":
        # the places that a choice by weight gives
        state["moves"], state["counts"], _ = _select(state["kv"], table, state["lens"], state["tokens"], case["keep"], 8, page, state["top"])
    return state


def run(state):
    c, kv, table, lens, tokens = state["case"], state["kv"], state["table"], state["lens"], state["tokens"]
    kind = c["kind"]
    if own:
        from tscale_b200 import ops
        if kind == "append":
            ops.paged_append(kv, table, lens, *state["new"], row_starts=state["starts"], tokens=tokens)
            return [x for x in kv if x is not None]
        if kind == "decode":
            out = ops.paged_decode(kv, table, lens, state["q"], state["q_scale"], c["window"], c["slope"], max_ctx=state["top"], out_dtype=FLOATS[c["out"]],
                                   tokens=tokens)
            return [out, kv[5]] if c["track"] else [out]
        if kind == "select":
            return ops.paged_evict_select(kv, table, lens, c["keep"], c["recent"], max_ctx=state["top"], tokens=tokens)
        ops.paged_evict_move(kv, table, state["moves"], state["counts"])
        return kv
    if kind == "append":
        _append(kv, table, lens, tokens, state["starts"], *state["new"], c["page"])
        return [x for x in kv if x is not None]
    if kind == "decode":
        out = _decode(kv, table, lens, tokens, state["q"], state["q_scale"], c, state["top"])
        return [out, kv[5]] if c["track"] else [out]
    if kind == "select":
        return _select(kv, table, lens, tokens, c["keep"], c["recent"], c["page"], state["top"])
    _move(kv, table, state["moves"], c["page"])
    return kv


# ---- the operators in plain torch

def _bytes(x):
    """8-bit codes as a type that indexing knows."""
    return x.view(torch.int8)


def _append(kv, table, lens, tokens, starts, k_new, ks_new, v_new, vs_new, page):
    k, v, ks, vs, pos, weight = kv
    rows, kvh, d = k_new.shape[0], k.shape[1], k.shape[3]
    row = torch.arange(rows, device=DEV, dtype=torch.int32)
    seq = torch.searchsorted(starts, row, right=True) - 1
    back = starts[seq + 1] - row  # 1: the sequence's newest
    slot = (lens[seq] - back).long()
    at, off = table[seq, slot // page].long(), slot % page
    _bytes(k)[at, :, off] = _bytes(k_new).view(rows, kvh, d)
    _bytes(v)[at, :, off] = _bytes(v_new).view(rows, kvh, d)
    ks[at, :, off] = ks_new.t().to(ks.dtype)
    vs[at, :, off] = vs_new.t().to(vs.dtype)
    if pos is not None:
        pos[at, :, off] = (tokens[seq] - back)[:, None].expand(rows, kvh)
        weight[at, :, off] = 0.0


def _decode(kv, table, lens, tokens, q, q_scale, c, top):
    k, v, ks, vs, pos, weight = kv
    seqs, kvh, d, page = q.shape[0], k.shape[1], k.shape[3], c["page"]
    group = c["heads"] // kvh
    slot = torch.arange(top, device=DEV)
    at, off = table[:, slot // page].clamp(min=0).long(), slot % page
    cur = ((lens if tokens is None else tokens) - 1)[:, None, None]
    where = slot.to(torch.int32).expand(seqs, kvh, top) if pos is None else pos[at, :, off].transpose(1, 2)
    far = cur - where
    seen = (slot < lens[:, None, None]) & ((far == 0) if c["window"] == 0 else (far >= 1) & (far <= c["window"]))
    keys = _bytes(k)[at, :, off].view(k.dtype).transpose(1, 2).float()
    qf = q.float().view(seqs, kvh, group, d)
    z = torch.matmul(qf, keys.transpose(2, 3))
    del keys
    z = z * ks[at, :, off].transpose(1, 2).float()[:, :, None] * (q_scale.view(seqs, kvh, group, 1) * (math.sqrt(1.0 / d) * 0.5 / 0.693147))
    z = z - c["slope"] * far[:, :, None].float()
    z = torch.where(seen[:, :, None], z, -math.inf)
    m = z.amax(-1, keepdim=True).clamp(min=0.0)
    p = torch.exp2(z - m)
    p = p / (p.sum(-1, keepdim=True) + torch.exp2(-m))
    del z
    vals = _bytes(v)[at, :, off].view(v.dtype).transpose(1, 2).float() * torch.where(seen, vs[at, :, off].transpose(1, 2).float(), 0.0)[..., None]
    out = torch.matmul(p, vals)
    if weight is not None:
        index = (at[:, None] * kvh + torch.arange(kvh, device=DEV)[:, None]) * page + off
        weight.view(-1).scatter_add_(0, index.reshape(-1), p.sum(2).reshape(-1))
    return out.reshape(seqs, -1).to(FLOATS[c["out"]])


def _select(kv, table, lens, tokens, keep, recent, page, top):
    pos, weight = kv[4], kv[5]
    seqs, kvh = table.shape[0], weight.shape[1]
    slot = torch.arange(top, device=DEV)
    at, off = table[:, slot // page].clamp(min=0).long(), slot % page
    w = weight[at, :, off].transpose(1, 2)
    newest = pos[at, :, off].transpose(1, 2) > (tokens - 1)[:, None, None] - recent
    live = slot < lens[:, None, None]
    w = torch.where(live, torch.where(newest, math.inf, w), -math.inf)
    order = w.sort(dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, slot.expand_as(order))
    over = (lens > keep)[:, None, None]
    kept = live & ((rank < keep) | ~over)
    hole, mover = over & ~kept & (slot < keep), over & kept & (slot >= keep)
    cap = max(1, min(keep, top - keep))
    moves = torch.full((seqs, kvh, cap + 1, 2), -1, dtype=torch.int32, device=DEV)  # the last entry takes what is none
    numbers = slot.to(torch.int32).expand(seqs, kvh, top)
    for_dst = torch.where(hole, hole.cumsum(-1) - 1, cap)
    for_src = torch.where(mover, mover.cumsum(-1) - 1, cap)
    moves[..., 0].scatter_(-1, for_dst, numbers)
    moves[..., 1].scatter_(-1, for_src, numbers)
    return moves[:, :, :cap].contiguous(), mover.sum(-1).to(torch.int32), lens.clamp(max=keep)


def _move(kv, table, moves, page):
    seq, head, entry = (moves[..., 0] >= 0).nonzero(as_tuple=True)
    dst, src = moves[seq, head, entry, 0].long(), moves[seq, head, entry, 1].long()
    to, of = table[seq, dst // page].long(), table[seq, src // page].long()
    k, v, ks, vs, pos, weight = kv
    k, v = _bytes(k), _bytes(v)
    k[to, head, dst % page] = k[of, head, src % page]
    v[to, head, dst % page] = v[of, head, src % page]
    ks[to, head, dst % page] = ks[of, head, src % page]
    vs[to, head, dst % page] = vs[of, head, src % page]
    pos[to, head, dst % page] = pos[of, head, src % page]
    weight[to, head, dst % page] = weight[of, head, src % page]


# ---- the definitions in 64 bits, one sequence at a time

def exact(case, seed):
    if case["kind"] != "decode":
        return None  # copies and choices: nothing is computed
    s = prepare(case, seed)
    k, v, ks, vs, pos, weight = s["kv"]
    kvh, d, page, n_seq = case["kvh"], case["d"], case["page"], case["seqs"]
    group = case["heads"] // kvh
    scale = 0.5 / 0.693147 / d ** 0.5
    lens = s["lens"].tolist()
    seen = lens if s["tokens"] is None else s["tokens"].tolist()
    out = torch.zeros((n_seq, kvh, group, d), dtype=torch.float64, device=DEV)
    total = None if weight is None else weight.double()
    for i, n in enumerate(lens):
        pages = s["table"][i, :-(-n // page)].long()
        rows = lambda x: (x.view(torch.int8)[pages].view(x.dtype) if x.element_size() == 1 else x[pages]).double().transpose(0, 1).flatten(1, 2)[:, :n]  # noqa: E731
        place = torch.arange(n, device=DEV, dtype=torch.float64).expand(kvh, n) if pos is None else rows(pos)
        dist = (seen[i] - 1) - place
        valid = dist == 0 if case["window"] == 0 else (dist > 0) & (dist <= case["window"])
        qi = s["q"][i].double().view(kvh, group, d) * s["q_scale"][i].double().view(kvh, group, 1) * scale
        logit = torch.einsum("hgd,hnd->hgn", qi, rows(k) * rows(ks)[..., None]) - case["slope"] * dist[:, None]
        e = torch.where(valid[:, None], torch.exp2(logit), 0.0)
        e = e / (1.0 + e.sum(-1, keepdim=True))
        out[i] = torch.einsum("hgn,hnd->hgd", e, rows(v) * rows(vs)[..., None])
        if total is not None:
            heads = torch.arange(kvh, device=DEV)[:, None]
            t = torch.arange(n, device=DEV)
            total[pages[t // page], heads, t % page] += e.sum(1)
    out = out.reshape(n_seq, -1)
    return [out] if total is None else [out, total]


def work(case):
    """Bytes that have to move and operations; lengths are those of seed 0."""
    kvh, n = case["kvh"], case["seqs"]
    if case["kind"] == "append":
        rows = sum(_lengths(case["rows_lo"], case["rows_hi"], n, 0))
        sb = 2 if case["scale"] == "f16" else 4
        return {"bytes": rows * kvh * (2 * 2 * case["d"] + 2 * (4 + sb) + (8 if case["track"] else 0)), "flops": 0}
    lens = _lengths(case["ctx_lo"], case["ctx_hi"], n, 0)
    if case["kind"] == "decode":
        d, sb = case["d"], 2 if case["scale"] == "f16" else 4
        if case["track"]:  # every slot's position is looked at
            keys = sum(min(x - 1, case["window"]) for x in lens)
            slots = sum(lens)
            size = keys * kvh * (2 * d + 2 * sb + 8) + slots * kvh * 4
        else:
            keys = sum(min(x - 1, case["window"]) for x in lens)
            size = keys * kvh * (2 * d + 2 * sb)
        return {"bytes": size + n * case["heads"] * d * 5, "flops": 4 * d * case["heads"] * keys}
    moved = sum(case["keep"] * (x - case["keep"]) // x for x in lens if x > case["keep"]) * kvh  # about: kept tokens are anywhere in the cache
    if case["kind"] == "select":
        return {"bytes": sum(x for x in lens if x > case["keep"]) * kvh * (8 if case["recent"] else 4) + moved * 8, "flops": 0}
    sb = 2 if case["scale"] == "f16" else 4
    return {"bytes": moved * (2 * (2 * case["d"] + 2 * sb + 8) + 8), "flops": 0}
