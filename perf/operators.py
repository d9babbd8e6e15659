"""Operators of a paged 4-bit latent cache, as performance cases: attention over it, writing and reading it, and the
management of its pages.

`run` computes a case with the package's entry points (`own`) or in plain torch, in 32 bits, with the same results.

Records of the cache are 416 bytes a token, two halves of 208: the codes of 256 latent values (128 bytes), the 16 scales of
their groups of 16 (one byte each), 32 rope values in bf16.  A scale byte is five bits of exponent e and three of mantissa m,
(8 + m) 2^(e - 18), 255 = NaN; a code is a sign and one of 0, .5, 1, 1.5, 2, 3, 4, 6.  A 32-bit word holds eight values, the
even ones in its low half; `SIGN` and `MAG` say where the four of a half have their bits.

Kinds
  attn      sparse attention of `tokens` query tokens for each of `batch` sequences over the latents that an indexer selected
  cache     one prefill chunk's traffic: `new` tokens' latents written to their cache rows, then the sequence's whole context
            read back as bf16 rows for the prefill kernel
  copy      `pairs` pages copied in every cache of `layers` layers
  turnover  a scheduler's step: finished and dropped sequences freed, new ones given pages, survivors forked
  compact   a fragmented pool moved to its lowest pages
"""
import math

import torch

own = False

DEV = "cuda"
PAGE = 64
RECORD = 416
LATENT, ROPE, GROUP = 512, 64, 16
SCALE = 192 ** -0.5
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
SIGN = (15, 12, 9, 14)                                  # of the value's 16-bit half
MAG = ((8, 7, 6), (5, 4, 3), (2, 1, 0), (11, 10, 13))   # bits of the level's number, highest first
K_BYTES, K_SCALE_BYTES = 128, 4                         # the indexer's key and its scale, which live in the same pages


def listed():
    return [
        # decode: one short conversation; the 128K batch; a tensor-parallel rank's heads; speculative tokens, odd lengths
        {"name": "attn_1x2k", "kind": "attn", "batch": 1, "tokens": 1, "heads": 128, "ctx": 2000, "topk": 2048, "ragged": False, "idle": False},
        {"name": "attn_64x128k", "kind": "attn", "batch": 64, "tokens": 1, "heads": 128, "ctx": 131072, "topk": 2048, "ragged": False, "idle": False},
        {"name": "attn_160x9k_tp8", "kind": "attn", "batch": 160, "tokens": 1, "heads": 16, "ctx": 9000, "topk": 2048, "ragged": True, "idle": False},
        {"name": "attn_64x20k_4", "kind": "attn", "batch": 64, "tokens": 4, "heads": 128, "ctx": 20011, "topk": 2048, "ragged": True, "idle": True},
        # a follow-up question on a cached 20K prompt; a whole chunk at the end of a 128K context
        {"name": "cache_257_of_20k", "kind": "cache", "new": 257, "ctx": 20011, "dtype": "f32"},
        {"name": "cache_8k_of_128k", "kind": "cache", "new": 8192, "ctx": 131072, "dtype": "bf16"},
        # a few pages between sequences; a long prefix
        {"name": "copy_5x2", "kind": "copy", "pool": 300, "pairs": 5, "layers": 2},
        {"name": "copy_700x16", "kind": "copy", "pool": 2000, "pairs": 700, "layers": 16},
        # beams of one prompt; a loaded server: half of its rows turn over
        {"name": "turnover_8", "kind": "turnover", "rows": 12, "pages": 40, "stay": 4, "fresh": 2, "forks": 4, "layers": 4},
        {"name": "turnover_200", "kind": "turnover", "rows": 200, "pages": 130, "stay": 90, "fresh": 40, "forks": 60, "layers": 2},
        # a small pool of one layer; a server's cache after hours of traffic
        {"name": "compact_200x1", "kind": "compact", "rows": 20, "pages": 20, "pool": 200, "layers": 1, "used": 0.6},
        {"name": "compact_6k_x8", "kind": "compact", "rows": 250, "pages": 128, "pool": 6000, "layers": 8, "used": 0.55},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "cache", "copy", "turnover", "compact"])
    if kind == "attn":
        batch = _log(rng, 1, 256)
        tokens = rng.choice([1, 1, 1, 2, 3, 4])
        tokens = min(tokens, 256 // batch) or 1
        heads = rng.choice([128, 128, 64, 32, 16, 8])
        return {"kind": kind, "batch": batch, "tokens": tokens, "heads": heads, "ctx": _log(rng, 1, min(131072, 64 * 131072 // batch)),
                "topk": rng.choice([2048, 2048, 2048, 1024, 512, 100]), "ragged": rng.random() < 0.7, "idle": rng.random() < 0.3}
    if kind == "cache":
        ctx = _log(rng, 1, 131072)
        return {"kind": kind, "new": _log(rng, 1, min(ctx, 8192)), "ctx": ctx, "dtype": rng.choice(["bf16", "bf16", "f32"])}
    if kind == "copy":
        layers = rng.choice([1, 2, 4, 8, 16])
        pool = _log(rng, 40, 32000 // layers)
        return {"kind": kind, "pool": pool, "pairs": _log(rng, 1, min(pool // 2, 11200 // layers)), "layers": layers}
    if kind == "turnover":
        rows = _log(rng, 6, 200)
        stay = rng.randint(2, rows - 4)
        fresh = rng.randint(1, rows - stay - 2)
        return {"kind": kind, "rows": rows, "pages": _log(rng, 2, min(400, 26000 // rows)), "stay": stay, "fresh": fresh,
                "forks": rng.randint(1, rows - stay - fresh), "layers": rng.choice([1, 2])}
    rows = _log(rng, 2, 250)
    pages = _log(rng, 2, 200)
    layers = rng.choice([1, 2, 4, 8])
    return {"kind": kind, "rows": rows, "pages": pages, "pool": max(16, min(rows * pages, 48000 // layers) * 3 // 4), "layers": layers,
            "used": rng.choice([0.2, 0.4, 0.55, 0.7, 0.9])}


# ---- the record, in plain torch -------------------------------------------------------------------------------------
def _quantise(x):
    """Latent values [N, 512] fp32 -> level numbers [N, 512], signs and scale bytes [N, 32]."""
    g = x.view(-1, LATENT // GROUP, GROUP)
    amax = g.abs().amax(-1)
    bad = ~torch.isfinite(amax)
    want = (torch.where(bad, torch.zeros_like(amax), amax) / torch.full_like(amax, 6.0)).clamp(2.0 ** -15, 61440.0)
    e = torch.frexp(want)[1] - 1
    scale = torch.round(torch.ldexp(want, 3 - e)) * torch.exp2((e - 3).float())          # four significant bits, ties to even
    e = torch.frexp(scale)[1] - 1
    byte = ((e + 15) * 8 + torch.ldexp(scale, 3 - e).int() - 8).masked_fill(bad, 255)
    y = (g / scale.unsqueeze(-1)).abs().masked_fill(bad.unsqueeze(-1), 0.0)
    # halfway cases go to the even level number: up from 0.75, 1.75 and 3.5
    n = ((y > 0.25).int() + (y >= 0.75).int() + (y > 1.25).int() + (y >= 1.75).int() + (y > 2.5).int() + (y >= 3.5).int() + (y > 5.0).int())
    return n.view(-1, LATENT), (torch.signbit(x)).int(), byte


def _records(kv):
    """Rows [N, 576] -> records uint8 [N, 416]."""
    n, sign, byte = _quantise(kv[:, :LATENT].float())
    n, sign = (t.view(-1, LATENT // 8, 4, 2) for t in (n, sign))             # word, k, half of the word
    word = torch.zeros(n.shape[0], LATENT // 8, dtype=torch.int64, device=kv.device)
    for k in range(4):
        half = sign[:, :, k].long() << SIGN[k]
        for bit, at in zip((2, 1, 0), MAG[k]):
            half |= ((n[:, :, k].long() >> bit) & 1) << at
        word |= half[..., 0] | (half[..., 1] << 16)
    word = torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32).view(torch.uint8).view(-1, 2, 128)
    rope = kv[:, LATENT:].to(torch.bfloat16).contiguous().view(torch.uint8).view(-1, 2, 64)
    return torch.cat((word, byte.to(torch.uint8).view(-1, 2, 16), rope), -1).view(-1, RECORD)


def _values(rec):
    """Records uint8 [..., 416] -> rows fp32 [..., 576]."""
    lead = rec.shape[:-1]
    h = rec.reshape(-1, 2, RECORD // 2)
    w = h[..., :128].contiguous().view(torch.int16).view(-1, LATENT // 8, 2).int()      # word, half of the word
    levels = torch.tensor(LEVELS, device=rec.device)
    out = torch.empty(w.shape[0], LATENT // 8, 4, 2, device=rec.device)
    for k in range(4):
        n = 0
        for at in MAG[k]:
            n = n * 2 + ((w >> at) & 1)
        out[:, :, k] = levels[n] * (1 - 2 * ((w >> SIGN[k]) & 1))
    b = h[..., 128:144].int()
    scale = ((8 + b % 8) * torch.exp2((b // 8 - 18).float())).masked_fill(b == 255, math.nan)
    lat = out.view(-1, LATENT // GROUP, GROUP) * scale.reshape(-1, LATENT // GROUP, 1)
    rope = h[..., 144:].contiguous().view(torch.bfloat16).float()
    return torch.cat((lat.view(-1, LATENT), rope.reshape(-1, ROPE)), -1).view(*lead, LATENT + ROPE)


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device=DEV, generator=g, dtype=dtype)


def _randint(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, device=DEV, generator=g)


def _rand_bytes(g, *shape):
    """Bytes that need not mean anything: pages are moved as they are."""
    n = math.prod(shape)
    return torch.randint(-2 ** 62, 2 ** 62, (-(-n // 8),), device=DEV, generator=g).view(torch.uint8)[:n].view(*shape)


def _caches(g, case, pool):
    """What a server keeps in its pages, for all layers: indexer keys, their scales, latents."""
    layers, rows = case["layers"], pool * PAGE
    return [_rand_bytes(g, layers, rows, K_BYTES), _rand_bytes(g, layers, rows, K_SCALE_BYTES), _rand_bytes(g, layers, rows, RECORD)]


def _pool_of(case):
    """Pages of a turnover's pool: room for every row, and somewhat more."""
    return case["rows"] * case["pages"] + 50


def _tables(g, rows, pages, ctx, pool):
    """Sequences of the lengths `ctx` in pages drawn from the pool; -1 behind their ends.  Every page has one holder."""
    used = (ctx + PAGE - 1) // PAGE
    ids = torch.randperm(pool, device=DEV, generator=g)[:rows * pages].int()
    if ids.numel() < rows * pages:                       # a tight pool: pages are dealt to the rows in order until they run out
        at = torch.cumsum(used, 0) - used
        pos = (at[:, None] + torch.arange(pages, device=DEV)).clamp_max(ids.numel() - 1)
        table = ids[pos]
    else:
        table = ids.view(rows, pages)
    table = torch.where(torch.arange(pages, device=DEV) < used[:, None], table, torch.full_like(table, -1))
    refs = torch.zeros(pool, dtype=torch.int32, device=DEV)
    refs[table[table >= 0].long()] = 1
    return table.contiguous(), refs


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    st = {"kind": kind}
    if kind == "attn":
        batch, tokens, ctx, topk = case["batch"], case["tokens"], case["ctx"], case["topk"]
        pages = -(-ctx // PAGE)
        some = _records(_randn(g, min(batch * pages * PAGE, 1 << 15), LATENT + ROPE))
        n = batch * pages * PAGE
        st["cache"] = some[_randint(g, 0, some.shape[0], n)] if n > some.shape[0] else some
        st["table"] = torch.randperm(batch * pages, device=DEV, generator=g).int().view(batch, pages)
        lens = _randint(g, ctx // 2 + 1, ctx + 1, batch) if case["ragged"] else torch.full((batch,), ctx, device=DEV)
        if case["idle"] and batch > 1:
            lens[int(_randint(g, 0, batch, 1))] = 0      # a row of the batch that no sequence uses
        lens = lens.repeat_interleave(tokens)
        # an indexer's selection: distinct positions in no particular order, -1 behind the last one
        if ctx <= topk:
            order = torch.argsort(torch.rand(batch * tokens, ctx, device=DEV, generator=g), -1)
            idx = torch.full((batch * tokens, topk), -1, device=DEV)
            seen = order < lens[:, None]
            slot = torch.cumsum(seen.int(), -1) - 1
            r, c = torch.nonzero(seen, as_tuple=True)
            idx[r, slot[r, c]] = order[r, c]
        else:                                            # one position in each of topk equal stretches of the context, shuffled
            span = lens[:, None].double() / topk
            j = torch.arange(topk, device=DEV)
            pos = ((j + torch.rand(batch * tokens, topk, device=DEV, generator=g, dtype=torch.float64)) * span).long()
            lo = (j * span).ceil().long()                # stretches that share no position
            pos = torch.minimum(torch.maximum(pos, lo), lens[:, None] - 1)
            pos = torch.where((pos >= lo) & (pos < ((j + 1) * span).ceil().long()), pos, torch.full_like(pos, -1))
            idx = pos.gather(1, torch.argsort(torch.rand(batch * tokens, topk, device=DEV, generator=g), -1))
            keep = torch.argsort((idx < 0).int(), dim=-1, stable=True)
            idx = idx.gather(1, keep)
        st["idx"] = idx.int().contiguous()
        st["q"] = _randn(g, batch * tokens, case["heads"], LATENT + ROPE, dtype=torch.bfloat16)
        st["tokens"] = tokens
    elif kind == "cache":
        new, ctx = case["new"], case["ctx"]
        pages = -(-ctx // PAGE)
        pool = pages + 7
        some = _records(_randn(g, min(pool * PAGE, 1 << 15), LATENT + ROPE))
        st["cache"] = some[_randint(g, 0, some.shape[0], pool * PAGE)]
        st["row"] = torch.randperm(pool, device=DEV, generator=g)[:pages].int()
        pos = torch.arange(ctx - new, ctx, device=DEV)
        st["slots"] = st["row"][pos // PAGE] * PAGE + (pos % PAGE).int()
        st["kv"] = _randn(g, new, LATENT + ROPE, dtype=torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
        st["ctx"] = ctx
    elif kind == "copy":
        st["caches"] = _caches(g, case, case["pool"])
        ids = torch.randperm(case["pool"], device=DEV, generator=g).int()
        st["src"], st["dst"] = ids[:case["pairs"]].clone(), ids[case["pairs"]:2 * case["pairs"]].clone()
    elif kind == "turnover":
        rows, pages, stay, fresh, forks = (case[k] for k in ("rows", "pages", "stay", "fresh", "forks"))
        ctx = _randint(g, 1, pages * PAGE + 1, rows)
        st["table"], st["refs"] = _tables(g, rows, pages, ctx, _pool_of(case))
        st["ctx"] = ctx.int()
        st["caches"] = _caches(g, case, _pool_of(case))
        order = torch.randperm(rows, device=DEV, generator=g).int()
        st["gone"] = order[stay:].clone()
        st["new"] = order[stay:stay + fresh].clone()
        st["max_new"] = pages * PAGE
        st["n_new"] = _randint(g, 1, pages * PAGE + 1, fresh).int()
        st["children"] = order[stay + fresh:stay + fresh + forks].clone()
        st["parents"] = order[_randint(g, 0, stay, forks)]
    else:
        rows, pages, pool = case["rows"], case["pages"], case["pool"]
        target = min(int(case["used"] * pool), pool - 1)
        used = _randint(g, 0, pages + 1, rows)
        fits = torch.cumsum(used, 0) <= target           # rows that the pool has room for; the others are empty
        ctx = torch.where(fits & (used > 0), used * PAGE - _randint(g, 0, PAGE, rows), torch.zeros_like(used))
        st["table"], st["refs"] = _tables(g, rows, pages, ctx, pool)
        st["caches"] = _caches(g, case, pool)
        st["new_table"], st["new_refs"] = torch.empty_like(st["table"]), torch.empty_like(st["refs"])
    return st


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _attend(st):
    """Attention in 32 bits over the selected latents."""
    q, pos = st["q"], st["idx"].long()
    seq = torch.arange(pos.shape[0], device=DEV) // st["tokens"]
    at = pos.clamp_min(0)
    page = st["table"][seq[:, None], at // PAGE].long()
    kv = _values(st["cache"][page * PAGE + at % PAGE])
    s = (q.float() @ kv.transpose(1, 2)) * SCALE
    s = s.masked_fill((pos < 0)[:, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return ((p @ kv[..., :LATENT]) / torch.where(total == 0, torch.ones_like(total), total)).to(torch.bfloat16)


def _copy(caches, src, dst, tokens=None):
    """Pages src -> dst of every cache, the first `tokens` tokens of each (all of them)."""
    for c in caches:
        paged = c.view(c.shape[0], -1, PAGE * c.shape[2]).view(torch.int64)      # whole words: a byte at a time is slow
        if tokens is None:
            paged[:, dst.long()] = paged[:, src.long()]
        else:
            paged = c.view(c.shape[0], -1, PAGE, c.shape[2])
            keep = (torch.arange(PAGE, device=DEV) < tokens[:, None])[None, :, :, None]
            paged[:, dst.long()] = torch.where(keep, paged[:, src.long()], paged[:, dst.long()])


def _pages(tokens):
    return (tokens + PAGE - 1) // PAGE


def _take(refs, count):
    """The `count` lowest free pages (count on the device: as many places as pages, those past the count are not used)."""
    free = refs == 0
    rank = torch.cumsum(free.int(), 0) - 1
    taken = free & (rank < count)
    fresh = torch.zeros(refs.shape[0] + 1, dtype=torch.int32, device=DEV)
    ids = torch.arange(refs.shape[0], dtype=torch.int32, device=DEV)
    fresh.scatter_(0, torch.where(taken, rank, torch.full_like(rank, refs.shape[0])).long(), ids)
    refs += taken.int()
    return fresh


def _turnover(st):
    table, ctx, refs = st["table"], st["ctx"], st["refs"]
    pages = table.shape[1]
    # finished and dropped rows
    gone = st["gone"].long()
    held = table[gone]
    refs.scatter_add_(0, held.clamp_min(0).flatten().long(), -(held >= 0).flatten().int())
    table[gone] = -1
    ctx[gone] = 0
    # new sequences
    new, n_new = st["new"].long(), st["n_new"]
    need = _pages(n_new)
    first = torch.cumsum(need, 0) - need
    fresh = _take(refs, need.sum())
    j = torch.arange(pages, device=DEV)
    table[new] = torch.where(j < need[:, None], fresh[(first[:, None] + j).clamp_max(refs.shape[0]).long()], torch.full((1, 1), -1, dtype=torch.int32, device=DEV))
    ctx[new] = n_new
    pos = torch.arange(st["max_new"], device=DEV)
    slots = table[new][:, pos // PAGE] * PAGE + (pos % PAGE).int()
    slots = torch.where(pos < n_new[:, None], slots, torch.full_like(slots, -1))
    # forks
    parents, children = st["parents"].long(), st["children"].long()
    lens = ctx[parents]
    tail = lens % PAGE
    part = (tail > 0).int()
    rank = torch.cumsum(part, 0) - part
    fresh = _take(refs, part.sum())
    rows = table[parents]
    whole = j < (lens // PAGE)[:, None]
    refs.scatter_add_(0, rows.clamp_min(0).flatten().long(), whole.flatten().int())
    last = (lens // PAGE).clamp_max(pages - 1).long()
    dst = fresh[rank.long()]
    src = rows.gather(1, last[:, None])[:, 0]
    kids = torch.where(whole, rows, torch.full_like(rows, -1))
    kids.scatter_(1, last[:, None], torch.where(part > 0, dst, kids.gather(1, last[:, None])[:, 0])[:, None])
    table[children] = kids
    ctx[children] = lens
    some = part > 0
    _copy(st["caches"], src[some], dst[some], tail[some])
    return {"table": table, "ctx": ctx, "refs": refs, "slots": slots, "caches": st["caches"]}


def _compact(st):
    table, refs = st["table"], st["refs"]
    live = refs > 0
    n_live = live.sum()
    ids = torch.arange(refs.shape[0], device=DEV)
    holes = torch.nonzero(~live & (ids < n_live))[:, 0]
    high = torch.nonzero(live & (ids >= n_live))[:, 0].flip(0)
    _copy(st["caches"], high, holes)
    remap = ids.int()
    remap[high] = holes.int()
    new_refs = torch.where(ids < n_live, refs, torch.zeros_like(refs))
    new_refs[holes] = refs[high]
    return {"table": torch.where(table >= 0, remap[table.clamp_min(0).long()], table), "refs": new_refs, "caches": st["caches"]}


def run(st):
    kind = st["kind"]
    if own:
        from llmdivedeep_b200 import ops
        if kind == "attn":
            return ops.sparse_mla_decode_paged(st["q"], st["cache"], st["table"], st["idx"], SCALE, tokens_per_seq=st["tokens"])
        if kind == "cache":
            ops.pack_latent4(st["kv"], st["cache"], st["slots"])
            return ops.unpack_latent4(st["cache"], st["ctx"], block_table=st["row"])
        if kind == "copy":
            ops.copy_pages(st["caches"], st["src"], st["dst"])
            return st["caches"]
        if kind == "turnover":
            table, ctx, refs = st["table"], st["ctx"], st["refs"]
            ops.free_pages(table, ctx, refs, st["gone"])
            slots = ops.extend_pages(table, ctx, refs, st["new"], st["n_new"], st["max_new"])
            ops.fork_pages(table, ctx, refs, st["parents"], st["children"], st["caches"])
            return {"table": table, "ctx": ctx, "refs": refs, "slots": slots, "caches": st["caches"]}
        table, refs = ops.compact_pages(st["table"], st["refs"], st["caches"], out=(st["new_table"], st["new_refs"]))
        return {"table": table, "refs": refs, "caches": st["caches"]}
    if kind == "attn":
        return _attend(st)
    if kind == "cache":
        st["cache"][st["slots"].long()] = _records(st["kv"])
        pos = torch.arange(st["ctx"], device=DEV)
        return _values(st["cache"][st["row"][pos // PAGE].long() * PAGE + pos % PAGE]).to(torch.bfloat16)
    if kind == "copy":
        _copy(st["caches"], st["src"], st["dst"])
        return st["caches"]
    return _turnover(st) if kind == "turnover" else _compact(st)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
PAGE_BYTES = PAGE * (K_BYTES + K_SCALE_BYTES + RECORD)


def work(case):
    kind = case["kind"]
    if kind == "attn":
        rows = case["batch"] * case["tokens"]
        ctx = case["ctx"] * (0.75 if case["ragged"] else 1.0)
        sel = min(ctx, case["topk"])
        keys = case["batch"] * min(ctx, sel * case["tokens"])            # latents that several tokens selected are read once
        return {"bytes": keys * RECORD + rows * (case["topk"] * 4 + case["heads"] * (1152 + 1024)), "flops": 2 * rows * sel * case["heads"] * 1088}
    if kind == "cache":
        wide = (LATENT + ROPE) * (2 if case["dtype"] == "bf16" else 4)
        return {"bytes": case["new"] * (wide + RECORD + 4) + case["ctx"] * (RECORD + (LATENT + ROPE) * 2), "flops": 0}
    if kind == "copy":
        return {"bytes": 2 * case["pairs"] * case["layers"] * PAGE_BYTES + 8 * case["pairs"], "flops": 0}
    if kind == "turnover":
        table = 4 * case["pages"] * (case["rows"] - case["stay"]) * 1.5          # rows emptied, rows filled to the half
        slots = 4 * case["fresh"] * case["pages"] * PAGE
        return {"bytes": 2 * case["forks"] * case["layers"] * PAGE_BYTES / 2 + table + slots + 8 * _pool_of(case), "flops": 0}
    used = min(case["used"], case["rows"] * (case["pages"] + 1) / 2 / case["pool"])
    moved = case["pool"] * used * (1 - used)
    return {"bytes": 2 * moved * case["layers"] * PAGE_BYTES + 8 * case["rows"] * case["pages"] + 8 * case["pool"], "flops": 0}


# ---- the same results in 64 bits ------------------------------------------------------------------------------------
def _decode_bits(rec):
    """Records [N, 416] -> rows in float64, bit by bit from the layout."""
    import numpy as np
    raw = np.ascontiguousarray(rec.cpu().numpy())
    out = np.empty((raw.shape[0], 576))
    for half in range(2):
        part = raw[:, 208 * half:208 * half + 208]
        bits = np.unpackbits(part[:, :128], axis=1, bitorder="little").reshape(-1, 64, 16).astype(np.int64)   # 16-bit halves of the words
        scale = part[:, 128:144].astype(np.int64)
        e, m = scale >> 3, scale & 7
        s = np.where(scale == 255, np.nan, (8 + m) * 2.0 ** (e - 18.0))
        for k in range(4):
            n = bits[:, :, MAG[k][0]] * 4 + bits[:, :, MAG[k][1]] * 2 + bits[:, :, MAG[k][2]]
            v = np.asarray(LEVELS, dtype=np.float64)[n] * np.where(bits[:, :, SIGN[k]] == 1, -1.0, 1.0)
            dim = (np.arange(64) // 2) * 8 + 2 * k + np.arange(64) % 2
            out[:, 256 * half + dim] = v * s[:, dim // 16]
        rope = part[:, 144:].copy().view(np.uint16).astype(np.uint32) << 16
        out[:, 512 + 32 * half:544 + 32 * half] = rope.view(np.float32)
    return torch.from_numpy(out)


def exact(case, seed):
    """Floating results in float64 from the same records and queries; None for pages, which are whole numbers."""
    kind = case["kind"]
    if kind == "cache":
        st = prepare(case, seed)
        x = st["kv"][:, :512].double().view(-1, 32, 16)
        grid = torch.tensor([(8 + m) * 2.0 ** (e - 18) for e in range(31) for m in range(8)], dtype=torch.float64, device=DEV)
        want = (x.abs().amax(-1) / 6).clamp(grid[0], grid[-1])
        up = torch.bucketize(want, grid).clamp_max(grid.numel() - 1)
        dn = (up - 1).clamp_min(0)
        a, b = want - grid[dn], grid[up] - want
        scale = grid[torch.where((a < b) | ((a == b) & (dn % 2 == 0)), dn, up)]
        levels = torch.tensor(LEVELS, dtype=torch.float64, device=DEV)
        y = (x / scale.unsqueeze(-1)).abs().unsqueeze(-1)
        far = (y - levels).abs() + torch.arange(8, device=DEV) % 2 * 1e-12       # the even level of two that are as near
        lat = levels[far.argmin(-1)] * scale.unsqueeze(-1) * torch.sign(x)
        rows = torch.cat((lat.view(-1, 512), st["kv"][:, 512:].to(torch.bfloat16).double()), -1)
        old = case["ctx"] - case["new"]
        pos = torch.arange(old, device=DEV)
        return torch.cat((_decode_bits(st["cache"][st["row"][pos // 64].long() * 64 + pos % 64]).to(DEV), rows))
    if kind != "attn" or case["batch"] * case["tokens"] * min(case["topk"], case["ctx"]) > 1 << 19:
        return None
    st = prepare(case, seed)
    out = torch.zeros(*st["q"].shape[:2], 512, dtype=torch.float64, device=DEV)
    for r in range(st["idx"].shape[0]):
        pos = st["idx"][r][st["idx"][r] >= 0].long()
        if pos.numel():
            at = st["table"][r // st["tokens"]][pos // 64].long() * 64 + pos % 64
            kv = _decode_bits(st["cache"][at]).to(DEV)
            p = torch.softmax(st["q"][r].double() @ kv.t() * SCALE, -1)
            out[r] = p @ kv[:, :512]
    return out
