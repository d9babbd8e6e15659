"""Operators of window layers and of drafted tokens, as performance cases: attention over a sliding window and the first tokens,
for prompts and over the paged latent caches; the indexer over a tree of drafted tokens; the acceptance of a path of them.

`run` computes a case with the package's entry points (`own`) or in plain torch, in 32 bits, with the same results.

A sequence of a batch holds ctx tokens in its pages, the last m of them drafted (m <= tokens); P = ctx - m.  Draft i sees the
P tokens before and, of the drafts, the ones that its 64-bit mask names, all before it, and itself; without masks the drafts are a
chain.  Position of a draft: P plus the number of drafts it sees, less one.

Kinds
  prefill   window attention of new tokens over the latents of their sequences, one behind a cached context or several packed
  decode    window attention of `tokens` query tokens for each of `batch` sequences over paged records of 656 or 416 bytes
  logits    the indexer's scores of `tokens` drafts for each of `batch` sequences over the paged key cache
  accept    `rows` sequences keep a path of their drafts: records of every layer move up, lengths and pages follow

Records: 656 bytes = 512 e4m3 values, 4 fp32 scales (128 values each), 64 bf16 rope values.  416 bytes = two halves of 208: the
codes of 256 values (128 bytes), the 16 scale bytes of their groups of 16, 32 bf16 rope values; a scale byte is five bits of exponent e and three of
mantissa m, (8 + m) 2^(e - 18); a 32-bit word holds eight codes, the even ones in its low half, `SIGN` and `MAG` say on which bits.
"""
import math
import random

import torch

own = False

DEV = "cuda"
PAGE = 64
LATENT, ROPE, GROUP = 512, 64, 16
SCALE = 192 ** -0.5
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
SIGN = (15, 12, 9, 14)                                  # of the value's 16-bit half
MAG = ((8, 7, 6), (5, 4, 3), (2, 1, 0), (11, 10, 13))   # bits of the level's number, highest first
K_BYTES, K_SCALE_BYTES = 128, 4                         # the indexer's key and its scale


def listed():
    return [
        # window layers of a prompt: a short one; a chunk behind 123K cached tokens; a rank's heads over several packed prompts; half of the heads
        {"name": "prefill_40", "kind": "prefill", "seqs": 1, "new": 40, "ctx": 40, "heads": 128, "window": 128, "first": 4},
        {"name": "prefill_8k_of_128k", "kind": "prefill", "seqs": 1, "new": 8192, "ctx": 131072, "heads": 128, "window": 4096, "first": 4},
        {"name": "prefill_packed_tp8", "kind": "prefill", "seqs": 12, "new": 9001, "ctx": 9001, "heads": 16, "window": 512, "first": 4},
        {"name": "prefill_2047_64", "kind": "prefill", "seqs": 1, "new": 2047, "ctx": 2500, "heads": 64, "window": 1024, "first": 128},
        # decode: one conversation; a long batch; drafted trees on a rank's heads; wide drafted trees of all heads
        {"name": "decode_1x2k", "kind": "decode", "batch": 1, "tokens": 1, "heads": 128, "ctx": 2000, "window": 512, "first": 4, "record": 416, "tree": False, "ragged": False},
        {"name": "decode_64x128k", "kind": "decode", "batch": 64, "tokens": 1, "heads": 128, "ctx": 131072, "window": 4096, "first": 64, "record": 656, "tree": False, "ragged": False},
        {"name": "tree_160x9k_tp8", "kind": "decode", "batch": 160, "tokens": 4, "heads": 16, "ctx": 9000, "window": 1024, "first": 4, "record": 416, "tree": True, "ragged": True},
        {"name": "tree_32x20k_13", "kind": "decode", "batch": 32, "tokens": 13, "heads": 128, "ctx": 20011, "window": 2048, "first": 64, "record": 656, "tree": True, "ragged": True},
        # the sparse layers' scores: drafts of one conversation; trees of four for a long batch
        {"name": "logits_1x2k_6", "kind": "logits", "batch": 1, "tokens": 6, "heads": 64, "ctx": 2000, "tree": True, "ragged": False},
        {"name": "logits_64x128k_4", "kind": "logits", "batch": 64, "tokens": 4, "heads": 64, "ctx": 131072, "tree": True, "ragged": False},
        # acceptance: a few conversations, two layers; a loaded server, sixteen layers
        {"name": "accept_8x2", "kind": "accept", "rows": 8, "tokens": 6, "pages": 20, "layers": 2},
        {"name": "accept_200x16", "kind": "accept", "rows": 200, "tokens": 13, "pages": 30, "layers": 16},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prefill", "prefill", "decode", "decode", "decode", "logits", "logits", "accept"])
    if kind == "prefill":
        heads = rng.choice([128, 128, 64, 32, 16, 8])
        window = _log(rng, 64, 4096)
        new = _log(rng, 1, 8192)
        if rng.random() < 0.4 and new > 40:
            seqs, ctx = rng.randint(2, min(24, new // 20)), new
        else:
            seqs, ctx = 1, _log(rng, new, 131072)
        return {"kind": kind, "seqs": seqs, "new": new, "ctx": ctx, "heads": heads, "window": window, "first": rng.choice([0, 1, 4, 64, 128])}
    if kind == "decode":
        batch = _log(rng, 1, 256)
        tokens = min(rng.choice([1, 1, 2, 3, 4, 7, 13, 24]), 512 // batch) or 1
        heads = rng.choice([128, 128, 64, 32, 16, 8])
        ctx = _log(rng, max(1, tokens), min(131072, 64 * 131072 // batch))
        window = _log(rng, 64, min(4096, 64 * 4096 // batch))
        return {"kind": kind, "batch": batch, "tokens": tokens, "heads": heads, "ctx": ctx, "window": window, "first": rng.choice([0, 1, 4, 64, 128]),
                "record": rng.choice([656, 416]), "tree": tokens > 1 and rng.random() < 0.7, "ragged": rng.random() < 0.7}
    if kind == "logits":
        batch = _log(rng, 1, 128)
        tokens = min(rng.choice([2, 3, 4, 5, 7, 8, 13, 24]), max(2, 256 // batch))
        heads = rng.choice([64, 64, 32, 16])
        return {"kind": kind, "batch": batch, "tokens": tokens, "heads": heads, "ctx": _log(rng, tokens, min(131072, 256 * 131072 // (batch * tokens))),
                "tree": rng.random() < 0.7, "ragged": rng.random() < 0.7}
    rows = _log(rng, 1, 200)
    tokens = rng.choice([1, 2, 4, 6, 13, 24])
    return {"kind": kind, "rows": rows, "tokens": tokens, "pages": rng.randint(2, 30), "layers": rng.choice([1, 2, 4, 8, 16])}


# ---- records, in plain torch ----------------------------------------------------------------------------------------
def _records4(kv):
    """Rows [N, 576] fp32 -> uint8 [N, 416]."""
    g = kv[:, :LATENT].view(-1, LATENT // GROUP, GROUP)
    want = (g.abs().amax(-1) / 6).clamp(2.0 ** -15, 61440.0)
    e = torch.frexp(want)[1] - 1
    scale = torch.round(torch.ldexp(want, 3 - e)) * torch.exp2((e - 3).float())
    e = torch.frexp(scale)[1] - 1
    byte = (e + 15) * 8 + torch.ldexp(scale, 3 - e).int() - 8
    steps = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=kv.device)
    n = torch.bucketize((g / scale.unsqueeze(-1)).abs(), steps).view(-1, LATENT // 8, 4, 2).int()
    sign = torch.signbit(g).view(-1, LATENT // 8, 4, 2).int()
    half = 0
    for k in range(4):
        half = half | (sign[:, :, k] << SIGN[k])
        for bit, at in zip((2, 1, 0), MAG[k]):
            half = half | (((n[:, :, k] >> bit) & 1) << at)
    word = torch.where(half >= 1 << 15, half - (1 << 16), half).to(torch.int16).view(-1, LATENT // 4).view(torch.uint8).view(-1, 2, 128)
    rope = kv[:, LATENT:].to(torch.bfloat16).contiguous().view(torch.uint8).view(-1, 2, 64)
    return torch.cat((word, byte.to(torch.uint8).view(-1, 2, 16), rope), -1).reshape(-1, 416)


def _records8(kv):
    """Rows [N, 576] fp32 -> uint8 [N, 656]."""
    g = kv[:, :LATENT].view(-1, 4, 128)
    scale = g.abs().amax(-1).clamp_min(1e-6) / 448
    code = (g / scale.unsqueeze(-1)).to(torch.float8_e4m3fn).view(torch.uint8).view(-1, LATENT)
    rope = kv[:, LATENT:].to(torch.bfloat16).contiguous().view(torch.uint8).view(-1, 128)
    return torch.cat((code, scale.view(torch.uint8).view(-1, 16), rope), -1)


def _values(rec):
    """Records uint8 [..., 656 or 416] -> rows fp32 [..., 576]."""
    lead, rec = rec.shape[:-1], rec.reshape(-1, rec.shape[-1])
    if rec.shape[1] == 656:
        lat = rec[:, :512].contiguous().view(torch.float8_e4m3fn).float().view(-1, 4, 128)
        lat = lat * rec[:, 512:528].contiguous().view(torch.float32).unsqueeze(-1)
        rope = rec[:, 528:].contiguous().view(torch.bfloat16).float()
        return torch.cat((lat.reshape(-1, LATENT), rope), -1).view(*lead, LATENT + ROPE)
    h = rec.view(-1, 2, 208)
    w = h[..., :128].contiguous().view(torch.int16).view(-1, LATENT // 8, 2).int()      # word, half of the word
    levels = torch.tensor(LEVELS, device=rec.device)
    out = torch.empty(w.shape[0], LATENT // 8, 4, 2, device=rec.device)
    for k in range(4):
        n = (((w >> MAG[k][0]) & 1) * 2 + ((w >> MAG[k][1]) & 1)) * 2 + ((w >> MAG[k][2]) & 1)
        out[:, :, k] = levels[n] * (1 - 2 * ((w >> SIGN[k]) & 1))
    b = h[..., 128:144].int()
    scale = (8 + b % 8) * torch.exp2((b // 8 - 18).float())
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
    """Bytes that need not mean anything: records are moved as they are."""
    n = math.prod(shape)
    return torch.randint(-2 ** 62, 2 ** 62, (-(-n // 8),), device=DEV, generator=g).view(torch.uint8)[:n].view(*shape)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _drafts(rng, case, batch, st):
    """What a drafting step hands on: how many drafts each sequence has, and their trees."""
    n = case["tokens"]
    st["n_new"] = st["tree"] = None
    m = [rng.randint(1, n) if case["ragged"] else n for _ in range(batch)]
    if n > 1 and case["ragged"]:
        st["n_new"] = _ints(m)
    if case["tree"]:
        masks = []
        for _ in range(batch):
            row = []
            for i in range(n):
                up = rng.randint(-1, i - 1)              # the draft before it on its path; -1: the cached token
                bits = (row[up] if up >= 0 else 0) | (1 << i)
                row.append(bits)
            masks.append([b - (1 << 64) if b >= 1 << 63 else b for b in row])
        st["tree"] = _ints(masks, torch.int64)
    return m


def prepare(case, seed):
    g, rng, kind = _gen(seed), random.Random(seed), case["kind"]
    st = {"kind": kind, "case": case}
    if kind == "prefill":
        new, ctx, seqs = case["new"], case["ctx"], case["seqs"]
        cuts = [0, *sorted(rng.sample(range(1, new), seqs - 1)), new]
        # first row, last row, first key, last key of each sequence
        st["spans"] = [(a, b, a if seqs > 1 else 0, b if seqs > 1 else ctx) for a, b in zip(cuts, cuts[1:])]
        st["ks"] = torch.cat([torch.full((b - a,), k0, dtype=torch.int32) for a, b, k0, k1 in st["spans"]]).to(DEV)
        st["ke"] = torch.cat([torch.arange(k1 - (b - a) + 1, k1 + 1, dtype=torch.int32) for a, b, k0, k1 in st["spans"]]).to(DEV)
        st["q"] = _randn(g, new, case["heads"], LATENT + ROPE, dtype=torch.bfloat16)
        st["kv"] = _randn(g, ctx, LATENT + ROPE, dtype=torch.bfloat16)
    elif kind in ("decode", "logits"):
        batch, tokens, ctx = case["batch"], case["tokens"], case["ctx"]
        pages = -(-ctx // PAGE)
        n = batch * pages * PAGE
        m = _drafts(rng, case, batch, st)
        lens = [rng.randint(max(ctx // 2, k), ctx) if case["ragged"] else ctx for k in m]
        st["ctx_len"] = _ints(lens)
        st["table"] = torch.randperm(batch * pages, device=DEV, generator=g).int().view(batch, pages)
        if kind == "decode":
            some = (_records8 if case["record"] == 656 else _records4)(_randn(g, min(n, 1 << 15), LATENT + ROPE))
            st["cache"] = some[_randint(g, 0, some.shape[0], n)] if n > some.shape[0] else some
            st["q"] = _randn(g, batch * tokens, case["heads"], LATENT + ROPE, dtype=torch.bfloat16)
        else:
            def e4m3(x):
                scale = x.abs().amax(-1).clamp_min(1e-6) / 448
                return (x / scale.unsqueeze(-1)).to(torch.float8_e4m3fn), scale
            k8, ksc = e4m3(_randn(g, min(n, 1 << 17), 128))
            if n > k8.shape[0]:
                at = _randint(g, 0, k8.shape[0], n)
                k8, ksc = k8.view(torch.uint8)[at].view(torch.float8_e4m3fn), ksc[at]
            q8, qsc = e4m3(_randn(g, batch * tokens, case["heads"], 128))
            st["k8"], st["kscale"], st["q8"] = k8, ksc, q8
            st["w"] = _randn(g, batch * tokens, case["heads"]) * qsc * (128 * case["heads"]) ** -0.5
            st["out"] = torch.full((batch * tokens, (ctx + 3) // 4 * 4), -math.inf, device=DEV)
    else:
        rows, tokens, pages, layers = case["rows"], case["tokens"], case["pages"], case["layers"]
        pool = rows * pages + 7
        ctx = [rng.randint(tokens, pages * PAGE) for _ in range(rows)]
        used = torch.arange(pages, device=DEV) < (_ints(ctx)[:, None] + PAGE - 1) // PAGE
        ids = torch.randperm(pool, device=DEV, generator=g)[:rows * pages].int().view(rows, pages)
        table = torch.where(used, ids, torch.full_like(ids, -1))
        refs = torch.zeros(pool, dtype=torch.int32, device=DEV)
        refs[table[used].long()] = 1
        # one buffer for the three, as the drafting step left them, and one for the step to work on
        st["before"] = torch.cat((table.flatten(), _ints(ctx), refs))
        st["now"] = st["before"].clone()
        st["table"], st["ctx_len"], st["refs"] = st["now"][:rows * pages].view(rows, pages), st["now"][rows * pages:rows * pages + rows], st["now"][rows * pages + rows:]
        st["rows"] = _ints(rng.sample(range(rows), rows))
        m = [rng.randint(1, tokens) for _ in range(rows)]
        keep = [rng.randint(0, k) for k in m]
        path = [sorted(rng.sample(range(k), c)) + [-1] * (tokens - c) for k, c in zip(m, keep)]
        st["n_new"], st["n_keep"], st["path"] = _ints(m), _ints(keep), _ints(path)
        st["caches"] = [_rand_bytes(g, layers, pool * PAGE, b) for b in (K_BYTES, K_SCALE_BYTES, 416)]
    return st


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _softmax_av(s, seen, v):
    """Softmax over the places of s [..., rows, heads, L] that are seen, times v [..., L, 512]; zeros where none is."""
    s = s.masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)))
    total = p.sum(-1, keepdim=True)
    o = (p.flatten(-3, -2) @ v).view(*p.shape[:-1], LATENT)
    return o.div_(torch.where(total == 0, torch.ones_like(total), total))


def _prefill(st):
    """Rows of a sequence in stretches whose scores fit, each against its sequence's first keys and the keys of its windows."""
    case, q = st["case"], st["q"]
    W, first, H = case["window"], case["first"], case["heads"]
    out = torch.empty(*q.shape[:2], LATENT, dtype=torch.bfloat16, device=DEV)
    most = max(1, (1 << 28) // (H * (W + first + 256)))
    for r0, r1, k0, k1 in st["spans"]:
        for a in range(r0, r1, most):
            b = min(r1, a + most)
            lo, hi = max(k0, k1 - (r1 - a) + 1 - W), k1 - (r1 - b)
            head = min(k0 + first, lo)                   # first keys that the windows' stretch does not have
            kv = torch.cat((st["kv"][k0:head], st["kv"][lo:hi])).float()
            pos = torch.cat((torch.arange(k0, head, device=DEV), torch.arange(lo, hi, device=DEV)))
            ke = st["ke"][a:b, None]
            seen = (pos < ke) & ((pos >= ke - W) | (pos < k0 + first))
            s = ((q[a:b].float().reshape(-1, LATENT + ROPE) @ kv.t()) * SCALE).view(b - a, H, -1)
            out[a:b] = _softmax_av(s, seen[:, None], kv[:, :LATENT]).to(torch.bfloat16)
    return out


def _paths(st):
    """Of every draft [B, n]: whether it is one, its tokens before the drafts [B], which drafts it sees [B, n, n] and their positions."""
    case = st["case"]
    B, n = case["batch"], case["tokens"]
    m = st["n_new"] if st["n_new"] is not None else st["ctx_len"].clamp_max(n)
    i = torch.arange(n, device=DEV)
    tree = torch.ones(B, n, n, dtype=torch.bool, device=DEV) if st["tree"] is None else ((st["tree"][:, :, None] >> i) & 1).bool()
    sees = (tree & (i < i[:, None])) | (i == i[:, None])
    P = st["ctx_len"] - m
    at = P[:, None, None] + torch.cumsum(sees.int(), -1) - 1             # of the drafts on a path, along it
    return i < m[:, None], P, sees, at


def _decode(st):
    case = st["case"]
    B, n, W, first = case["batch"], case["tokens"], case["window"], case["first"]
    live, P, sees, at = _paths(st)
    L = min(W + n, case["ctx"])                                          # keys that the windows of a sequence reach over
    lo = (st["ctx_len"] - L).clamp_min(0)
    head = torch.arange(min(first, case["ctx"]), device=DEV).expand(B, -1)
    pos = torch.cat((torch.where(head < lo[:, None], head, torch.full_like(head, -1)), lo[:, None] + torch.arange(L, device=DEV)), 1)
    pos = torch.where(pos < st["ctx_len"][:, None], pos, torch.full_like(pos, -1))
    page = st["table"].gather(1, (pos.clamp_min(0) // PAGE)).long()
    kv = _values(st["cache"][page * PAGE + pos.clamp_min(0) % PAGE])     # [B, keys, 576]
    own_at = at[:, :, -1]                                                # the draft's position [B, n]
    d = (pos - P[:, None]).clamp(0, n - 1)[:, None].expand(-1, n, -1)    # which draft a key is
    before = pos[:, None] < P[:, None, None]
    where = torch.where(before, pos[:, None].expand(-1, n, -1), at.gather(2, d))
    seen = (before | sees.gather(2, d)) & ((where < first) | (where > own_at[:, :, None] - W)) & (pos >= 0)[:, None] & live[:, :, None]
    q = st["q"].float().view(B, -1, LATENT + ROPE)
    s = ((q @ kv.transpose(1, 2)) * SCALE).view(B, n, case["heads"], -1)
    o = _softmax_av(s, seen[:, :, None], kv[..., :LATENT])
    return o.reshape(B * n, case["heads"], LATENT).to(torch.bfloat16)


def _logits(st):
    case = st["case"]
    B, n, H, ctx = case["batch"], case["tokens"], case["heads"], case["ctx"]
    live, P, sees, _ = _paths(st)
    pos = torch.arange(ctx, device=DEV)
    rows = st["table"][:, pos // PAGE].long() * PAGE + pos % PAGE
    k = st["k8"].view(torch.uint8)[rows].view(torch.float8_e4m3fn).float()
    s = (st["q8"].float().view(B, n * H, 128) @ k.transpose(1, 2)).clamp_min_(0).view(B, n, H, ctx)
    s = (st["w"].view(B, n, 1, H) @ s).squeeze(2).mul_(st["kscale"][rows][:, None])
    d = (pos - P[:, None]).clamp(0, n - 1)[:, None].expand(-1, n, -1)
    seen = (pos < st["ctx_len"][:, None])[:, None] & ((pos < P[:, None])[:, None] | sees.gather(2, d)) & live[:, :, None]
    return s.masked_fill_(~seen, -math.inf).view(B * n, ctx)


def _accept(st):
    table, ctx, refs, rows = st["table"], st["ctx_len"], st["refs"], st["rows"].long()
    P = ctx[rows] - st["n_new"]
    k = torch.arange(st["path"].shape[1], device=DEV)
    i, k = torch.nonzero(k < st["n_keep"][:, None], as_tuple=True)
    src, dst = P[i] + st["path"][i, k], P[i] + k
    src, dst = (table[rows[i], (p // PAGE).long()].long() * PAGE + p % PAGE for p in (src, dst))
    for c in st["caches"]:
        words = c.view(torch.int32)
        words[:, dst] = words[:, src]
    ctx[rows] = (P + st["n_keep"]).int()
    gone = (torch.arange(table.shape[1], device=DEV) >= ((ctx + PAGE - 1) // PAGE)[:, None]) & (table >= 0)
    refs.scatter_add_(0, table.clamp_min(0).flatten().long(), -gone.flatten().int())
    table.masked_fill_(gone, -1)
    return {"table": table, "ctx": ctx, "refs": refs, "caches": st["caches"]}


def run(st):
    kind, case = st["kind"], st["case"]
    if own:
        from llmdivedeep_b200 import ops
        if kind == "prefill":
            return ops.window_mla_prefill(st["q"], st["kv"], st["ks"], st["ke"], case["window"], case["first"], SCALE)
        if kind == "decode":
            return ops.window_mla_decode_paged(st["q"], st["cache"], st["table"], st["ctx_len"], case["window"], case["first"], SCALE,
                                               tokens_per_seq=case["tokens"], n_new=st["n_new"], tree=st["tree"])
        if kind == "logits":
            return ops.fp8_paged_mqa_logits(st["q8"], st["w"], st["k8"], st["kscale"], st["table"], st["ctx_len"], case["ctx"], out=st["out"],
                                            tokens_per_seq=case["tokens"], n_new=st["n_new"], tree=st["tree"])
        st["now"].copy_(st["before"])
        ops.accept_drafts(st["table"], st["ctx_len"], st["refs"], st["rows"], st["n_new"], st["path"], st["n_keep"], st["caches"])
        return {"table": st["table"], "ctx": st["ctx_len"], "refs": st["refs"], "caches": st["caches"]}
    if kind == "prefill":
        return _prefill(st)
    if kind == "decode":
        return _decode(st)
    if kind == "logits":
        return _logits(st)
    st["now"].copy_(st["before"])
    return _accept(st)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "prefill":
        new, ctx, W, first, H, seqs = (case[k] for k in ("new", "ctx", "window", "first", "heads", "seqs"))
        per = new / seqs                                                 # packed sequences: as if of one length
        past = ctx - new if seqs == 1 else 0
        most = min(W + first, past + per)
        rising = max(0.0, min(per, most - past))                         # rows whose windows are not full yet
        pairs = seqs * (rising * (past + rising / 2) + (per - rising) * most)
        keys = seqs * min(past + per, W + first + per)
        return {"bytes": new * H * (1152 + 1024) + keys * 1152, "flops": 2 * pairs * H * 1088}
    if kind == "decode":
        n = (case["tokens"] + 1) / 2 if case["ragged"] and case["tokens"] > 1 else case["tokens"]
        ctx = case["ctx"] * (0.75 if case["ragged"] else 1.0)
        seen = min(ctx, case["window"] + case["first"])
        keys = case["batch"] * min(ctx, seen + n - 1)
        return {"bytes": keys * case["record"] + case["batch"] * n * case["heads"] * (1152 + 1024), "flops": 2 * case["batch"] * n * seen * case["heads"] * 1088}
    if kind == "logits":
        n = (case["tokens"] + 1) / 2 if case["ragged"] else case["tokens"]
        ctx = case["ctx"] * (0.75 if case["ragged"] else 1.0)
        rows = case["batch"] * n
        return {"bytes": case["batch"] * ctx * (K_BYTES + K_SCALE_BYTES) + rows * (case["heads"] * 132 + ctx * 4), "flops": 2 * rows * ctx * case["heads"] * 128}
    moved = case["rows"] * (case["tokens"] + 1) / 4
    return {"bytes": 2 * moved * case["layers"] * (K_BYTES + K_SCALE_BYTES + 416) + 8 * case["rows"] * (case["tokens"] + 4), "flops": 0}


# ---- the same results in 64 bits ------------------------------------------------------------------------------------
def _decode_bits(rec):
    """Records [N, 656 or 416] -> rows in float64, from the layout."""
    import numpy as np
    raw = np.ascontiguousarray(rec.cpu().numpy())
    out = np.empty((raw.shape[0], 576))
    if raw.shape[1] == 656:
        b = raw[:, :512].astype(np.int64)
        e, m = (b >> 3) & 15, b & 7
        v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0)) * np.where(b >> 7, -1.0, 1.0)
        out[:, :512] = v * np.repeat(raw[:, 512:528].copy().view(np.float32).astype(np.float64), 128, axis=1)
        out[:, 512:] = (raw[:, 528:].copy().view(np.uint16).astype(np.uint32) << 16).view(np.float32)
        return torch.from_numpy(out)
    for half in range(2):
        part = raw[:, 208 * half:208 * half + 208]
        bits = np.unpackbits(part[:, :128], axis=1, bitorder="little").reshape(-1, 64, 16).astype(np.int64)   # 16-bit halves of the words
        scale = part[:, 128:144].astype(np.int64)
        s = (8 + (scale & 7)) * 2.0 ** ((scale >> 3) - 18.0)
        for k in range(4):
            n = bits[:, :, MAG[k][0]] * 4 + bits[:, :, MAG[k][1]] * 2 + bits[:, :, MAG[k][2]]
            v = np.asarray(LEVELS, dtype=np.float64)[n] * np.where(bits[:, :, SIGN[k]] == 1, -1.0, 1.0)
            dim = (np.arange(64) // 2) * 8 + 2 * k + np.arange(64) % 2
            out[:, 256 * half + dim] = v * s[:, dim // 16]
        rope = part[:, 144:].copy().view(np.uint16).astype(np.uint32) << 16
        out[:, 512 + 32 * half:544 + 32 * half] = rope.view(np.float32)
    return torch.from_numpy(out)


def _seen_by(st, b):
    """(draft, positions it sees) of sequence b, each from the draft's path token by token."""
    case = st["case"]
    n, ctx = case["tokens"], int(st["ctx_len"][b])
    m = int(st["n_new"][b]) if st["n_new"] is not None else min(n, ctx)
    P = ctx - m
    for i in range(m):
        mask = int(st["tree"][b, i]) if st["tree"] is not None else -1
        path = torch.cat((torch.arange(P), torch.tensor([P + j for j in range(i) if mask >> j & 1] + [P + i])))
        if "window" in case:
            k = torch.arange(path.numel())
            path = path[(k < case["first"]) | (k > path.numel() - 1 - case["window"])]
        yield i, path.to(DEV)


def exact(case, seed):
    """Floating results in float64 from the same inputs; None for what moves, which are whole numbers, and for large cases."""
    kind = case["kind"]
    if kind == "accept":
        return None
    n = case.get("tokens", 1)
    if kind == "prefill":
        st = prepare(case, seed)
        q, kv, ks, ke = st["q"], st["kv"].double(), st["ks"].tolist(), st["ke"].tolist()
        out = torch.zeros(*q.shape[:2], 512, dtype=torch.float64, device=DEV)
        step = max(1, min(64, 8192 // case["heads"]))
        a = 0
        while a < len(ks):                                               # rows of one sequence, a few at a time, every key between
            b = a + 1
            while b < len(ks) and b - a < step and ks[b] == ks[a]:
                b += 1
            at = list(range(ks[a], min(ks[a] + case["first"], ke[b - 1])))
            at = torch.tensor(at + list(range(max(ks[a] + len(at), ke[a] - case["window"]), ke[b - 1])), device=DEV)
            end = torch.tensor(ke[a:b], device=DEV)[:, None, None]
            hidden = (at >= end) | ((at < end - case["window"]) & (at >= ks[a] + case["first"]))
            s = torch.einsum("thd,sd->ths", q[a:b].double(), kv[at]) * SCALE
            out[a:b] = torch.einsum("ths,sd->thd", torch.softmax(s.masked_fill_(hidden, -math.inf), -1), kv[at, :512])
            a = b
        return out
    if kind == "decode":
        if case["batch"] * min(case["ctx"], case["window"] + case["first"] + n) > 300000 or case["batch"] * n > 1024:
            return None
        st = prepare(case, seed)
        out = torch.zeros(*st["q"].shape[:2], 512, dtype=torch.float64, device=DEV)
        for b in range(case["batch"]):
            paths = list(_seen_by(st, b))
            pos = torch.unique(torch.cat([path for _, path in paths])) if paths else None
            kv = _decode_bits(st["cache"][st["table"][b][pos // 64].long() * 64 + pos % 64]).to(DEV) if paths else None
            for i, path in paths:
                x = kv[torch.searchsorted(pos, path)]
                out[b * n + i] = torch.softmax(st["q"][b * n + i].double() @ x.t() * SCALE, -1) @ x[:, :512]
        return out
    if case["batch"] * n * case["ctx"] > 1 << 26:
        return None
    st = prepare(case, seed)
    out = torch.full((case["batch"] * n, case["ctx"]), -math.inf, dtype=torch.float64, device=DEV)
    for b in range(case["batch"]):
        for i, pos in _seen_by(st, b):
            at = st["table"][b][pos // 64].long() * 64 + pos % 64
            s = torch.relu(st["k8"].view(torch.uint8)[at].view(torch.float8_e4m3fn).double() @ st["q8"][b * n + i].double().t())
            out[b * n + i, pos] = (s @ st["w"][b * n + i].double()) * st["kscale"][at].double()
    return out
