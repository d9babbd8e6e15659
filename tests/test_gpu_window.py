"""Attention over a sliding window and the first tokens, for prompts and over the paged latent caches, against 64 bits."""
import random

import pytest
import torch

from llmdivedeep_b200 import layer, ops
from oracle import drafts_oracle as D

pytestmark = pytest.mark.gpu
SCALE = 192 ** -0.5
# The output's rounding to bf16 is 1.7e-3 of it (2-norm: half a step of 2^-8, uniform over a binade), that of P to bf16 as much again of a sum of
# many terms, that of the exchanged half scores to fp16 less than half of it for scores of order one.  Three times their root sum of
# squares; a single value by 2^-6 of the row's largest.
REL, MOST = 7.5e-3, 2.0 ** -6


def check(out, want, rel=REL, most=MOST):
    got, want = out.double(), want.to(out.device)
    err, size = (got - want).norm(dim=-1), want.norm(dim=-1)
    assert bool((err <= rel * size).all()), float((err / size.clamp_min(1e-30)).max())
    assert bool(((got - want).abs().amax(-1) <= most * want.abs().amax(-1)).all())


def rows(n, *shape, seed=0, gain=1.0):
    g = torch.Generator().manual_seed(seed + n)
    return (torch.randn(n, *shape, 576, generator=g) * gain).to(torch.bfloat16).cuda()


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32).cuda()


# heads that fill a tile, share one, and lie across two; windows shorter and longer than a block of keys; first tokens that overlap the window
@pytest.mark.parametrize("T,S,H,window,first", [
    (1, 1, 128, 1, 0), (1, 1, 1, 5, 3), (40, 40, 128, 128, 4), (130, 300, 128, 64, 0), (7, 500, 128, 200, 70), (200, 200, 16, 50, 4), (77, 400, 16, 130, 64),
    (300, 300, 1, 40, 3), (50, 90, 3, 33, 5), (33, 700, 64, 128, 128), (9, 2100, 8, 2048, 4), (5, 130, 256, 100, 1), (7, 150, 192, 64, 0), (21, 333, 100, 65, 2),
    (400, 400, 128, 5, 2), (500, 500, 128, 64, 0), (300, 3000, 128, 130, 4), (131, 400, 2, 70, 1),
    (65, 65, 32, 1, 0), (64, 1000, 40, 1000, 0), (3, 200, 128, 1 << 30, 0), (3, 200, 16, 7, 1 << 30), (150, 5000, 128, 4096, 4), (2, 9000, 16, 1 << 31, 0),
])
def test_prompts(T, S, H, window, first):
    q, kv = rows(T, H, seed=S), rows(S, seed=H)
    out = torch.full((T, H, 512), 9.0, dtype=torch.bfloat16, device="cuda")
    assert ops.window_mla_prefill(q, kv, None, None, window, first, SCALE, out=out) is out
    ops.check_status("cuda")
    check(out, D.attend(q, kv, D.prompt_sees(T, S, window, first), SCALE))


@pytest.mark.parametrize("H", [128, 16, 48, 1])
@pytest.mark.parametrize("window,first", [(40, 3), (200, 0), (64, 64)])
def test_packed_prompts_and_rows_that_see_nothing(H, window, first):
    """Sequences side by side, of one token and of many, rows without a window, windows that begin before 0 or end behind S."""
    lens = [1, 70, 3, 130, 64, 2, 33]
    ks = torch.cat([torch.full((n,), sum(lens[:i])) for i, n in enumerate(lens)])
    ke = torch.arange(sum(lens)) + 1
    S = sum(lens)
    ke[5], ks[6], ke[6] = ks[5], 50, 20
    ks[0], ke[-1] = -7, S + 9
    q, kv = rows(S, H), rows(S, seed=3)
    out = ops.window_mla_prefill(q, kv, i32(ks), i32(ke), window, first, SCALE)
    ops.check_status("cuda")
    want = D.attend(q, kv, D.prompt_sees(S, S, window, first, ks, ke), SCALE)
    check(out, want)
    assert bool((out[5:7] == 0).all())


@pytest.mark.parametrize("H", [128, 16, 5])
@pytest.mark.parametrize("first", [1, 4, 8, 9, 16, 17])
def test_first_tokens_and_windows_that_end_anywhere_in_a_block(H, first):
    """Windows whose last block has room for the first tokens, just not, or none of its own; two sequences of them side by side, rows between that see nothing."""
    n, S, at = 24, 900, 400                               # a sequence of 400 tokens and one of 500
    g = torch.Generator().manual_seed(first)
    for window in (33, 64 - first, 65 - first, 64, 65, 129, 150):
        last = torch.cat((torch.arange(370, 370 + n), at + torch.arange(200, 200 + n)))
        ks = torch.cat((torch.zeros(n), torch.full((n,), at))).long()
        ke = last + 1
        none = torch.randperm(2 * n, generator=g)[:5]
        ke[none] = ks[none]
        q, kv = rows(2 * n, H, seed=window), rows(S, seed=first)
        sees = D.prompt_sees(2 * n, S, window, first, ks, ke)
        check(ops.window_mla_prefill(q, kv, i32(ks), i32(ke), window, first, SCALE), D.attend(q, kv, sees, SCALE))
        for bad in (0, at + first - 1, at + first, 372 - window, 394, 600 - window):      # keys that are no numbers: first tokens, one behind them, ends of windows
            dirty = kv.clone()
            dirty[bad, 300], dirty[bad, 30] = float("nan"), float("inf")
            out = ops.window_mla_prefill(q, dirty, i32(ks), i32(ke), window, first, SCALE)
            touched = sees[:, bad].cuda()
            assert bool((~out[touched].isfinite()).flatten(1).any(1).all())
            check(out[~touched], D.attend(q, kv, sees, SCALE).cuda()[~touched])
        ops.check_status("cuda")


@pytest.mark.parametrize("H", [128, 16, 5])
def test_rows_in_any_order(H):
    """Rows of a rank that has every other stretch of a sequence, and rows in no order at all."""
    S, window, first = 700, 90, 4
    for pos in (torch.cat([torch.arange(a, a + 50) for a in range(0, 700, 100)]), torch.randperm(S, generator=torch.Generator().manual_seed(1))[:260]):
        q, kv = rows(len(pos), H), rows(S, seed=9)
        out = ops.window_mla_prefill(q, kv, None, i32(pos + 1), window, first, SCALE)
        ops.check_status("cuda")
        check(out, D.attend(q, kv, D.prompt_sees(len(pos), S, window, first, None, pos + 1), SCALE))


@pytest.mark.parametrize("H", [128, 16])
@pytest.mark.parametrize("T", [12, 400])
def test_few_and_many_rows_with_and_without_room_for_parts(H, T):
    q, kv = rows(T, H, seed=1), rows(900, seed=2)
    want = D.attend(q, kv, D.prompt_sees(T, 900, 500, 70), SCALE)
    for room in (0, 100000, None):
        ws = None if room is None else torch.empty(room, dtype=torch.uint8, device="cuda")
        check(ops.window_mla_prefill(q, kv, None, None, 500, 70, SCALE, workspace=ws), want)
    ops.check_status("cuda")


@pytest.mark.parametrize("H", [128, 16])
@pytest.mark.parametrize("gain", [4.0, 30.0])
def test_wide_scores(H, gain):
    """Rows that one key takes over.  A half score that is sent in fp16 is off by 2^-11 of itself at most: with scores of |q| |k| / 2 = gain * 12
    a half in the mean, four sigma of them and the scale, an exponent of `score` is off by 2^-11 of that, and P by as much, relatively."""
    q, kv = rows(70, H, seed=5, gain=gain), rows(600, seed=6)
    score = 4 * gain * 17 * SCALE
    check(ops.window_mla_prefill(q, kv, None, None, 300, 4, SCALE), D.attend(q, kv, D.prompt_sees(70, 600, 300, 4), SCALE), REL + 2 * score * 2.0 ** -11,
          MOST + 4 * score * 2.0 ** -11)
    ops.check_status("cuda")


@pytest.mark.parametrize("H", [128, 64, 16, 3])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_a_row_does_not_see_leaves_it_as_it_is(H, bad):
    """A key that some rows see and others do not, keys of another sequence, keys behind the last: rows that see it are no numbers, the others right."""
    T, S, window, first = 90, 260, 60, 3
    ks = torch.cat((torch.zeros(50), torch.full((40,), 160))).long()
    ke = torch.cat((torch.arange(100, 150), torch.arange(201, 241))).long()
    q, kv = rows(T, H, seed=8), rows(S, seed=8)
    for at, dim in ((1, 700 % 576), (120, 511), (230, 0), (155, 300), (250, 20), (161, 256)):
        dirty = kv.clone()
        dirty[at, dim] = bad
        sees = D.prompt_sees(T, S, window, first, ks, ke)
        out = ops.window_mla_prefill(q, dirty, i32(ks), i32(ke), window, first, SCALE)
        ops.check_status("cuda")
        touched = sees[:, at].cuda()
        assert bool((~out[touched].isfinite()).flatten(1).any(1).all())
        check(out[~touched], D.attend(q, kv, sees, SCALE).cuda()[~touched])


@pytest.mark.parametrize("H", [16, 40])
def test_numbers_that_are_none_in_parts(H):
    """Few rows over many keys: the keys are cut into parts, and a part's rows are done again by themselves."""
    q, kv = rows(20, H, seed=3), rows(900, seed=4)
    sees = D.prompt_sees(20, 900, 600, 70)
    want = D.attend(q, kv, sees, SCALE)
    for at in (282, 290, 300, 885, 899):
        dirty = kv.clone()
        dirty[at, 40], dirty[at, 400] = float("nan"), float("inf")
        out = ops.window_mla_prefill(q, dirty, None, None, 600, 70, SCALE)
        ops.check_status("cuda")
        touched = sees[:, at].cuda()
        assert bool((~out[touched].isfinite()).flatten(1).any(1).all())
        check(out[~touched], want[~touched])


@pytest.mark.parametrize("T", [600, 7402])
def test_numbers_that_are_none_in_every_unit(T):
    """Every second key is none, every row sees itself alone: as many rows to be done again as there are units, more than a list of them holds."""
    q, kv = rows(T, 64, seed=1), rows(T, seed=2)
    kv[1::2] = float("nan")
    out = ops.window_mla_prefill(q, kv, None, None, 1, 0, SCALE)
    ops.check_status("cuda")
    assert torch.equal(out[::2], kv[::2, None, :512].expand(-1, 64, -1)) and bool(out[1::2].isnan().all())


def test_a_query_that_is_no_number_is_its_rows_own_affair():
    q, kv = rows(300, 16, seed=1), rows(3000, seed=2)
    want = ops.window_mla_prefill(q, kv, None, None, 2000, 4, SCALE)
    dirty = q.clone()
    dirty[7, 3], dirty[120] = float("nan"), float("inf")
    out = ops.window_mla_prefill(dirty, kv, None, None, 2000, 4, SCALE)
    ops.check_status("cuda")
    keep = torch.ones(300, 16, dtype=torch.bool, device="cuda")
    keep[7, 3], keep[120] = False, False
    assert torch.equal(out[keep], want[keep]) and bool((~out[~keep].isfinite()).any(-1).all())


def test_keys_past_two_gigabytes():
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("needs 8 GB")
    S = 2000000
    far, near, q = torch.empty(S, 576, dtype=torch.bfloat16, device="cuda"), rows(300, seed=5), rows(20, 16, seed=6)
    far[:10], far[-290:] = near[:10], near[10:]
    far[10:-290] = float("nan")
    out = ops.window_mla_prefill(q, far, None, None, 250, 10, SCALE)
    ops.check_status("cuda")
    check(out, D.attend(q, near, D.prompt_sees(20, 300, 250, 10), SCALE))


def test_other_strides_streams_and_a_graph():
    q, kv = rows(30, 16, seed=1), rows(100, seed=2)
    want = ops.window_mla_prefill(q, kv, None, None, 40, 2, SCALE)
    wide, far = torch.zeros(30, 16, 640, dtype=torch.bfloat16, device="cuda"), torch.zeros(576, 100, dtype=torch.bfloat16, device="cuda")
    wide[:, :, 8:584] = q
    far.copy_(kv.t())
    assert torch.equal(ops.window_mla_prefill(wide[:, :, 8:584], far.t(), None, None, 40, 2, SCALE), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.window_mla_prefill(q, kv, None, None, 40, 2, SCALE)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    graph, out = torch.cuda.CUDAGraph(), torch.zeros_like(want)
    with torch.cuda.graph(graph):
        ops.window_mla_prefill(q, kv, None, None, 40, 2, SCALE, out=out)
    q2 = rows(30, 16, seed=77)
    want2 = ops.window_mla_prefill(q2, kv, None, None, 40, 2, SCALE)
    for x, w in ((q, want), (q2, want2)):
        q.copy_(x.clone())
        graph.replay()
        assert torch.equal(out, w)
    ops.check_status("cuda")


def test_prompt_tensors_of_other_forms_are_refused():
    q, kv = rows(4, 16), rows(9)
    args = dict(q=q, kv=kv, ks=None, ke=None, window=4, first=0, scale=SCALE)
    for bad in (dict(q=q.half()), dict(kv=kv.float()), dict(q=q[:, :, :512]), dict(kv=kv[:, :512]), dict(kv=kv.cpu()), dict(ke=torch.ones(4, device="cuda")), dict(ks=i32([0, 0])),
                dict(window=0), dict(first=-1), dict(kv=kv[:3]), dict(out=torch.empty(4, 16, 512, device="cuda")), dict(scale=0.0),
                dict(out=torch.empty(4, 16, 1024, dtype=torch.bfloat16, device="cuda")[:, :, ::2]), dict(workspace=torch.empty(64, 2, dtype=torch.uint8, device="cuda")[:, 0])):
        with pytest.raises(ops.DsaError):
            ops.window_mla_prefill(**{**args, **bad})
    assert ops.window_mla_prefill(q[:0], kv, None, None, 4, 0, SCALE).shape == (0, 16, 512)
    assert bool((ops.window_mla_prefill(q, kv[:0], None, i32([0, 0, 1, 5]), 4, 0, SCALE) == 0).all())


# ---- decode ---------------------------------------------------------------------------------------------------------
class Case:
    """Sequences in pages of random order; records that no sequence has read as NaN."""

    def __init__(self, B, per, H, ctx, record, seed, n_new=None, tree=False, gain=1.0, spare=3):
        rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
        self.B, self.per, self.ctx = B, per, ctx
        self.max_ctx = -(-max(max(ctx), 1) // 64) * 64
        P = self.max_ctx // 64
        pool = B * P + spare
        kv = torch.randn(pool * 64, 576, generator=g).to(torch.bfloat16).cuda()
        self.table = torch.randperm(pool, generator=g)[:B * P].int().view(B, P)
        self.rec = layer.pack_latent_cache(kv) if record == 656 else ops.pack_latent4(kv)
        values = D.record_values(self.rec)
        used = torch.zeros(pool * 64, dtype=torch.bool)
        at = self.table.long()[:, torch.arange(self.max_ctx) // 64] * 64 + torch.arange(self.max_ctx) % 64
        for b in range(B):
            used[at[b, :max(ctx[b], 0)]] = True
        self.rec[~used.cuda()] = 255
        self.kv = values[at].cuda()                        # [B, max_ctx, 576]
        self.q = (torch.randn(B * per, H, 576, generator=g) * gain).to(torch.bfloat16).cuda()
        self.n_new = n_new
        self.tree = D.random_tree(rng, B, per) if tree else None

    def args(self):
        return dict(q=self.q, cache=self.rec, block_table=self.table.cuda(), ctx_len=i32(self.ctx), tokens_per_seq=self.per, n_new=None if self.n_new is None else i32(self.n_new),
                    tree=None if self.tree is None else self.tree.cuda())

    def sees(self, window, first):
        return D.draft_sees(self.B, self.per, self.ctx, self.max_ctx, self.n_new, self.tree, window, first)

    def want(self, window, first):
        return D.attend(self.q, self.kv.repeat_interleave(self.per, 0), self.sees(window, first), SCALE)


@pytest.mark.parametrize("record", [656, 416])
@pytest.mark.parametrize("B,per,H,ctx,window,first", [
    (1, 1, 128, [1], 64, 4), (1, 1, 128, [64], 64, 0), (1, 1, 128, [2000], 512, 4), (3, 1, 128, [700, 0, 65], 100, 70), (2, 1, 16, [900, 333], 1 << 30, 0), (5, 1, 8, [200, 1, 2, 64, 129], 33, 1),
    (2, 3, 128, [500, 2], 128, 4), (2, 4, 16, [900, 700], 300, 64), (3, 7, 16, [128, 7, 66], 64, 0), (1, 100, 2, [333], 20, 3), (2, 5, 64, [321, 64], 2, 1), (1, 2, 200, [300], 90, 0),
    (80, 1, 128, [130] * 80, 100, 4), (40, 4, 48, [190] * 40, 64, 2), (1, 24, 128, [4000], 2048, 64),
])
def test_chains(record, B, per, H, ctx, window, first):
    c = Case(B, per, H, ctx, record, seed=B + per + H)
    out = torch.full((B * per, H, 512), 9.0, dtype=torch.bfloat16, device="cuda")
    for room in (0, None):
        ops.window_mla_decode_paged(**c.args(), window=window, first=first, scale=SCALE, out=out, workspace=None if room is None else torch.empty(0, dtype=torch.uint8, device="cuda"))
        ops.check_status("cuda")
        check(out, c.want(window, first))


@pytest.mark.parametrize("record", [656, 416])
@pytest.mark.parametrize("H", [128, 16, 40])
@pytest.mark.parametrize("per,window,first", [(4, 100, 4), (13, 5, 2), (64, 30, 0), (2, 1, 0), (9, 3, 80), (24, 700, 64)])
def test_trees(record, H, per, window, first):
    """Trees in sequences that are longer than the window, shorter, and made of drafts alone; rows without a token, an idle sequence."""
    ctx = [600, 70, per, 0, 130]
    c = Case(5, per, H, ctx, record, seed=per + H, n_new=[per, max(1, per // 2), per, 0, 1], tree=True)
    out = ops.window_mla_decode_paged(**c.args(), window=window, first=first, scale=SCALE)
    ops.check_status("cuda")
    check(out, c.want(window, first))
    assert bool((out.view(5, per, -1)[3] == 0).all()) and bool((out.view(5, per, -1)[4, 1:] == 0).all())


@pytest.mark.parametrize("record", [656, 416])
@pytest.mark.parametrize("H,per,window,first", [(128, 13, 100, 0), (128, 5, 70, 40), (64, 9, 1, 0), (200, 4, 300, 3), (16, 64, 33, 0), (5, 100, 40, 2), (2, 300, 64, 1), (40, 30, 1 << 30, 0)])
@pytest.mark.parametrize("tree", [False, True])
def test_many_rows_a_sequence(record, H, per, window, first, tree):
    """Sequences of several units, with room for their records as rows and without; lengths of drafts alone, pages that are none."""
    if tree and per > 64:
        pytest.skip("a tree has at most 64 drafts")
    ctx, n_new = [700, per, 0, 333], [per, per, 0, max(1, per - 2)]
    ctx[3] = max(333, per)
    c = Case(4, per, H, ctx, record, seed=per + H, n_new=n_new, tree=tree)
    want = c.want(window, first)
    args = c.args()
    none = torch.empty(0, dtype=torch.uint8, device="cuda")
    for ws in (None, none):
        check(ops.window_mla_decode_paged(**args, window=window, first=first, scale=SCALE, workspace=ws), want)
    ops.check_status("cuda")
    hole = int((ctx[0] - per) // 64)                                      # the page of the first draft, and of tokens before
    args["block_table"][0, hole] = -1
    sees = c.sees(window, first)
    sees[:per, hole * 64:hole * 64 + 64] = False
    want = D.attend(c.q, c.kv.repeat_interleave(per, 0), sees, SCALE)
    for ws in (None, none):
        check(ops.window_mla_decode_paged(**args, window=window, first=first, scale=SCALE, workspace=ws), want)
        with pytest.raises(ops.DsaError, match="out of range"):
            ops.check_status("cuda")


@pytest.mark.parametrize("record", [656, 416])
def test_many_rows_a_sequence_and_records_that_are_no_numbers(record):
    c = Case(2, 11, 64, [400, 90], record, seed=7, tree=True)
    sees, clean = c.sees(100, 2), c.want(100, 2)
    for b, pos in ((0, 389), (0, 395), (0, 399), (1, 1), (1, 85)):
        dirty = c.args()
        dirty["cache"] = c.rec.clone()
        dirty["cache"][int(c.table[b, pos // 64]) * 64 + pos % 64] = 255
        out = ops.window_mla_decode_paged(**dirty, window=100, first=2, scale=SCALE)
        ops.check_status("cuda")
        touched = torch.zeros(22, dtype=torch.bool)
        touched[b * 11:(b + 1) * 11] = sees[b * 11:(b + 1) * 11, pos]
        assert bool(out[touched.cuda()].isnan().flatten(1).any(1).all())
        check(out[~touched.cuda()], clean[~touched.cuda()])


def test_masks_are_held_to_the_drafts_before():
    c = Case(2, 6, 16, [90, 64], 416, seed=4, n_new=[6, 4], tree=True)
    a = ops.window_mla_decode_paged(**c.args(), window=40, first=2, scale=SCALE)
    c.tree = c.tree | torch.tensor([-1 << i for i in range(6)])           # its own bit and all behind
    assert torch.equal(a, ops.window_mla_decode_paged(**c.args(), window=40, first=2, scale=SCALE))
    c.tree = torch.full_like(c.tree, 0)                                   # each draft alone behind the cached tokens
    check(ops.window_mla_decode_paged(**c.args(), window=40, first=2, scale=SCALE), c.want(40, 2))
    ops.check_status("cuda")


@pytest.mark.parametrize("record", [656, 416])
@pytest.mark.parametrize("H,per,tree", [(128, 1, False), (16, 4, False), (16, 6, True), (128, 6, True)])
def test_records_that_are_no_numbers(record, H, per, tree):
    """A record of NaN: the rows that see it are none, those that do not are right, drafts of other branches among them."""
    c = Case(3, per, H, [300, 150, 80], record, seed=H + per, tree=tree)
    sees, clean = c.sees(100, 2), c.want(100, 2)
    for b, pos in ((0, 299), (0, 300 - per), (1, 1), (1, 149 - per // 2), (0, 199), (2, 79), (0, 150)):
        dirty = c.args()
        dirty["cache"] = c.rec.clone()
        dirty["cache"][int(c.table[b, pos // 64]) * 64 + pos % 64] = 255
        out = ops.window_mla_decode_paged(**dirty, window=100, first=2, scale=SCALE)
        ops.check_status("cuda")
        touched = torch.zeros(3 * per, dtype=torch.bool)
        touched[b * per:(b + 1) * per] = sees[b * per:(b + 1) * per, pos]
        assert bool(out[touched.cuda()].isnan().flatten(1).any(1).all())
        check(out[~touched.cuda()], clean[~touched.cuda()])


@pytest.mark.parametrize("record", [656, 416])
@pytest.mark.parametrize("H", [128, 16])
def test_records_that_are_no_numbers_in_parts(record, H):
    c = Case(2, 5, H, [1500, 900], record, seed=H, tree=True)
    sees, clean = c.sees(1 << 20, 0), c.want(1 << 20, 0)
    for b, pos in ((0, 1496), (0, 1498), (1, 896), (1, 300)):
        dirty = c.args()
        dirty["cache"] = c.rec.clone()
        dirty["cache"][int(c.table[b, pos // 64]) * 64 + pos % 64] = 255
        out = ops.window_mla_decode_paged(**dirty, window=1 << 20, first=0, scale=SCALE)
        ops.check_status("cuda")
        touched = torch.zeros(10, dtype=torch.bool)
        touched[b * 5:(b + 1) * 5] = sees[b * 5:(b + 1) * 5, pos]
        assert bool(out[touched.cuda()].isnan().flatten(1).any(1).all())
        check(out[~touched.cuda()], clean[~touched.cuda()])


@pytest.mark.parametrize("record", [656, 416])
@pytest.mark.parametrize("B", [1, 3, 5, 9, 30])
@pytest.mark.parametrize("H", [64, 128, 200])
def test_units_of_fewer_rows_and_parts(record, B, H):
    """Small calls: units of 32, 64 and 128 rows, up to sixteen parts, room for some of them."""
    c = Case(B, 1, H, ([1100, 1, 700, 0, 64, 1100, 129, 1000, 500] * 4)[:B], record, seed=B + H)
    want = c.want(1000, 70)
    for room in (0, 3000000, None):
        ws = None if room is None else torch.empty(room, dtype=torch.uint8, device="cuda")
        check(ops.window_mla_decode_paged(**c.args(), window=1000, first=70, scale=SCALE, workspace=ws), want)
    ops.check_status("cuda")


def test_bad_lengths_and_pages_are_flagged_and_skipped():
    c = Case(6, 4, 16, [100, 100, 100, 100, 100, 100], 416, seed=2, n_new=[4, 5, -1, 4, 3, 4])
    args = c.args()
    args["ctx_len"] = i32([100, 100, 100, 3, 129, 100])
    args["block_table"][5, 0] = 10000
    args["block_table"][0, 1] = -5
    out = ops.window_mla_decode_paged(**args, window=1 << 20, first=0, scale=SCALE, max_ctx=128)
    with pytest.raises(ops.DsaError, match="out of range"):
        ops.check_status("cuda")
    assert bool((out.view(6, 4, -1)[1:5] == 0).all())
    c.n_new = [4, 0, 0, 0, 0, 4]
    sees = c.sees(1 << 20, 0)
    sees[:4, 64:], sees[20:, :64] = False, False                          # pages that are none are not seen
    check(out, D.attend(c.q, c.kv.repeat_interleave(4, 0), sees, SCALE))


def test_decode_tensors_of_other_forms_are_refused():
    c = Case(2, 3, 16, [100, 90], 416, seed=1, n_new=[3, 2], tree=True)
    args = dict(c.args(), window=10, first=1, scale=SCALE)
    for bad in (dict(q=c.q.float()), dict(q=c.q[:5]), dict(q=c.q[:, :, :512].contiguous()), dict(cache=c.rec[:, :400]), dict(cache=c.rec[:63]), dict(cache=c.rec.int()), dict(ctx_len=i32([1])),
                dict(ctx_len=i32([9, 9]).long()), dict(n_new=i32([1, 1, 1])), dict(tree=args["tree"].int()), dict(tree=args["tree"][:, :2]), dict(tokens_per_seq=0), dict(tokens_per_seq=4),
                dict(block_table=args["block_table"].long()), dict(block_table=args["block_table"][:1]), dict(max_ctx=129), dict(window=0), dict(first=-1), dict(q=c.q.cpu()),
                dict(out=torch.empty(6, 16, 512, device="cuda"))):
        with pytest.raises(ops.DsaError):
            ops.window_mla_decode_paged(**{**args, **bad})
    big = torch.zeros(65, 1, 576, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ops.DsaError, match="64"):
        ops.window_mla_decode_paged(big, c.rec, args["block_table"][:1], i32([100]), 4, 0, SCALE, 65, tree=torch.zeros(1, 65, dtype=torch.int64, device="cuda"))
    assert ops.window_mla_decode_paged(**dict(args, q=c.q[:0], block_table=args["block_table"][:0], ctx_len=i32([]), n_new=i32([]), tree=args["tree"][:0])).shape == (0, 16, 512)


def test_the_module_takes_prompts_and_caches():
    m = layer.WindowMLA(SCALE, 40, 2)
    q, kv = rows(9, 16), rows(30)
    assert torch.equal(m(q, kv), ops.window_mla_prefill(q, kv, None, None, 40, 2, SCALE))
    c = Case(2, 3, 16, [100, 90], 656, seed=1, n_new=[3, 2], tree=True)
    a = c.args()
    assert torch.equal(m(a["q"], a["cache"], block_table=a["block_table"], ctx_len=a["ctx_len"], tokens_per_seq=3, n_new=a["n_new"], tree=a["tree"]),
                       ops.window_mla_decode_paged(**a, window=40, first=2, scale=SCALE))


def test_cache_rows_past_two_gigabytes():
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("needs 8 GB")
    c = Case(2, 2, 16, [128, 100], 416, seed=3)
    pages = 84000
    far = torch.empty(pages * 64, 416, dtype=torch.uint8, device="cuda")
    a = c.args()
    want = ops.window_mla_decode_paged(**a, window=90, first=2, scale=SCALE)
    for i in range(2):
        for j in range(2):
            far[(pages - 1 - 2 * i - j) * 64:(pages - 2 * i - j) * 64] = c.rec[int(c.table[i, j]) * 64:int(c.table[i, j]) * 64 + 64]
    a.update(cache=far, block_table=i32([[pages - 1, pages - 2], [pages - 3, pages - 4]]))
    assert torch.equal(ops.window_mla_decode_paged(**a, window=90, first=2, scale=SCALE), want)
    ops.check_status("cuda")


def test_decode_in_two_graphs_and_on_two_streams():
    c, d = Case(2, 3, 16, [700, 90], 416, seed=1, tree=True), Case(2, 3, 16, [500, 640], 416, seed=2, tree=True)
    want = [ops.window_mla_decode_paged(**x.args(), window=400, first=2, scale=SCALE) for x in (c, d)]
    graphs, outs, args = [], [], [c.args(), d.args()]
    for a in args:
        g, out = torch.cuda.CUDAGraph(), torch.zeros(6, 16, 512, dtype=torch.bfloat16, device="cuda")
        with torch.cuda.graph(g):
            ops.window_mla_decode_paged(**a, window=400, first=2, scale=SCALE, out=out)
        graphs.append(g)
        outs.append(out)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    args[0]["ctx_len"].copy_(i32([300, 88]))
    graphs[0].replay()
    assert torch.equal(outs[0], ops.window_mla_decode_paged(**args[0], window=400, first=2, scale=SCALE))
    ops.check_status("cuda")
