"""Drafted tokens on the GPU: the indexer over a tree, the selection, one step against a step for each draft, the acceptance of a path, and a
speculative round over a paged cache."""
import random

import numpy as np
import pytest
import torch

from llmdivedeep_b200 import layer, ops
from oracle import drafts_oracle as D
from tests.test_gpu_pages import Both, ints
from tests.test_gpu_window import check as check_attention

pytestmark = pytest.mark.gpu
SCALE = 192 ** -0.5


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32).cuda()


def quantised(x):
    return ops.fp8_quant_per_block(x, 128)


class Case:
    def __init__(self, B, per, H, ctx, seed, n_new=None, tree=False, w_dtype=torch.float32):
        g = torch.Generator().manual_seed(seed)
        self.B, self.per, self.H, self.ctx, self.n_new = B, per, H, ctx, n_new
        self.max_ctx = max(max(ctx), 1)
        P = -(-self.max_ctx // 64)
        pool = B * P + 2
        self.k8, self.ksc = quantised(torch.randn(pool * 64, 128, generator=g).cuda())
        self.q8, qs = quantised(torch.randn(B * per, H, 128, generator=g).cuda())
        self.w = (torch.randn(B * per, H, generator=g).cuda() * qs * (128 * H) ** -0.5).to(w_dtype)
        self.table = torch.randperm(pool, generator=g)[:B * P].int().view(B, P).cuda()
        self.tree = D.random_tree(random.Random(seed), B, per) if tree else None

    def lens(self):
        return dict(ctx_len=i32(self.ctx), tokens_per_seq=self.per, n_new=None if self.n_new is None else i32(self.n_new), tree=None if self.tree is None else self.tree.cuda())

    def logits(self, **more):
        return ops.fp8_paged_mqa_logits(self.q8, self.w, self.k8, self.ksc, self.table, max_ctx=self.max_ctx, **{**self.lens(), **more})

    def sees(self):
        return D.draft_sees(self.B, self.per, self.ctx, self.max_ctx, self.n_new, self.tree).cuda()

    def want(self):
        at = torch.arange(self.max_ctx, device="cuda")
        rows = (self.table[:, at // 64].long() * 64 + at % 64).repeat_interleave(self.per, 0)
        sees = self.sees()
        return torch.cat([D.logits(self.q8[t:t + 1], self.w[t:t + 1], self.k8.view(torch.uint8)[rows[t:t + 1]].view(ops.FP8), self.ksc[rows[t:t + 1]], sees[t:t + 1])
                          for t in range(self.B * self.per)])


def check_logits(got, want, ctx, per):
    """Exact products, sums of 128 and of 64 terms in fp32: each of the 64 + 128 additions rounds by 2^-24 of a partial sum, which is at most the sum of the terms'
    magnitudes, and so at most eight times the spread of the scores here (64 terms of either sign)."""
    for r in range(want.shape[0]):
        c = ctx[r // per]
        end = min(want.shape[1], -(-c // 128) * 128)
        g, w = got[r, :end].double(), want[r, :end]
        assert torch.equal(torch.isinf(g), torch.isinf(w)) and bool((g[torch.isinf(g)] < 0).all())
        fine = torch.isfinite(w)
        if fine.any():
            assert float((g - w)[fine].abs().max()) <= 192 * 2.0 ** -24 * 8 * float(w[fine].abs().max())


@pytest.mark.parametrize("H", [64, 32, 16])
@pytest.mark.parametrize("B,per,ctx,tree", [
    (1, 2, [2], False), (1, 4, [130], True), (2, 3, [700, 64], True), (1, 6, [2000], True), (3, 5, [128, 0, 129], False), (2, 8, [515, 1000], True), (1, 13, [900], True),
    (2, 1, [300, 5], True), (1, 64, [257], True), (1, 70, [200], False), (40, 4, [300] * 40, True),
])
def test_logits(H, B, per, ctx, tree):
    c = Case(B, per, H, ctx, seed=B + per + H, tree=tree)
    out = torch.full((B * per + 1, c.max_ctx + 9), 7.0, device="cuda")
    got = c.logits(out=out)
    ops.check_status("cuda")
    check_logits(got, c.want(), ctx, per)
    assert bool((out[B * per:] == 7).all()) and bool((out[:, c.max_ctx:] == 7).all())
    for r in range(B * per):                              # untouched behind the tile that the sequence ends in
        assert bool((out[r, -(-ctx[r // per] // 128) * 128:] == 7).all())
    assert torch.equal(c.logits()[:, 0].nan_to_num(), got[:, 0].nan_to_num()) or 0 in ctx


@pytest.mark.parametrize("per", [2, 3, 5, 9])
@pytest.mark.parametrize("w_dtype", [torch.float32, torch.bfloat16])
def test_logits_of_ragged_drafts(per, w_dtype):
    n_new = [per, 1, max(1, per - 1), 0]
    c = Case(4, per, 64, [500, 1, 64, 90], seed=per, n_new=n_new, tree=True, w_dtype=w_dtype)
    got = c.logits()
    ops.check_status("cuda")
    check_logits(got, c.want(), c.ctx, per)


@pytest.mark.parametrize("H", [64, 32, 16])
@pytest.mark.parametrize("per", [1, 2, 3, 5, 8])
def test_logits_of_a_draft_are_those_of_a_decode_step(H, per):
    """Bit for bit: drafts that are checked together and tokens that are made one by one select the same keys."""
    c = Case(3, per, H, [500, 33, 640], seed=per)
    got = c.logits(n_new=i32([per] * 3))
    for i in range(per):
        ctx = [x - per + i + 1 for x in c.ctx]
        one = ops.fp8_paged_mqa_logits(c.q8[i::per], c.w[i::per], c.k8, c.ksc, c.table, i32(ctx), c.max_ctx)
        for b in range(3):
            assert torch.equal(got[b * per + i, :ctx[b]], one[b, :ctx[b]])


def test_logits_bad_lengths_and_pages():
    c = Case(5, 3, 64, [200] * 5, seed=4, n_new=[3, 4, -1, 3, 3])
    ctx = i32([200, 200, 200, 2, 201])
    c.table[0, 1] = 1 << 20
    got = c.logits(ctx_len=ctx, out=torch.full((15, 200), 7.0, device="cuda"))
    with pytest.raises(ops.DsaError, match="out of range"):
        ops.check_status("cuda")
    assert bool((got[3:] == 7).all()) and bool(torch.isneginf(got[:3, 64:128]).all()) and bool(got[:3, :64].isfinite().all())


def test_forms_that_are_refused():
    c = Case(2, 3, 64, [200, 100], seed=4, tree=True)
    for bad in (dict(tree=c.tree.int().cuda()), dict(tree=c.tree[:1].cuda()), dict(n_new=i32([1])), dict(ctx_len=i32([1, 2, 3])), dict(tokens_per_seq=4), dict(tokens_per_seq=0),
                dict(max_ctx=257), dict(out=torch.empty(6, 100, device="cuda")), dict(out=torch.empty(6, 200, dtype=torch.bfloat16, device="cuda")), dict(tree=c.tree)):
        with pytest.raises(ops.DsaError):
            ops.fp8_paged_mqa_logits(c.q8, c.w, c.k8, c.ksc, c.table, **{**dict(max_ctx=200), **c.lens(), **bad})
    with pytest.raises(ops.DsaError):
        ops.fp8_paged_mqa_logits(c.q8[:, :8].contiguous(), c.w[:, :8], c.k8, c.ksc, c.table, max_ctx=200, **c.lens())
    logits = torch.zeros(6, 200, device="cuda")
    lens = c.lens()
    for bad in (dict(logits=logits.double()), dict(logits=logits[:5]), dict(logits=logits.t()), dict(out=torch.empty(6, 5, dtype=torch.int32, device="cuda")), dict(ctx_len=i32([1])),
                dict(logits=logits[:1].expand(6, 200))):
        with pytest.raises(ops.DsaError):
            ops.topk_select_drafts(**{**dict(logits=logits, k=4, **lens), **bad})


# ---- selection ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("k", [1, 16, 100, 600])
@pytest.mark.parametrize("tree", [True, False])
def test_selection(k, tree):
    """Sets of the k largest seen positions; rows that see fewer have all of them and nothing else."""
    per, ctx, n_new = 7, [700, 90, 7, 0, 130], [7, 7, 5, 0, 1]
    c = Case(5, per, 64, ctx, seed=k, n_new=n_new, tree=tree)
    logits = c.logits()
    lens = c.lens()
    idx = ops.topk_select_drafts(logits, k, **lens).cpu()
    sees = c.sees().cpu()
    for r in range(5 * per):
        got = sorted(x for x in idx[r].tolist() if x >= 0)
        at = torch.nonzero(sees[r])[:, 0]
        best = at[torch.sort(logits[r].cpu()[at], descending=True, stable=True)[1][:k]]
        assert got == sorted(best.tolist()) and len(set(got)) == len(got)
    assert ops.topk_select_drafts(logits, 0, **lens).shape == (35, 0)


@pytest.mark.parametrize("k", [4, 150])
def test_scores_that_are_no_numbers_select_nothing_unseen(k):
    """Most scores of a row -inf or NaN of either sign: what its draft does not see is not in its list all the same."""
    per, ctx = 5, 200
    c = Case(3, per, 64, [ctx] * 3, seed=k, tree=True)
    c.tree = torch.tensor([1, 0, 1, 4, 8], dtype=torch.int64).expand(3, per).contiguous()
    logits = c.logits()
    logits[:per, 2:ctx - per] = -float("inf")
    logits[per:2 * per, 2:ctx - per] = float("nan")
    logits[2 * per:, 2:ctx - per] = -torch.full((), float("nan"), device="cuda")
    idx = ops.topk_select_drafts(logits, k, **c.lens()).cpu()
    sees = c.sees().cpu()
    for r in range(3 * per):
        got = [x for x in idx[r].tolist() if x >= 0]
        assert all(bool(sees[r, x]) for x in got) and len(set(got)) == len(got)


def test_keys_that_are_no_numbers_where_a_draft_does_not_see():
    """Another draft's key, and what lies behind the sequence in its last page: values, and a scale, that are none."""
    per, ctx = 4, [300, 70]
    c = Case(2, per, 64, ctx, seed=5, tree=True)
    c.tree = torch.tensor([[1, 0, 1, 2]] * 2, dtype=torch.int64)
    clean = c.logits()
    k8, ksc = c.k8.view(torch.uint8).clone(), c.ksc.clone().view(-1)
    for b in range(2):
        row = lambda s: int(c.table[b, s // 64]) * 64 + s % 64
        k8[row(ctx[b] - per)] = 0x7f                      # draft 0, which 2 descends from and 1 and 3 do not
        ksc[row(ctx[b] - per + 2)] = float("inf")         # draft 2, which nobody else sees
        for s in range(ctx[b], -(-ctx[b] // 64) * 64):
            k8[row(s)], ksc[row(s)] = 0xff, float("nan")
    c.k8, c.ksc = k8.view(ops.FP8), ksc.view_as(c.ksc)
    got = c.logits()
    for r in (1, 3, 5, 7):
        end = min(c.max_ctx, -(-ctx[r // per] // 128) * 128)
        assert torch.equal(got[r, :end], clean[r, :end])
    for r in (0, 2, 4, 6):
        P = ctx[r // per] - per
        assert torch.equal(got[r, :P], clean[r, :P])


def test_logits_in_two_graphs_and_on_two_streams():
    """One set of inputs, outputs of their own: replays in either order, and two calls at once, give what a call gave."""
    a, b = Case(3, 4, 64, [700, 90, 333], seed=1, tree=True), Case(2, 2, 32, [1200, 64], seed=2)
    want = [x.logits().clone() for x in (a, b)]
    idx = [ops.topk_select_drafts(w, 64, **x.lens()).clone() for w, x in zip(want, (a, b))]
    lens = [x.lens() for x in (a, b)]
    outs, sel, graphs = [], [], []
    for x, ln in zip((a, b), lens):
        o, s, gr = torch.empty(x.B * x.per, x.max_ctx, device="cuda"), torch.empty(x.B * x.per, 64, dtype=torch.int32, device="cuda"), torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(gr, stream=side):
            ops.fp8_paged_mqa_logits(x.q8, x.w, x.k8, x.ksc, x.table, max_ctx=x.max_ctx, out=o, **ln)
            ops.topk_select_drafts(o, 64, out=s, **ln)
        outs.append(o), sel.append(s), graphs.append(gr)
    pick = lambda x, o: torch.cat([o[r, :-(-x.ctx[r // x.per] // 128) * 128] for r in range(x.B * x.per)])
    seen = [pick(x, w) for x, w in zip((a, b), want)]
    for order in ((0, 1), (1, 0), (0, 0, 1, 1)):
        for o, s in zip(outs, sel):
            o.fill_(3.0), s.fill_(-7)
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        for x, o, s, w, k in zip((a, b), outs, sel, seen, idx):
            assert torch.equal(pick(x, o), w) and torch.equal(s.sort(1)[0], k.sort(1)[0])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(4):
        for i, (x, ln, st) in enumerate(zip((a, b), lens, streams)):
            with torch.cuda.stream(st):
                got[i] = ops.fp8_paged_mqa_logits(x.q8, x.w, x.k8, x.ksc, x.table, max_ctx=x.max_ctx, **ln)
    torch.cuda.synchronize()
    for x, o, w in zip((a, b), got, seen):
        assert torch.equal(pick(x, o), w)


def test_no_context_at_all():
    """Tables without a page: scores of no columns, lists of no positions."""
    q8, _ = quantised(torch.randn(6, 64, 128, device="cuda"))
    k8, ksc = quantised(torch.randn(64, 128, device="cuda"))
    table, lens = torch.empty(2, 0, dtype=torch.int32, device="cuda"), dict(ctx_len=i32([0, 0]), tokens_per_seq=3)
    logits = ops.fp8_paged_mqa_logits(q8, torch.ones(6, 64, device="cuda"), k8, ksc, table, max_ctx=0, **lens)
    assert logits.shape == (6, 0)
    idx = ops.topk_select_drafts(logits, 5, **lens)
    ops.check_status("cuda")
    assert bool((idx == -1).all()) and idx.shape == (6, 5)


@pytest.mark.parametrize("record", [656, 416])
@pytest.mark.parametrize("per,k", [(4, 64), (6, 512)])
def test_a_step_of_drafts_is_a_step_of_each(record, per, k):
    """Every draft's selection and output against a decode step of one token whose sequence is the draft's path."""
    ctx, n_new, H = [640, 100, 77], [per, per - 1, 1], 128
    c = Case(3, per, 64, ctx, seed=per + k, n_new=n_new, tree=True)
    g = torch.Generator().manual_seed(9)
    kv = torch.randn(c.k8.shape[0], 576, generator=g).to(torch.bfloat16).cuda()
    rec = layer.pack_latent_cache(kv) if record == 656 else ops.pack_latent4(kv)
    q = torch.randn(3 * per, H, 576, generator=g).to(torch.bfloat16).cuda()
    ws = layer.DecodeWorkspace(3 * per, H, c.max_ctx, k, "cuda")
    lens = c.lens()
    idx, out = layer.dsa_draft_step(c.q8, c.w, c.k8, c.ksc, c.table, lens["ctx_len"], q, rec, SCALE, ws, per, lens["n_new"], lens["tree"])
    idx, out = idx.clone(), out.clone()
    one = layer.DecodeWorkspace(1, H, c.max_ctx, k, "cuda")
    for b in range(3):
        for i in range(per):
            r = b * per + i
            path = D.draft_paths(ctx[b], n_new[b], i, c.tree[b], per)
            if path is None:
                assert bool((idx[r] == -1).all()) and bool((out[r] == 0).all())
                continue
            pages = -(-len(path) // 64)
            table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
            at = torch.tensor(path, device="cuda")
            rows = torch.zeros(pages * 64, dtype=torch.long, device="cuda")
            rows[:len(path)] = c.table[b][at // 64].long() * 64 + at % 64
            single = layer.dsa_decode_step(c.q8[r:r + 1], c.w[r:r + 1], c.k8.view(torch.uint8)[rows].view(ops.FP8), c.ksc[rows], torch.nn.functional.pad(table, (0, c.table.shape[1] - pages)),
                                           i32([len(path)]), q[r:r + 1], rec[rows], SCALE, one)
            want = at[single[0][0][single[0][0] >= 0].long()]
            assert sorted(idx[r][idx[r] >= 0].tolist()) == sorted(want.tolist())
            # both are off by their own roundings
            err = (out[r].double() - single[1][0].double()).norm() / single[1][0].double().norm()
            assert float(err) <= 2 * 7.5e-3
    ops.check_status("cuda")


# ---- acceptance -----------------------------------------------------------------------------------------------------
class Drafting(Both):
    def __init__(self, *a, **k):
        super().__init__(*a, **k)
        self.o.__class__ = D.Pool

    def accept(self, rows, n_new, path, n_keep, status=0):
        path = np.asarray(path, np.int32)
        path = path.reshape(len(rows), -1) if len(rows) else path
        ops.accept_drafts(self.table, self.ctx, self.refs, ints(rows), ints(n_new), ints(path), ints(n_keep), self.caches)
        self.o.accept(rows, n_new, path, n_keep)
        self.same(status)


@pytest.mark.parametrize("B,P,per,layers,widths", [(4, 3, 5, 2, (128, 4, 416)), (9, 5, 64, 1, (656,)), (30, 4, 13, 3, (132, 4, 416, 20)), (1, 1, 1, 1, (4,)), (3, 8, 200, 1, (128,))])
def test_paths_are_kept(B, P, per, layers, widths):
    rng = random.Random(B * per)
    p = Drafting(B, P, B * P + 1, layers, widths=widths)
    p.extend(range(B), [rng.randint(0, P * 64 - per) for _ in range(B)], P * 64)
    for _ in range(3):
        rows = rng.sample(range(B), rng.randint(1, B))
        n_new = [rng.randint(0, min(per, P * 64 - int(p.o.ctx[r]))) for r in rows]
        p.extend(rows, n_new, per)
        n_keep = [rng.randint(0, m) for m in n_new]
        p.accept(rows, n_new, [sorted(rng.sample(range(m), k)) + [-1] * (per - k) for m, k in zip(n_new, n_keep)], n_keep)
    p.accept([], [], np.zeros((0, 3)), [])


def test_edges_of_pages():
    p = Drafting(6, 4, 30)
    p.extend(range(6), [64, 60, 128, 63, 200, 1], 256)
    p.extend(range(6), [5, 9, 64, 2, 56, 63], 64)
    # nothing kept at a page's start, across a page's end, a page kept whole, the first page's last place, a full table, everything
    p.accept(range(6), [5, 9, 64, 2, 56, 63], [[0] * 64, [0, 2, 3, 5, 8] + [0] * 59, list(range(64)), [1] + [0] * 63, [55] + [0] * 63, list(range(63)) + [0]], [0, 5, 64, 1, 1, 63])


def test_rows_that_make_no_sense_stay_as_they_are():
    p = Drafting(8, 3, 30)
    p.extend(range(8), [10, 70, 100, 40, 50, 60, 64, 128], 192)
    p.accept([0, 1, 2, 3, 4, 5, 6, -1, 8, 0], [4, 71, 3, 5, 5, -1, 3, 1, 1, 2], [[0, 3], [0, 1], [1, 1], [3, 2], [0, 5], [0, 1], [0, 1], [0, 1], [0, 1], [0, 1]], [2, 2, 2, 2, 2, 0, 3, 1, 1, 1], status=2)
    p.table[2, 1], p.o.table[2, 1] = 99, 99
    p.accept([2], [40], [[5]], [1], status=2)
    p.table[7, 1], p.o.table[7, 1] = -1, -1
    p.accept([7], [3], [[0]], [1], status=2)


def test_pages_that_another_sequence_holds_are_not_written():
    p = Drafting(4, 4, 30)
    p.extend([0], [64 + 20], 128)
    p.extend([0], [44], 64)
    p.fork([0], [1])                                       # both pages are full, and shared
    p.accept([0], [44], [list(range(44))], [44])           # everything stays: nothing is written
    p.accept([0], [44], [[0, 2]], [2], status=2)
    p.accept([0], [64], [[]], [0])                         # the shared page goes as a whole
    p.accept([1], [64], [[3]], [1])                        # now it is the other's own
    p.extend([0, 1], [3, 3], 4)


@pytest.mark.parametrize("others", [0, 7])
def test_rows_are_judged_before_any_changes(others):
    """A row that drops a page and one that keeps drafts in it, in one call of few rows and of more: the second is refused, in either order."""
    for order in ((0, 1), (1, 0)):
        p = Drafting(2 + others, 4, 60)
        p.extend(range(2 + others), [128] + [0] + [20] * others, 128)
        p.fork([0], [1])                                   # both pages are full, and shared
        rows = list(order) + list(range(2, 2 + others))
        p.accept(rows, [64, 64] + [3] * others, [[0, 1] if r > 1 else [3, 0] for r in rows], [2 if r > 1 else 0 if r == 0 else 1 for r in rows], status=2)


def test_few_rows_that_make_no_sense_stay_as_they_are():
    p = Drafting(8, 3, 30, 2)
    p.extend(range(8), [10, 70, 100, 40, 50, 60, 64, 128], 192)
    p.accept([0, 1, 3, 4, 8, 0], [4, 71, 5, 5, 1, 2], [[0, 3], [0, 1], [3, 2], [0, 5], [0, 1], [0, 1]], [2, 2, 2, 2, 1, 1], status=2)
    p.accept([7], [100], [[99]], [1])


def test_accept_refused():
    p = Drafting(2, 2, 9)
    args = dict(block_table=p.table, ctx_len=p.ctx, refs=p.refs, rows=ints([0]), n_new=ints([1]), path=ints([[0]]), n_keep=ints([1]), caches=p.caches)
    for bad in (dict(path=ints([0])), dict(path=ints([[0]]).long()), dict(path=ints([[0], [1]])), dict(n_new=ints([1, 1])), dict(n_keep=ints([])), dict(rows=ints([[0]])),
                dict(path=ints([[0, 1, 2]])[:, ::2]), dict(refs=p.refs.long()), dict(caches=[p.caches[0][:, :64]]), dict(rows=ints([0]).cpu())):
        with pytest.raises(ops.DsaError):
            ops.accept_drafts(**{**args, **bad})


# ---- together -------------------------------------------------------------------------------------------------------
def test_speculative_rounds_over_a_paged_cache():
    """Drafts written, a sparse and a window layer over their tree, a path accepted: the cache holds what one token at a time would have written, and the outputs
    of the accepted path are those of its tokens alone."""
    rng, g = random.Random(3), torch.Generator().manual_seed(3)
    B, per, H, k, window, first = 3, 5, 16, 48, 40, 2
    cache, plain = (layer.PagedCache(2, 40, B, 320, "cuda") for _ in range(2))
    ws, one = layer.DecodeWorkspace(B * per, H, 320, k, "cuda"), layer.DecodeWorkspace(B, H, 320, k, "cuda")

    def tokens(*n):
        kv = torch.randn(*n, 576, generator=g).to(torch.bfloat16).cuda()
        k8, ksc = quantised(torch.randn(*n, 128, generator=g).cuda())
        return kv, k8, ksc

    lens = [130, 64, 7]
    prompt = [tokens(B, 130) for _ in range(2)]
    for c in (cache, plain):
        slots = c.extend([0, 1, 2], lens, 130)
        for l in range(2):
            c.write(l, slots, *prompt[l])
    for _ in range(4):
        m = [per, rng.randint(1, per), 2]
        tree = D.random_tree(rng, B, per)
        drafts = [tokens(B, per) for _ in range(2)]
        slots = cache.extend([0, 1, 2], m, per)
        for l in range(2):
            cache.write(l, slots, *drafts[l])
        q8, qs = quantised(torch.randn(B * per, 64, 128, generator=g).cuda())
        w = torch.randn(B * per, 64, generator=g).cuda() * qs / 90
        q = torch.randn(B * per, H, 576, generator=g).to(torch.bfloat16).cuda()
        n_new, t = i32(m), tree.cuda()
        idx, out = (x.clone() for x in cache.decode_drafts(0, q8, w, q, SCALE, ws, per, n_new, t))
        near = cache.window(1, q, window, first, SCALE, per, n_new, t)
        leaf = [rng.randint(0, x - 1) for x in m]
        path = [[j for j in range(i) if int(tree[b, i]) >> j & 1] + [i] for b, i in enumerate(leaf)]
        keep = [len(x) for x in path]
        before = cache.ctx.tolist()
        cache.accept([0, 1, 2], m, [x + [-1] * (per - len(x)) for x in path], keep)
        # the same path, token by token
        for s in range(max(keep)):
            some = [b for b in range(B) if s < keep[b]]
            slots = plain.extend(some, [1] * len(some), 1)
            pick = torch.tensor([path[b][s] for b in some])
            rows = torch.tensor([b * per for b in some]) + pick
            for l in range(2):
                plain.write(l, slots, *[x[some, pick] for x in drafts[l]])
            for b, r in zip(some, rows.tolist()):
                lone = torch.where(torch.arange(B, device="cuda") == b, plain.ctx, 0).int()
                pad = [torch.zeros_like(x[:1]).expand(B, *x.shape[1:]).clone() for x in (q8.view(torch.uint8), w, q)]
                for x, y in zip(pad, (q8.view(torch.uint8), w, q)):
                    x[b] = y[r]
                i1, o1 = layer.dsa_decode_step(pad[0].view(ops.FP8), pad[1], plain.k8[0], plain.k_scale[0], plain.table, lone, pad[2], plain.latent[0], SCALE, one)
                pos = torch.tensor([x if x < before[b] - m[b] else before[b] - m[b] + path[b][x - before[b] + m[b]] for x in i1[b][i1[b] >= 0].tolist()])
                assert sorted(pos.tolist()) == sorted(idx[r][idx[r] >= 0].tolist())
                check_attention(out[r:r + 1], o1[b:b + 1].double(), 2 * 7.5e-3, 2.0 ** -5)
                n1 = ops.window_mla_decode_paged(pad[2], plain.latent[1], plain.table, lone, window, first, SCALE)
                check_attention(near[r:r + 1], n1[b:b + 1].double(), 2 * 7.5e-3, 2.0 ** -5)
        assert cache.ctx.tolist() == plain.ctx.tolist()
        for b in range(B):
            n = int(plain.ctx[b])
            at = torch.arange(n, device="cuda")
            for x, y in zip(cache.caches, plain.caches):
                rx, ry = (c.table[b][at // 64].long() * 64 + at % 64 for c in (cache, plain))
                assert torch.equal(x.view(torch.uint8)[:, rx] if x.dtype == ops.FP8 else x[:, rx], y.view(torch.uint8)[:, ry] if y.dtype == ops.FP8 else y[:, ry])
        assert int((cache.refs > 0).sum()) == int(((cache.ctx + 63) // 64).sum())
    ops.check_status("cuda")


def test_a_round_in_a_graph():
    """Indexer, selection, attention and acceptance captured once and replayed with other lengths, trees and paths."""
    B, per, H = 2, 4, 16
    c = Case(B, per, 64, [200, 150], seed=5, n_new=[4, 3], tree=True)
    kv = torch.randn(c.k8.shape[0], 576, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    q = torch.randn(B * per, H, 576, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    rec = ops.pack_latent4(kv)
    refs = torch.zeros(c.k8.shape[0] // 64, dtype=torch.int32, device="cuda")
    refs[c.table.flatten().long()] = 1
    lens, rows = c.lens(), i32([0, 1])
    path, keep = i32([[0, 2, -1, -1], [1, -1, -1, -1]]), i32([2, 1])
    ws = layer.DecodeWorkspace(B * per, H, c.max_ctx, 64, "cuda")
    state = [t.clone() for t in (c.table, lens["ctx_len"], refs, rec)]

    def step():
        idx, out = layer.dsa_draft_step(c.q8, c.w, c.k8, c.ksc, c.table, lens["ctx_len"], q, rec, SCALE, ws, per, lens["n_new"], lens["tree"])
        ops.accept_drafts(c.table, lens["ctx_len"], refs, rows, lens["n_new"], path, keep, [rec])
        return idx, out

    def restore():
        for t, s in zip((c.table, lens["ctx_len"], refs, rec), state):
            t.copy_(s)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
        restore()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for n, tree, p, kp in (([4, 3], c.tree, [[0, 2, -1, -1], [1, -1, -1, -1]], [2, 1]), ([2, 4], c.tree.flip(0), [[1, -1, -1, -1], [0, 1, 2, 3]], [1, 4])):
        lens["n_new"].copy_(i32(n))
        lens["tree"].copy_(tree)
        path.copy_(i32(p))
        keep.copy_(i32(kp))
        restore()
        want = [t.clone() for t in step()] + [t.clone() for t in (c.table, lens["ctx_len"], refs, rec)]
        restore()
        ws.idx.zero_(), ws.out.zero_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip((ws.idx, ws.out, c.table, lens["ctx_len"], refs, rec), want))
    ops.check_status("cuda")
