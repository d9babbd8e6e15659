"""Drafts over tables with pages that are none: what stands there is in no draft's list, and in no draft's output."""
import pytest
import torch

from llmdivedeep_b200 import layer, ops
from oracle import drafts_oracle as D
from tests.test_gpu_drafts import SCALE, Case, i32
from tests.test_gpu_window import check

pytestmark = pytest.mark.gpu


def holes(c, at):
    """Takes pages `at` [(sequence, page)] out of the table; what its drafts see is left without them."""
    sees = c.sees().cpu()
    for (b, page), none in zip(at, [-1, 1 << 20, -(1 << 31), c.k8.shape[0] // 64] * len(at)):
        c.table[b, page] = none
        sees[b * c.per:(b + 1) * c.per, page * 64:page * 64 + 64] = False
    return sees


def flagged():
    with pytest.raises(ops.DsaError, match="out of range"):
        ops.check_status("cuda")


@pytest.mark.parametrize("k", [4, 100, 630, 2048])
@pytest.mark.parametrize("per,tree", [(1, True), (5, True), (5, False), (13, True), (70, False)])
def test_selection(per, tree, k):
    """The page that the drafts are in, the first one, one in the middle, all of a sequence's; lists longer and shorter than what is left."""
    c = Case(4, per, 64, [700, 333, 130, 500], seed=per + k, n_new=[per, max(1, per - 1), per, 0], tree=tree)
    sees = holes(c, [(0, 0), (0, 4), (1, (333 - per) // 64), (2, 0), (2, 1), (2, 2)])
    logits = c.logits()
    flagged()
    idx = ops.topk_select_drafts(logits, k, **c.lens()).cpu()
    ops.check_status("cuda")
    for r in range(4 * per):
        got = sorted(x for x in idx[r].tolist() if x >= 0)
        at = torch.nonzero(sees[r])[:, 0]
        best = at[torch.sort(logits[r].cpu()[at], descending=True, stable=True)[1][:k]]
        assert got == sorted(best.tolist()), r


@pytest.mark.parametrize("record", [656, 416])
@pytest.mark.parametrize("tree", [True, False])
def test_a_step(record, tree):
    """k above what is left: the step's output is attention over all of it."""
    per, H, ctx = 5, 128, [300, 90, 64]
    c = Case(3, per, 64, ctx, seed=3, tree=tree)
    g = torch.Generator().manual_seed(9)
    kv = torch.randn(c.k8.shape[0], 576, generator=g).to(torch.bfloat16).cuda()
    rec = layer.pack_latent_cache(kv) if record == 656 else ops.pack_latent4(kv)
    q = torch.randn(3 * per, H, 576, generator=g).to(torch.bfloat16).cuda()
    at = torch.arange(c.max_ctx)
    values = D.record_values(rec).cuda()[(c.table[:, (at // 64).cuda()].long() * 64 + (at % 64).cuda())]
    sees = holes(c, [(0, 2), (1, 1), (2, 0)])
    ws = layer.DecodeWorkspace(3 * per, H, c.max_ctx, 512, "cuda")
    lens = c.lens()
    idx, out = layer.dsa_draft_step(c.q8, c.w, c.k8, c.ksc, c.table, lens["ctx_len"], q, rec, SCALE, ws, per, lens["n_new"], lens["tree"])
    flagged()
    for r in range(3 * per):
        assert sorted(x for x in idx[r].tolist() if x >= 0) == torch.nonzero(sees[r])[:, 0].tolist()
    check(out, D.attend(q, values.repeat_interleave(per, 0), sees, SCALE))
    want = ops.window_mla_decode_paged(q, rec, c.table, i32(ctx), 1 << 20, 0, SCALE, per, lens["n_new"], lens["tree"])
    flagged()
    check(want, D.attend(q, values.repeat_interleave(per, 0), sees, SCALE))
