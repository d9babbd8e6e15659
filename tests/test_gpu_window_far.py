"""Queries, outputs and scores of more than four gigabytes: offsets that pass 32 bits, in elements and in bytes."""
import math

import pytest
import torch

from llmdivedeep_b200 import layer, ops
from oracle import drafts_oracle as D
from tests.test_gpu_drafts import check_logits, quantised
from tests.test_gpu_window import SCALE, check, i32

pytestmark = pytest.mark.gpu
FAR = [14563, 14564, 16383, 16384, 29127, 29128, 32767, 32768]          # rows of 128 heads on either side of 2^31 and 2^32 bytes of queries and of outputs


def room(gigabytes):
    if torch.cuda.mem_get_info()[0] < gigabytes << 30:
        pytest.skip(f"needs {gigabytes} GB")


def test_prompt():
    room(24)
    T, H, window, first = 34000, 128, 70, 3
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(T, H, 576, generator=g, device="cuda", dtype=torch.bfloat16)
    kv = torch.randn(T, 576, generator=g, device="cuda", dtype=torch.bfloat16)
    assert q.numel() > 2 ** 31 and T * H * 512 * 2 > 2 ** 32
    ke = torch.arange(1, T + 1, dtype=torch.int32, device="cuda")
    ke[T - 9] = 0                                          # a row that sees nothing
    out = ops.window_mla_prefill(q, kv, None, ke, window, first, SCALE)
    ops.check_status("cuda")
    at = torch.tensor([0, 1, *FAR, T - 40, T - 9, T - 2, T - 1])
    keys = torch.cat((torch.arange(first), *(torch.arange(max(0, t + 1 - window), t + 1) for t in at.tolist()))).unique()
    sees = (keys < ke.cpu()[at, None]) & ((keys < first) | (keys >= ke.cpu()[at, None] - window))
    check(out[at.cuda()], D.attend(q[at.cuda()], kv[keys.cuda()], sees, SCALE))
    assert bool((out[T - 9] == 0).all())


@pytest.mark.parametrize("record", [656, 416])
@pytest.mark.parametrize("per", [1, 5])
def test_decode(record, per):
    """By records, and by rows made of them first; all sequences read the same pages."""
    room(24)
    B, H, ctx = 34000 // per, 128, 100
    g = torch.Generator(device="cuda").manual_seed(2)
    kv = torch.randn(128, 576, generator=g, device="cuda", dtype=torch.bfloat16)
    rec = layer.pack_latent_cache(kv) if record == 656 else ops.pack_latent4(kv)
    q = torch.randn(B * per, H, 576, generator=g, device="cuda", dtype=torch.bfloat16)
    table = i32([[1, 0]]).expand(B, 2).contiguous()
    lens = torch.full((B,), ctx, dtype=torch.int32, device="cuda")
    lens[B - 2] = 0
    out = ops.window_mla_decode_paged(q, rec, table, lens, 40, 2, SCALE, per)
    ops.check_status("cuda")
    values = D.record_values(rec)[torch.cat((torch.arange(64, 128), torch.arange(64)))].cuda()
    seqs = torch.tensor(sorted({0, *(r // per for r in FAR), B - 2, B - 1}))
    at = (seqs[:, None] * per + torch.arange(per)).flatten()
    sees = D.draft_sees(len(seqs), per, [0 if b == B - 2 else ctx for b in seqs.tolist()], 128, None, None, 40, 2)
    check(out[at.cuda()], D.attend(q[at.cuda()], values, sees, SCALE))
    assert bool((out.view(B, -1)[B - 2] == 0).all())


def test_scores_and_selection():
    room(12)
    B, per, H, ctx, k = 2050, 4, 64, 131072, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    k8, ksc = quantised(torch.randn(ctx, 128, generator=g, device="cuda"))
    q8, qs = quantised(torch.randn(B * per, H, 128, generator=g, device="cuda"))
    w = torch.randn(B * per, H, generator=g, device="cuda") * qs * (128 * H) ** -0.5
    table = torch.randperm(ctx // 64, generator=g, device="cuda").int()
    lens = torch.full((B,), ctx, dtype=torch.int32, device="cuda")
    logits = ops.fp8_paged_mqa_logits(q8, w, k8, ksc, table.expand(B, -1).contiguous(), lens, ctx, tokens_per_seq=per)
    idx = ops.topk_select_drafts(logits, k, lens, per)
    ops.check_status("cuda")
    assert logits.numel() * 4 > 2 ** 32
    s = torch.arange(ctx, device="cuda")
    rows = table[s // 64].long() * 64 + s % 64
    for r in (0, 4095, 4096, 8191, 8192, B * per - 1):     # on either side of 2^29 and 2^30 scores
        sees = (s < ctx - per + r % per + 1)[None]
        want = D.logits(q8[r:r + 1], w[r:r + 1], k8.view(torch.uint8)[rows][None].view(ops.FP8), ksc[rows][None], sees)
        check_logits(logits[r:r + 1], want, [ctx], 1)
        best = torch.sort(logits[r].masked_fill(~sees[0], -math.inf), descending=True, stable=True)[1][:k]
        assert sorted(idx[r].tolist()) == sorted(best.tolist())
