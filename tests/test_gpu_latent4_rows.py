"""Attention over the 4-bit cache by the number of query rows: calls of at most 32 heads go to one kernel or another by it, calls of more
heads are cut into full rounds and a split last one.  The forms that each of them has to hold, against 64 bits."""
import numpy as np
import pytest
import torch

from llmdivedeep_b200 import layer, ops
from oracle import latent4_oracle as L
from tests.test_gpu_latent4 import REL, attention_case, check_attention

pytestmark = pytest.mark.gpu
SCALE = 192 ** -0.5


def on_gpu(*ts):
    return [t.cuda() for t in ts]


@pytest.mark.parametrize("B,H,K", [(76, 64, 600), (76, 128, 520), (150, 128, 512), (40, 200, 520)])
@pytest.mark.parametrize("tokens", [1, 2])
def test_full_rounds_of_pairs_and_a_split_last_one(B, H, K, tokens):
    """74 pairs (37 of more than 128 heads) and two or three queries more, whose lists are cut: with room for the parts and without."""
    q, rec, table, idx = attention_case(B // tokens, tokens, H, 12, K, seed=B + H, lens=[K, K, 300, K, 0, 65, K])
    out = torch.full((B, H, 512), 9.0, dtype=torch.bfloat16, device="cuda")
    for room in (None, torch.empty(0, dtype=torch.uint8, device="cuda")):
        ops.sparse_mla_decode_paged(*on_gpu(q, rec, table, idx), SCALE, out=out, tokens_per_seq=tokens, workspace=room)
        ops.check_status("cuda")
        check_attention(out, q, rec, table, idx, SCALE, tokens)


@pytest.mark.parametrize("H", [16, 32])
@pytest.mark.parametrize("gain", [4.0, 30.0])
@pytest.mark.parametrize("B,K", [(20, 600), (150, 130)])
def test_few_heads_wide_scores(H, gain, B, K):
    """References that grow many times, rows that one key takes over, in parts of lists (20 rows) and in whole ones (150).  Nothing but P is
    rounded: a score's error is that of 36 sums in fp32, 2^-23 of the largest each, four sigma of |score| * scale."""
    q, rec, table, idx = attention_case(B, 1, H, -(-K // 64), K, seed=int(gain) + H + B, gain=gain)
    out = ops.sparse_mla_decode_paged(*on_gpu(q, rec, table, idx), SCALE)
    ops.check_status("cuda")
    want = L.attend(q.double().numpy(), rec.numpy(), table.numpy(), idx.numpy(), SCALE)
    err = np.linalg.norm(out.double().cpu().numpy() - want, axis=-1) / np.linalg.norm(want, axis=-1)
    score = 4 * gain * 24 * SCALE
    assert (err <= REL + 2 * score * 36 * 2.0 ** -23).all(), float(err.max())


@pytest.mark.parametrize("H", [16, 32])
@pytest.mark.parametrize("B,K", [(20, 200), (20, 2000), (160, 100)])
def test_few_heads_numbers_that_are_none_stay_where_they_are(H, B, K):
    """A NaN in a record that one row selected, in its first block, in a later part of its list: that row is NaN, the others have no
    trace of it."""
    q, rec, table, idx = attention_case(B, 1, H, -(-K // 64), K, seed=H + B + K)
    args = on_gpu(q, rec, table, idx)
    clean = ops.sparse_mla_decode_paged(*args, SCALE)
    poison = torch.full((416,), 255, dtype=torch.uint8)            # NaN scales, NaN rope values
    for row, slot in ((7, 3), (11, K - 1), (B - 1, K // 2)):
        dirty, p = rec.clone(), int(idx[row, slot])
        dirty[int(table[row, p // 64]) * 64 + p % 64] = poison
        out = ops.sparse_mla_decode_paged(args[0], dirty.cuda(), *args[2:], SCALE)
        ops.check_status("cuda")
        others = torch.arange(B, device="cuda") != row
        assert bool(out[row].isnan().all()) and torch.equal(out[others], clean[others])


@pytest.mark.parametrize("H", [16, 32])
@pytest.mark.parametrize("B", [20, 150])
def test_few_heads_a_row_is_the_same_as_one_of_several_and_alone(H, B):
    q, rec, table, idx = on_gpu(*attention_case(B // 2, 2, H, 8, 400, seed=17))
    both = ops.sparse_mla_decode_paged(q, rec, table, idx, 0.07, tokens_per_seq=2)
    assert torch.equal(both, ops.sparse_mla_decode_paged(q, rec, table, idx, 0.07, tokens_per_seq=2))
    assert torch.equal(both, ops.sparse_mla_decode_paged(q, rec, table.repeat_interleave(2, 0), idx, 0.07))


def test_few_heads_cache_rows_past_two_gigabytes():
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("needs 8 GB")
    pages, T = 84000, 20
    cache = torch.empty(pages * 64, 416, dtype=torch.uint8, device="cuda")
    g = torch.Generator().manual_seed(0)
    kv = torch.randn(128, 576, generator=g)
    table = torch.tensor([[pages - 1, pages - 70]], dtype=torch.int32)
    pos = torch.arange(128)
    slots = (table[0][pos // 64] * 64 + (pos % 64).int()).int().cuda()
    ops.pack_latent4(kv.cuda(), cache, slots)
    for H in (16, 32):
        q = torch.randn(T, H, 576, generator=g).to(torch.bfloat16)
        idx = torch.stack([torch.randperm(128, generator=g).int() for _ in range(T)])
        out = ops.sparse_mla_decode_paged(q.cuda(), cache, table.cuda(), idx.cuda(), 0.07, tokens_per_seq=T)
        ops.check_status("cuda")
        check_attention(out, q, cache[slots.long()].cpu(), torch.tensor([[0, 1]], dtype=torch.int32), idx, 0.07, T)


@pytest.mark.parametrize("H", [16, 32])
@pytest.mark.parametrize("B", [20, 150])
def test_few_heads_streams_and_graphs(H, B):
    """On a side stream behind the tensors' own, and replayed from a graph, twice in a row, with other inputs in the same buffers."""
    cases = [attention_case(B, 1, H, 5, 300, seed=s) for s in (1, 2)]
    want = [ops.sparse_mla_decode_paged(*on_gpu(*c), 0.07) for c in cases]
    bufs = on_gpu(*cases[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.sparse_mla_decode_paged(*bufs, 0.07)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want[0])
    ws = torch.empty(ops._lib.load().dsa_sparse_mla_decode_records_workspace_bytes(416, B, H, 300), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sparse_mla_decode_paged(*bufs, 0.07, out=out, workspace=ws)
    for c, w in zip(cases[::-1], want[::-1]):
        for b, t in zip(bufs, c):
            b.copy_(t)
        for _ in range(2):
            out.fill_(9)
            graph.replay()
            assert torch.equal(out, w)


@pytest.mark.parametrize("B", [12, 13, 20, 24, 25, 160])
@pytest.mark.parametrize("H", [16, 32])
def test_decode_steps_of_few_heads(B, H):
    """Steps in a row, those of up to 24 sequences with each kernel under the end of the one before: lists, output, and the same from the
    single calls."""
    from tests.test_gpu_decode import make_cache
    P, K = 12, 256
    q8, w, k8, ksc, table, ctx = make_cache(B, P, 64, seed=B)
    g = torch.Generator().manual_seed(B)
    rec = ops.pack_latent4(torch.randn(k8.shape[0], 576, generator=g).cuda())
    ctx[B // 2] = 0                                                # a row that no sequence uses
    dev = on_gpu(q8, w, k8, ksc, table, ctx)
    ws = layer.DecodeWorkspace(B, H, P * 64, K, "cuda")
    steps = [torch.randn(B, H, 576, generator=g).to(torch.bfloat16) for _ in range(4)]
    outs = []
    for q in steps:
        idx, out = layer.dsa_decode_step(*dev, q.cuda(), rec, 0.06, ws)
        outs.append((idx.clone(), out.clone()))
    ops.check_status("cuda")
    for q, (idx, out) in zip(steps, outs):
        assert torch.equal((idx >= 0).sum(1), dev[5].clamp_max(K)) and torch.equal(idx, outs[0][0])
        assert not bool(out[B // 2].any())
        assert torch.equal(out, ops.sparse_mla_decode_paged(q.cuda(), rec, dev[4], idx, 0.06))
    check_attention(outs[-1][1], steps[-1], rec.cpu(), table, outs[-1][0].cpu(), 0.06)
