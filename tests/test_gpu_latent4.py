"""The paged 4-bit latent cache on the GPU: writing, reading, and attention over it, against numpy in 64 bits."""
import numpy as np
import pytest
import torch

from llmdivedeep_b200 import layer, ops
from oracle import latent4_oracle as L

pytestmark = pytest.mark.gpu
# Attention: the output's rounding to bf16 alone is 1.7e-3 of it (2-norm: 2^-8 times the mean of a uniform error over a binade), the
# rounding of P to bf16 as much again of a sum of that many terms, that of the exchanged half scores to fp16 less than half of it for
# scores of order one.  Three times their root sum of squares; a single value by 2^-6 of the row's largest.
REL, MOST = 7.5e-3, 2.0 ** -6


def rope_bytes(kv):
    return kv[:, 512:].to(torch.bfloat16).contiguous().view(torch.uint8).numpy()


def wide_rows(n, seed, dtype=torch.float32):
    """Rows whose scales span most of the format, with ties, zeros and numbers that are none."""
    g = torch.Generator().manual_seed(seed)
    kv = torch.randn(n, 576, generator=g) * torch.exp(2 * torch.randn(n, 1, generator=g))
    kv[0, :16] = 0
    if n > 5:
        kv[1, 5], kv[2, 40], kv[3, 530] = float("inf"), float("nan"), float("nan")
        kv[4, :16] = torch.tensor([6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, -.25, -.75, -1.25, -1.75, -2.5, -3.5, -5, -6])
        kv[5, :16], kv[5, 16:32] = 3e8, 1e-8
    if n > 300:
        # halfway cases by the thousand: multiples of a quarter of the scale, and scales halfway between two (13 / 96 = 6.5 / 8 / 6)
        kv[10:200, :512] = torch.randint(-24, 25, (190, 512), generator=g) * 0.25 * 1.125
        kv[200:300, :512] = torch.randint(-13, 14, (100, 512), generator=g) * 0.75
    return kv.to(dtype)


@pytest.mark.parametrize("n", [1, 7, 64, 1001])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("form", ["dense", "wide", "columns"])
def test_records_are_the_definition_byte_for_byte(n, dtype, form):
    kv = wide_rows(n, n, dtype)
    want = L.records(kv.double().numpy(), rope_bytes(kv))
    if form == "dense":
        x = kv.cuda()
    elif form == "wide":
        x = torch.zeros(n, 640, dtype=dtype, device="cuda")[:, 32:608]
        x.copy_(kv)
    else:
        x = torch.empty(576, n, dtype=dtype, device="cuda").t()
        x.copy_(kv)
    rec = ops.pack_latent4(x)
    ops.check_status("cuda")
    bad = ~np.isfinite(kv.double().numpy()[:, :512]).reshape(n, 32, 16).all(-1)
    got = rec.cpu().numpy().reshape(n, 2, 208)
    w = want.reshape(n, 2, 208)
    np.testing.assert_array_equal(got[:, :, 128:144], w[:, :, 128:144])
    # a NaN's bits in the rope part may be another NaN's, and a group without a value has no codes to compare
    words = np.ascontiguousarray(got[:, :, :128]).view("<u8").reshape(n, 32), np.ascontiguousarray(w[:, :, :128]).view("<u8").reshape(n, 32)
    np.testing.assert_array_equal(words[0][~bad], words[1][~bad])
    np.testing.assert_array_equal(L.decode(rec.cpu().numpy()), L.decode(want))


@pytest.mark.parametrize("n,pages", [(1, 1), (63, 1), (64, 1), (65, 2), (1000, 17)])
def test_written_by_slot_and_read_by_table(n, pages):
    g = torch.Generator().manual_seed(n)
    pool = pages + 3
    table = torch.randperm(pool, generator=g)[:pages].int()
    pos = torch.arange(n)
    slots = table[pos // 64] * 64 + (pos % 64).int()
    kv = wide_rows(n, n + 1)
    cache = torch.full((pool * 64, 416), 7, dtype=torch.uint8, device="cuda")
    k8 = torch.randint(0, 256, (n, 128), generator=g, dtype=torch.uint8).cuda().view(ops.FP8)
    ksc = torch.randn(n, generator=g).cuda()
    kcache, kscale = torch.zeros(pool * 64, 128, dtype=torch.uint8, device="cuda").view(ops.FP8), torch.zeros(pool * 64, device="cuda")
    skip = slots.clone()
    if n > 60:
        skip[::5] = -1                                             # tokens that are not to be written
    before = cache.clone()
    ops.pack_latent4(kv.cuda(), cache, skip.cuda(), keys=(k8, ksc, kcache, kscale))
    kept = skip >= 0
    rec = L.records(kv.double().numpy(), rope_bytes(kv))
    want = before.cpu().numpy()
    want[skip[kept].long()] = rec[kept.numpy()]
    np.testing.assert_array_equal(np.nan_to_num(L.decode(cache.cpu().numpy()), nan=-1e9), np.nan_to_num(L.decode(want), nan=-1e9))
    untouched = np.setdiff1d(np.arange(pool * 64), skip[kept].numpy())
    np.testing.assert_array_equal(cache.cpu().numpy()[untouched], 7)
    assert torch.equal(kcache.view(torch.uint8)[skip[kept].long().cuda()], k8.view(torch.uint8)[kept.cuda()])
    assert torch.equal(kscale[skip[kept].long().cuda()], ksc[kept.cuda()]) and int((kscale != 0).sum()) == int(kept.sum())
    ops.pack_latent4(kv.cuda(), cache, slots.cuda())
    rows = ops.unpack_latent4(cache, n, table.cuda())
    out = torch.full((n, 640), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.unpack_latent4(cache, n, table.cuda(), out=out[:, 16:592])
    ops.check_status("cuda")
    want = L.values(kv.double().numpy())
    want[:, 512:] = kv[:, 512:].to(torch.bfloat16).double().numpy()
    np.testing.assert_array_equal(rows.double().cpu().numpy(), want)
    np.testing.assert_array_equal(out[:, 16:592].double().cpu().numpy(), want)
    assert bool((out[:, :16] == 3).all() and (out[:, 592:] == 3).all())
    assert torch.equal(ops.unpack_latent4(cache)[slots.long().cuda()].nan_to_num(-7.0), rows.nan_to_num(-7.0))


def test_bad_slots_and_pages_are_flagged_and_skipped():
    kv = torch.randn(3, 576, device="cuda")
    cache = torch.zeros(64, 416, dtype=torch.uint8, device="cuda")
    ops.pack_latent4(kv, cache, torch.tensor([5, 64, 1 << 30], dtype=torch.int32, device="cuda"))
    with pytest.raises(ops.DsaError, match="out of range"):
        ops.check_status("cuda")
    assert int((cache != 0).any(1).sum()) == 1
    rows = ops.unpack_latent4(cache, 130, torch.tensor([0, 9, -1], dtype=torch.int32, device="cuda"))
    with pytest.raises(ops.DsaError, match="out of range"):
        ops.check_status("cuda")
    assert bool((rows[64:] == 0).all()) and bool((rows[5] != 0).any())


def test_tensors_of_other_forms_are_refused():
    kv = torch.randn(4, 576, device="cuda")
    cache = torch.zeros(64, 416, dtype=torch.uint8, device="cuda")
    slots = torch.arange(4, dtype=torch.int32, device="cuda")
    for bad in (dict(kv=kv.half()), dict(kv=kv[:, :512]), dict(cache=cache[:, :400]), dict(cache=cache.int()), dict(slots=slots[:3]), dict(slots=slots.long()),
                dict(kv=kv.cpu()), dict(keys=(kv, kv, kv, kv)), dict(cache=torch.zeros(64, 832, dtype=torch.uint8, device="cuda")[:, :416])):
        with pytest.raises(ops.DsaError):
            ops.pack_latent4(**{**dict(kv=kv, cache=cache, slots=slots), **bad})
    table = torch.zeros(1, dtype=torch.int32, device="cuda")
    for bad in (dict(n=65), dict(n=-1), dict(block_table=table.long()), dict(block_table=table[None]), dict(out=torch.empty(64, 576, device="cuda")),
                dict(out=torch.empty(64, 580, dtype=torch.bfloat16, device="cuda")[:, :576])):
        with pytest.raises(ops.DsaError):
            ops.unpack_latent4(cache, **{**dict(n=64, block_table=table), **bad})
    q = torch.zeros(4, 16, 576, dtype=torch.bfloat16, device="cuda")
    idx = torch.zeros(4, 8, dtype=torch.int32, device="cuda")
    tables = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    assert ops.sparse_mla_decode_paged(q, cache, tables, idx, 0.1, tokens_per_seq=2).shape == (4, 16, 512)
    for bad in (dict(tokens_per_seq=1), dict(tokens_per_seq=0), dict(idx=idx[:3]), dict(q=q[:, :, :512].contiguous()), dict(cache=cache[:, :400].contiguous()),
                dict(cache=cache[:63]), dict(idx=idx.long())):
        with pytest.raises(ops.DsaError):
            ops.sparse_mla_decode_paged(**{**dict(q=q, cache=cache, block_table=tables, idx=idx, scale=0.1, tokens_per_seq=2), **bad})
    assert ops.pack_latent4(kv[:0]).shape == (0, 416) and ops.unpack_latent4(cache, 0).shape == (0, 576)


def attention_case(B, tokens, H, P, K, seed, gain=1.0, lens=None):
    g = torch.Generator().manual_seed(seed)
    pool = B * P + 2
    kv = torch.randn(pool * 64, 576, generator=g).to(torch.bfloat16)
    rec = torch.from_numpy(L.records(kv.double().numpy(), rope_bytes(kv)))
    table = torch.randperm(pool, generator=g)[:B * P].int().view(B, P)
    q = (torch.randn(B * tokens, H, 576, generator=g) * gain).to(torch.bfloat16)
    idx = torch.full((B * tokens, K), -1, dtype=torch.int32)
    for r in range(B * tokens):
        n = min(K, (P * 64 if lens is None else lens[r % len(lens)]))
        idx[r, :n] = torch.randperm(P * 64, generator=g)[:n].int()
    return q, rec, table, idx


def check_attention(out, q, rec, table, idx, scale, tokens=1):
    want = L.attend(q.double().numpy(), rec.numpy(), table.numpy(), idx.numpy(), scale, tokens)
    got = out.double().cpu().numpy()
    err, size = np.linalg.norm(got - want, axis=-1), np.linalg.norm(want, axis=-1)
    assert (err <= REL * size).all(), float((err / np.maximum(size, 1e-30)).max())
    assert (np.abs(got - want).max(-1) <= MOST * np.abs(want).max(-1)).all()


# heads on both sides of each tile's edge; one page and many; a last block of every length class; one query, full rounds of pairs and more
@pytest.mark.parametrize("B,tokens,H,P,K", [
    (1, 1, 128, 1, 1), (1, 1, 128, 1, 64), (1, 1, 128, 3, 65), (2, 1, 128, 40, 2048), (3, 3, 128, 9, 500), (1, 1, 1, 5, 257), (5, 1, 8, 9, 300),
    (2, 2, 16, 36, 2048), (9, 1, 17, 6, 200), (4, 1, 32, 20, 1024), (3, 1, 33, 5, 129), (2, 1, 64, 36, 2048), (2, 1, 129, 5, 300), (1, 1, 256, 36, 2048),
    (75, 1, 16, 2, 100), (40, 4, 16, 2, 128), (150, 1, 8, 1, 64),
])
def test_attention_against_64_bits(B, tokens, H, P, K):
    q, rec, table, idx = attention_case(B, tokens, H, P, K, seed=B * 131 + H + K)
    out = ops.sparse_mla_decode_paged(q.cuda(), rec.cuda(), table.cuda(), idx.cuda(), 192 ** -0.5, tokens_per_seq=tokens)
    ops.check_status("cuda")
    check_attention(out, q, rec, table, idx, 192 ** -0.5, tokens)


@pytest.mark.parametrize("B", [1, 2, 3, 4, 9, 10])
@pytest.mark.parametrize("H", [40, 64, 100, 128, 200])
@pytest.mark.parametrize("room", [0, 2, None])
def test_few_rows_by_groups_of_heads_and_parts(B, H, room):
    """The units of small calls are groups of heads and parts of lists; a workspace holds some of the parts, or none."""
    K = 1100
    q, rec, table, idx = attention_case(B, 1, H, 20, K, seed=B + H, lens=[K, 1, 700, 0, 64, 129, K, 500, 1000, 64][:B])
    need = None if room is None else torch.empty(room * B * H * 514 * 4, dtype=torch.uint8, device="cuda")
    out = ops.sparse_mla_decode_paged(q.cuda(), rec.cuda(), table.cuda(), idx.cuda(), 192 ** -0.5, workspace=need)
    ops.check_status("cuda")
    check_attention(out, q, rec, table, idx, 192 ** -0.5)


@pytest.mark.parametrize("B,tokens,H,P,K,lens", [
    (13, 1, 16, 33, 2048, [2048, 0, 1, 1000, 64, 65, 2048]), (7, 4, 9, 9, 512, [0, 512, 63, 300, 1]), (24, 1, 32, 20, 1100, [1100, 0, 129, 640]),
    (70, 1, 16, 5, 300, [300, 0, 64, 17]), (149, 1, 16, 3, 130, [130, 0, 1, 64, 65]), (160, 1, 24, 3, 192, [192, 5, 0]), (300, 1, 8, 2, 128, [128, 0, 3]),
])
def test_few_heads_of_many_rows(B, tokens, H, P, K, lens):
    """Short lists, holes and rows without keys, whole lists, stretches and equal parts of lists, NaN in what nobody selected."""
    q, rec, table, idx = attention_case(B, tokens, H, P, K, seed=B + H, lens=lens)
    g = torch.Generator().manual_seed(B)
    idx[::4] = torch.where(torch.rand(idx[::4].shape, generator=g) < 0.3, torch.full_like(idx[::4], -1), idx[::4])
    q[1::5] *= 4                                                   # references that grow
    seen = torch.zeros(rec.shape[0], dtype=torch.bool)
    for r in range(B * tokens):
        pos = idx[r][idx[r] >= 0].long()
        seen[table[r // tokens][pos // 64].long() * 64 + pos % 64] = True
    rec[~seen] = 255
    out = torch.full((B * tokens, H, 512), 9.0, dtype=torch.bfloat16, device="cuda")
    for room in (None, torch.empty(0, dtype=torch.uint8, device="cuda")):
        ops.sparse_mla_decode_paged(q.cuda(), rec.cuda(), table.cuda(), idx.cuda(), 192 ** -0.5, out=out, tokens_per_seq=tokens, workspace=room)
        ops.check_status("cuda")
        check_attention(out, q, rec, table, idx, 192 ** -0.5, tokens)


@pytest.mark.parametrize("H", [8, 16, 32, 64, 128])
def test_lists_that_are_short_empty_or_full_of_holes(H):
    lens = [0, 1, 2, 63, 64, 65, 128, 300, 0, 511, 512]
    q, rec, table, idx = attention_case(11, 1, H, 9, 512, seed=H, lens=lens)
    g = torch.Generator().manual_seed(H)
    idx[7] = torch.where(torch.rand(512, generator=g) < 0.5, idx[7], torch.full_like(idx[7], -1))      # holes
    idx[9, :400] = -1                                                                                  # a late start
    idx[10] = -5                                                                                       # any negative is empty
    out = torch.full((11, H, 512), 9.0, dtype=torch.bfloat16, device="cuda")
    ops.sparse_mla_decode_paged(q.cuda(), rec.cuda(), table.cuda(), idx.cuda(), 0.06, out=out)
    ops.check_status("cuda")
    assert bool((out[0] == 0).all() and (out[8] == 0).all() and (out[10] == 0).all())
    check_attention(out, q, rec, table, idx, 0.06)


@pytest.mark.parametrize("H", [16, 128])
@pytest.mark.parametrize("gain", [4.0, 30.0])
def test_wide_scores(H, gain):
    """Maxima that grow past the softmax reference, rows that one key takes over.  The kernel rounds half scores to fp16: their
    error in the exponent is scale * 2^-11 * |half score|, so that much more is allowed."""
    q, rec, table, idx = attention_case(2, 1, H, 20, 1200, seed=int(gain) + H, gain=gain)
    out = ops.sparse_mla_decode_paged(q.cuda(), rec.cuda(), table.cuda(), idx.cuda(), 192 ** -0.5)
    ops.check_status("cuda")
    want = L.attend(q.double().numpy(), rec.numpy(), table.numpy(), idx.numpy(), 192 ** -0.5)
    err = np.linalg.norm(out.double().cpu().numpy() - want, axis=-1) / np.linalg.norm(want, axis=-1)
    half = gain * 24 * 192 ** -0.5 * 4                             # four sigma of |half score| * scale
    assert (err <= REL + 2 * half * 2.0 ** -11).all(), float(err.max())


@pytest.mark.parametrize("H", [16, 64, 128])
def test_numbers_that_are_none_stay_where_they_are(H):
    """NaN and infinities in records nobody selected, in pages nobody has, behind the context's end: no trace of them.  In a selected
    record: in that query's rows and no others."""
    q, rec, table, idx = attention_case(3, 1, H, 6, 200, seed=H)
    seen = torch.zeros(rec.shape[0], dtype=torch.bool)
    for b in range(3):
        pos = idx[b].long()
        seen[table[b][pos // 64].long() * 64 + pos % 64] = True
    poison = torch.full((416,), 255, dtype=torch.uint8)            # NaN scales, NaN rope values
    dirty = rec.clone()
    dirty[~seen] = poison
    out = ops.sparse_mla_decode_paged(q.cuda(), dirty.cuda(), table.cuda(), idx.cuda(), 192 ** -0.5)
    clean = ops.sparse_mla_decode_paged(q.cuda(), rec.cuda(), table.cuda(), idx.cuda(), 192 ** -0.5)
    assert torch.equal(out, clean)
    p = int(idx[1, 77])
    dirty[int(table[1, p // 64]) * 64 + p % 64] = poison
    out = ops.sparse_mla_decode_paged(q.cuda(), dirty.cuda(), table.cuda(), idx.cuda(), 192 ** -0.5)
    ops.check_status("cuda")
    assert torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2]) and bool(out[1].isnan().all())


def test_bad_positions_and_pages_are_flagged_and_skipped():
    for B, H in ((2, 16), (20, 16), (2, 128)):
        q, rec, table, idx = attention_case(B, 1, H, 4, 100, seed=3)
        bad, tab = idx.clone(), table.clone()
        bad[0, 3], bad[0, 70] = 256, 1 << 30                       # at max_ctx, far past it
        tab[1, 2] = 9999                                           # a page that is none
        out = ops.sparse_mla_decode_paged(q.cuda(), rec.cuda(), tab.cuda(), bad.cuda(), 0.05)
        with pytest.raises(ops.DsaError, match="out of range"):
            ops.check_status("cuda")
        idx[0, 3] = idx[0, 70] = -1
        idx[1][(idx[1] >= 128) & (idx[1] < 192)] = -1
        check_attention(out, q, rec, table, idx, 0.05)


@pytest.mark.parametrize("H", [16, 128])
def test_a_row_does_not_depend_on_its_place_in_a_full_round(H):
    q, rec, table, idx = attention_case(4, 2, H, 8, 400, seed=17)
    run = lambda q, i, t, n: ops.sparse_mla_decode_paged(q.contiguous().cuda(), rec.cuda(), t.contiguous().cuda(), i.contiguous().cuda(), 0.07, tokens_per_seq=n)
    both = run(q, idx, table, 2)
    again = run(q, idx, table, 2)
    assert torch.equal(both, again)
    alone = run(q, idx, table.repeat_interleave(2, 0), 1)          # the same rows as sequences of their own
    assert torch.equal(both, alone)


def test_cache_rows_past_two_gigabytes():
    """Record addresses beyond 32 bits: a cache of 5.4 M rows, the selected ones at its end."""
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("needs 8 GB")
    pages, H = 84000, 16
    cache = torch.empty(pages * 64, 416, dtype=torch.uint8, device="cuda")
    g = torch.Generator().manual_seed(0)
    kv = torch.randn(128, 576, generator=g)
    table = torch.tensor([[pages - 1, pages - 70]], dtype=torch.int32)
    pos = torch.arange(128)
    slots = (table[0][pos // 64] * 64 + (pos % 64).int()).int()
    ops.pack_latent4(kv.cuda(), cache, slots.cuda())
    rows = ops.unpack_latent4(cache, 128, table[0].cuda())
    np.testing.assert_array_equal(rows[:, :512].double().cpu().numpy(), L.values(kv.double().numpy())[:, :512])
    for H in (16, 128):
        q = torch.randn(1, H, 576, generator=g).to(torch.bfloat16)
        idx = torch.randperm(128, generator=g).int()[None]
        out = ops.sparse_mla_decode_paged(q.cuda(), cache, table.cuda(), idx.cuda(), 0.07)
        ops.check_status("cuda")
        small = cache[slots.long().cuda()].cpu()
        check_attention(out, q, small, torch.tensor([[0, 1]], dtype=torch.int32), idx, 0.07)


@pytest.mark.parametrize("H", [16, 128])
def test_streams_and_graphs(H):
    """On a side stream behind the tensors' own, and replayed from a graph with other inputs in the same buffers."""
    cases = [attention_case(2, 1, H, 33, 2048, seed=s) for s in (1, 2)]
    want = [ops.sparse_mla_decode_paged(*(t.cuda() for t in c), 0.07) for c in cases]
    bufs = [t.cuda() for t in cases[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.sparse_mla_decode_paged(*bufs, 0.07)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want[0])
    ws = torch.empty(ops._lib.load().dsa_sparse_mla_decode_records_workspace_bytes(416, 2, H, 2048), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sparse_mla_decode_paged(*bufs, 0.07, out=out, workspace=ws)
    for c, w in zip(cases[::-1], want[::-1]):
        for b, t in zip(bufs, c):
            b.copy_(t)
        graph.replay()
        assert torch.equal(out, w)


@pytest.mark.parametrize("B", [1, 3, 30])
def test_decode_step_and_module_over_4_bits(B):
    """layer.dsa_decode_step and SparseMLA take the 4-bit cache where they take the FP8 one."""
    from tests.test_gpu_decode import make_cache
    P, H, K = 12, 64, 256
    q8, w, k8, ksc, table, ctx = make_cache(B, P, 64, seed=B)
    g = torch.Generator().manual_seed(B)
    kv = torch.randn(k8.shape[0], 576, generator=g)
    rec = ops.pack_latent4(kv.cuda())
    q = torch.randn(B, H, 576, generator=g).to(torch.bfloat16)
    ws = layer.DecodeWorkspace(B, H, P * 64, K, "cuda")
    idx, out = layer.dsa_decode_step(*(t.cuda() for t in (q8, w, k8, ksc, table, ctx, q)), rec, 0.06, ws)
    ops.check_status("cuda")
    assert bool(((idx >= 0).sum(1).cpu() == ctx.clamp_max(K)).all())
    check_attention(out, q, rec.cpu(), table, idx.cpu(), 0.06)
    again = layer.SparseMLA(0.06)(q.cuda(), rec, idx, table.cuda())
    assert torch.equal(out, again)


@pytest.mark.parametrize("H", [16, 128])
@pytest.mark.parametrize("tokens", [2, 5])
def test_several_tokens_over_fp8_records(H, tokens):
    """FP8 records with several query rows a sequence: bit for bit what the rows get as sequences of their own."""
    B, P, K = 3, 9, 300
    q, _, table, idx = attention_case(B, tokens, H, P, K, seed=tokens, lens=[300, 0, 65, 17])
    g = torch.Generator().manual_seed(1)
    cache = layer.pack_latent_cache(torch.randn((B * P + 2) * 64, 576, generator=g).bfloat16().cuda())
    q, table, idx = q.cuda(), table.cuda(), idx.cuda()
    got = ops.sparse_mla_decode_paged(q, cache, table, idx, 0.07, tokens_per_seq=tokens)
    want = ops.sparse_mla_decode_paged(q, cache, table.repeat_interleave(tokens, 0), idx, 0.07)
    ops.check_status("cuda")
    assert torch.equal(got, want) and bool((got[1] == 0).all()) and bool(got[0].any())
