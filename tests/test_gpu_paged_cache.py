"""layer.PagedCache: what a serving loop does with the 4-bit cache and its pages, against the tokens themselves."""
import numpy as np
import pytest
import torch

from llmdivedeep_b200 import layer, ops
from oracle import dsa_oracle as O
from oracle import latent4_oracle as L

pytestmark = pytest.mark.gpu


def test_a_serving_loop_keeps_every_sequence():
    """Prompts, decode tokens, forks, frees and compactions in turn over two layers.  All positions are selected, so a step's output is
    the attention over the tokens that the sequence holds, whatever pages they are in."""
    rng, g = np.random.default_rng(2), torch.Generator().manual_seed(2)
    B, heads, max_ctx, layers = 5, 16, 320, 2
    cache = layer.PagedCache(layers, 24, B, max_ctx, "cuda")
    ws = layer.DecodeWorkspace(B, heads, max_ctx, max_ctx, "cuda")
    tokens = [[] for _ in range(B)]                    # per row: a list of [layers, 576] values as they read back
    addresses = [t.data_ptr() for t in (cache.table, cache.ctx, cache.refs, *cache.caches)]

    def append(rows, n_new):
        most = max(n_new)
        slots = cache.extend(rows, n_new, most)
        kv = torch.randn(layers, len(rows), most, 576, generator=g).to(torch.bfloat16)
        k8, ks = O.fp8_quant_per_block(torch.randn(len(rows), most, 128, generator=g), 128)
        for lay in range(layers):
            cache.write(lay, slots, kv[lay].cuda(), k8.cuda(), ks.cuda())
        for i, r in enumerate(rows):
            for t in range(n_new[i]):
                tokens[r].append(kv[:, i, t].double().numpy())

    def free_pages():
        return int((cache.refs == 0).sum())

    for step in range(60):
        order = list(map(int, rng.permutation(B)))
        kind = int(rng.integers(5))
        if kind <= 1:                                  # prompts and decode tokens
            rows = order[:2]
            n_new = [int(min(rng.choice([1, 1, 30, 64, 100]), max_ctx - len(tokens[r]))) for r in rows]
            need = sum(-(-(len(tokens[r]) + n) // 64) - -(-len(tokens[r]) // 64) for r, n in zip(rows, n_new))
            if max(n_new) and need <= free_pages():
                append(rows, n_new)
        elif kind == 2:
            empty = [r for r in order if not tokens[r]][:2]
            held = [r for r in order if tokens[r]]
            if empty and held and len(empty) <= free_pages():
                parents = [held[0]] * len(empty)
                cache.fork(parents, empty)
                for c in empty:
                    tokens[c] = list(tokens[held[0]])
        elif kind == 3:
            cache.free(order[:1])
            tokens[order[0]] = []
        else:
            cache.compact()
            used = int((cache.refs > 0).sum())
            assert bool((cache.refs[:used] > 0).all())
        assert cache.ctx.tolist() == [len(t) for t in tokens]
        if step % 6 == 5:
            q = torch.randn(B, heads, 576, generator=g).to(torch.bfloat16)
            q8, qs = O.fp8_quant_per_block(torch.randn(B, 64, 128, generator=g), 128)
            w = O.fold_weights(torch.randn(B, 64, generator=g) / 8, qs, 128)
            lay = step % layers
            idx, out = cache.decode(lay, q8.cuda(), w.cuda(), q.cuda(), 192 ** -0.5, ws)
            for r in range(B):
                n = len(tokens[r])
                assert sorted(idx[r][idx[r] >= 0].tolist()) == list(range(n))
                if n == 0:
                    assert not bool(out[r].any())
                    continue
                vals = L.values(np.stack([t[lay] for t in tokens[r]]))
                np.testing.assert_array_equal(cache.read(lay, r, n).double().cpu().numpy(), vals)
                s = q[r].double().numpy() @ vals.T * 192 ** -0.5
                p = np.exp(s - s.max(-1, keepdims=True))
                want = p / p.sum(-1, keepdims=True) @ vals[:, :512]
                err = np.linalg.norm(out[r].double().cpu().numpy() - want, axis=-1)
                assert (err <= 7.5e-3 * np.linalg.norm(want, axis=-1)).all()      # test_gpu_latent4.py's bound
    ops.check_status("cuda")
    assert addresses == [t.data_ptr() for t in (cache.table, cache.ctx, cache.refs, *cache.caches)]


def test_a_full_pool_is_said_and_nothing_is_lost():
    cache = layer.PagedCache(1, 3, 3, 256, "cuda")
    a = cache.extend([0], [128], 128)
    b = cache.extend([1, 2], [64, 1], 64)              # one page too many
    with pytest.raises(ops.DsaError, match="too few free pages"):
        ops.check_status("cuda")
    assert bool((b == -1).all()) and cache.ctx.tolist() == [128, 0, 0] and int(cache.refs.sum()) == 2
    kv = torch.randn(2, 64, 576, device="cuda")
    cache.write(0, b, kv, torch.zeros(2, 64, 128, device="cuda").to(ops.FP8), torch.ones(2, 64, device="cuda"))      # goes nowhere
    assert not bool(cache.latent.any())
    assert sorted(a[0].tolist()) == list(range(128))
    cache.free([0])
    assert bool((cache.extend([1, 2], [64, 1], 64)[0] >= 0).all())
    ops.check_status("cuda")


def test_prefill_over_a_cached_prefix():
    """A chunk of new tokens behind a cached prompt: written, read back with the prefix, attended over by the prefill kernel."""
    g = torch.Generator().manual_seed(0)
    cache = layer.PagedCache(1, 12, 1, 700, "cuda")
    kv = torch.randn(500, 576, generator=g).to(torch.bfloat16)
    k8, ks = O.fp8_quant_per_block(torch.randn(500, 128, generator=g), 128)
    for a, b in ((0, 333), (333, 500)):
        slots = cache.extend([0], [b - a], b - a)
        cache.write(0, slots, kv[a:b].cuda(), k8[a:b].cuda(), ks[a:b].cuda())
    q = torch.randn(167, 128, 576, generator=g).to(torch.bfloat16)
    idx = torch.full((167, 256), -1, dtype=torch.int32)
    for i in range(167):
        idx[i] = torch.randperm(334 + i, generator=g)[:256].int()
    rows = cache.read(0, 0, 500)
    out = ops.sparse_mla_prefill(q.cuda(), rows, idx.cuda(), 192 ** -0.5)
    direct = ops.sparse_mla_decode_paged(q.cuda(), cache.latent[0], cache.table, idx.cuda(), 192 ** -0.5, tokens_per_seq=167)
    ops.check_status("cuda")
    want = O.sparse_mla(q[::29], torch.from_numpy(L.values(kv.double().numpy())).to(torch.bfloat16), idx[::29], 192 ** -0.5)
    for got in (out, direct):
        err = (got.float().cpu()[::29] - want).abs()
        assert float(err.max()) <= 2e-2 and float(err.mean()) <= 2e-3
