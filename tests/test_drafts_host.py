"""Window layers and drafted tokens without a GPU: refusals of the C ABI, and what the oracle says of small cases."""
import random

import numpy as np
import pytest
import torch

from llmdivedeep_b200 import _lib, build, layer, ops
from oracle import drafts_oracle as D


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def refused(lib, rc, code, what):
    assert rc == code and what in lib.dsa_last_error_string(), (rc, lib.dsa_last_error_string())


PREFILL = dict(q=16, kv=16, ks=None, ke=None, out=16, T=4, H=16, S=4, window=8, first=0, scale=0.1, ws=None, nbytes=0, status=None, stream=None)
DECODE = dict(q=16, cache=16, width=416, table=16, stride=2, ctx=16, n_new=None, tree=None, per=2, out=16, B=3, H=16, window=8, first=0, pages=9, max_ctx=128,
              scale=0.1, ws=None, nbytes=0, status=None, stream=None)
LOGITS = dict(q=16, w=16, w_dtype=0, k=16, kscale=16, table=16, stride=2, ctx=16, n_new=None, tree=None, per=2, logits=16, ld=128, B=3, H=64, D=128, pages=9,
              max_ctx=128, status=None, stream=None)
SELECT = dict(logits=16, ld=128, ctx=16, n_new=None, tree=None, per=2, B=3, max_ctx=128, k=4, out=16, ws=16, nbytes=24, stream=None)
ACCEPT = dict(table=16, stride=2, P=2, B=3, ctx=16, refs=16, pages=9, rows=16, n_new=16, path=16, path_stride=4, n_keep=16, n=2, caches=None, n_caches=0, ws=16,
              nbytes=1 << 20, status=None, stream=None)


@pytest.mark.parametrize("change,code,what", [
    (dict(T=-1), -1, b"negative"), (dict(S=-1), -1, b"negative"), (dict(H=-1), -1, b"negative"), (dict(window=0), -1, b"window"), (dict(first=-1), -1, b"first"),
    (dict(scale=0.0), -5, b"scale"), (dict(scale=float("nan")), -5, b"scale"), (dict(q=None), -5, b"NULL"), (dict(kv=None), -5, b"NULL"), (dict(out=None), -5, b"NULL"),
    (dict(q=8), -2, b"aligned"), (dict(kv=4), -2, b"aligned"), (dict(out=24), -2, b"aligned"), (dict(T=1 << 20, H=1 << 12), -1, b"2^31"), (dict(ws=8), -3, b"aligned"),
])
def test_prompt_calls_refused(lib, change, code, what):
    refused(lib, lib.dsa_window_mla_prefill(*{**PREFILL, **change}.values()), code, what)


@pytest.mark.parametrize("change,code,what", [
    (dict(B=-1), -1, b"negative"), (dict(per=0), -1, b"tokens_per_seq"), (dict(per=65, tree=16), -1, b"64"), (dict(tree=12), -2, b"tree"), (dict(width=576), -1, b"records"),
    (dict(window=0), -1, b"window"), (dict(scale=-1.0), -5, b"scale"), (dict(ctx=None), -5, b"NULL"), (dict(cache=None), -5, b"NULL"), (dict(table=None), -5, b"NULL"),
    (dict(q=8), -2, b"aligned"), (dict(max_ctx=129), -1, b"shorter"), (dict(pages=1 << 26), -1, b"too large"), (dict(B=1 << 20, H=1 << 12), -1, b"too large"),
    (dict(B=1 << 30, per=4), -1, b"query rows"), (dict(ws=8), -3, b"aligned"), (dict(max_ctx=-1), -1, b"negative"), (dict(pages=-1), -1, b"negative"),
])
def test_decode_calls_refused(lib, change, code, what):
    refused(lib, lib.dsa_window_mla_decode_paged(*{**DECODE, **change}.values()), code, what)


@pytest.mark.parametrize("change,code,what", [
    (dict(B=-1), -1, b"negative"), (dict(per=0), -1, b"tokens_per_seq"), (dict(per=65, tree=16), -1, b"64"), (dict(H=8), -1, b"unsupported"), (dict(D=64), -1, b"unsupported"),
    (dict(w=None), -5, b"NULL"), (dict(w_dtype=3), -5, b"w_dtype"), (dict(ld=127), -1, b"ld_logits"), (dict(ld=1 << 26), -1, b"too large"), (dict(max_ctx=200, ld=200), -1, b"shorter"),
    (dict(k=8), -2, b"aligned"), (dict(kscale=8), -2, b"aligned"), (dict(pages=-1), -1, b"negative"),
])
def test_logits_calls_refused(lib, change, code, what):
    refused(lib, lib.dsa_indexer_logits_drafts(*{**LOGITS, **change}.values()), code, what)


@pytest.mark.parametrize("change,code,what", [
    (dict(k=-1), -1, b"negative"), (dict(k=70000), -1, b"65535"), (dict(ld=127), -1, b"ld_logits"), (dict(out=None), -5, b"NULL"), (dict(ws=None), -3, b"workspace"),
    (dict(nbytes=23), -3, b"workspace"), (dict(ws=18), -3, b"workspace"), (dict(per=65, tree=16), -1, b"64"),
])
def test_selection_calls_refused(lib, change, code, what):
    refused(lib, lib.dsa_topk_select_drafts(*{**SELECT, **change}.values()), code, what)


@pytest.mark.parametrize("change,code,what", [
    (dict(n=-1), -1, b"negative"), (dict(path_stride=-1), -1, b"negative"), (dict(path=None), -5, b"NULL"), (dict(rows=None), -5, b"NULL"), (dict(n_keep=None), -5, b"NULL"),
    (dict(stride=1), -1, b"overlap"), (dict(refs=None), -5, b"NULL"), (dict(ws=None), -3, b"workspace"), (dict(nbytes=8), -3, b"workspace"), (dict(B=1 << 19), -1, b"262144"),
])
def test_accept_calls_refused(lib, change, code, what):
    refused(lib, lib.dsa_accept_drafts(*{**ACCEPT, **change}.values()), code, what)


def test_empty_calls_do_nothing(lib):
    assert lib.dsa_window_mla_prefill(*{**PREFILL, "T": 0, "q": None}.values()) == 0
    assert lib.dsa_window_mla_decode_paged(*{**DECODE, "B": 0, "q": None}.values()) == 0
    assert lib.dsa_window_mla_decode_paged(*{**DECODE, "H": 0, "q": None}.values()) == 0
    assert lib.dsa_indexer_logits_drafts(*{**LOGITS, "B": 0, "q": None}.values()) == 0
    assert lib.dsa_topk_select_drafts(*{**SELECT, "k": 0, "logits": None}.values()) == 0
    assert lib.dsa_accept_drafts(*{**ACCEPT, "n": 0, "rows": None}.values()) == 0


def test_tensors_on_the_cpu_are_refused():
    q, kv = torch.zeros(2, 16, 576, dtype=torch.bfloat16), torch.zeros(4, 576, dtype=torch.bfloat16)
    rec, table, ints = torch.zeros(64, 416, dtype=torch.uint8), torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    logits = torch.zeros(2, 64)
    for call in (lambda: ops.window_mla_prefill(q, kv, None, None, 4, 0, 0.1),
                 lambda: ops.window_mla_decode_paged(q, rec, table, ints, 4, 0, 0.1, tokens_per_seq=2),
                 lambda: ops.fp8_paged_mqa_logits(torch.zeros(2, 64, 128).to(ops.FP8), torch.zeros(2, 64), torch.zeros(64, 128).to(ops.FP8), torch.zeros(64), table, ints, 64,
                                                  tokens_per_seq=2),
                 lambda: ops.topk_select_drafts(logits, 4, ints, 2),
                 lambda: ops.accept_drafts(table, ints, ints, ints, ints, table, ints, [rec]),
                 lambda: layer.WindowMLA(0.1, 4)(q, kv)):
        with pytest.raises(ops.DsaError, match="CUDA"):
            call()
    with pytest.raises(ops.DsaError, match="block_table"):
        layer.WindowMLA(0.1, 4)(q, rec)


def test_oracle_a_chain_is_a_tree_without_branches_and_a_prompt():
    for ctx, m, window, first in ((20, 7, 4, 2), (7, 7, 3, 0), (30, 1, 50, 0), (12, 5, 2, 9)):
        chain = D.draft_sees(1, 8, [ctx], 40, [m], None, window, first)
        assert torch.equal(chain, D.draft_sees(1, 8, [ctx], 40, [m], torch.full((1, 8), -1), window, first))
        assert torch.equal(chain[:m, :ctx], D.prompt_sees(m, ctx, window, first)) and not chain[m:].any() and not chain[:, ctx:].any()


def test_oracle_a_path_of_a_tree_sees_what_a_sequence_of_its_own_would():
    rng = random.Random(1)
    tree = D.random_tree(rng, 1, 12)
    sees = D.draft_sees(1, 12, [50], 64, [12], tree, 5, 3)
    for i in range(12):
        path = D.draft_paths(50, 12, i, tree[0], 12)
        alone = D.prompt_sees(1, len(path), 5, 3)[0]
        assert [s for k, s in enumerate(path) if alone[k]] == torch.nonzero(sees[i])[:, 0].tolist()


def test_oracle_accept():
    table = np.array([[3, 1, -1], [2, -1, -1]], np.int32)
    cache = np.arange(5 * 64, dtype=np.int64).reshape(1, 5 * 64, 1)
    pool = D.Pool(table, np.array([70, 10], np.int32), np.array([0, 1, 1, 1, 0], np.int32), [cache])
    pool.accept([0, 1], [9, 4], np.array([[1, 2, 5], [0, 3, -1]]), [3, 2])
    assert pool.status == 0 and pool.ctx.tolist() == [64, 8] and pool.table.tolist() == [[3, -1, -1], [2, -1, -1]] and pool.refs.tolist() == [0, 0, 1, 1, 0]
    got = pool.caches[0][0, :, 0]
    assert got[3 * 64 + 61:3 * 64 + 64].tolist() == [3 * 64 + 62, 3 * 64 + 63, 1 * 64 + 2] and got[2 * 64 + 6:2 * 64 + 8].tolist() == [2 * 64 + 6, 2 * 64 + 9]
