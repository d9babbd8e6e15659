"""Scratch that the caller gives: what is not a block of its own bytes is refused."""
import pytest
import torch

from llmdivedeep_b200 import layer, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width", [416, 656])
@pytest.mark.parametrize("tokens", [1, 2])
def test_attention(width, tokens):
    T, H, K = 4, 16, 1024
    q = torch.randn(T, H, 576, device="cuda").bfloat16()
    kv = torch.randn(1024, 576, device="cuda").bfloat16()
    cache = ops.pack_latent4(kv) if width == 416 else layer.pack_latent_cache(kv)
    table = torch.arange(16, dtype=torch.int32, device="cuda").repeat(T // tokens, 1)
    idx = torch.stack([torch.randperm(1024, device="cuda") for _ in range(T)]).int()
    need = ops._lib.load().dsa_sparse_mla_decode_records_workspace_bytes(width, T, H, K)
    want = ops.sparse_mla_decode_paged(q, cache, table, idx, 0.07, tokens_per_seq=tokens)
    room = torch.empty(2 * need, dtype=torch.uint8, device="cuda")
    for bad in (room[:1].expand(need), room[::2], room.view(2, need).t()):
        with pytest.raises(ops.DsaError, match="contiguous"):
            ops.sparse_mla_decode_paged(q, cache, table, idx, 0.07, workspace=bad, tokens_per_seq=tokens)
    assert torch.equal(want, ops.sparse_mla_decode_paged(q, cache, table, idx, 0.07, workspace=room, tokens_per_seq=tokens))
    ops.check_status("cuda")


def test_indexer():
    q, k = torch.randn(64, 64, 128, device="cuda").to(ops.FP8), torch.randn(300, 128, device="cuda").to(ops.FP8)
    ke = torch.full((64,), 300, dtype=torch.int32, device="cuda")
    args = q, k, torch.ones(300, device="cuda"), torch.rand(64, 64, device="cuda"), None, ke, 32
    need = ops._lib.load().dsa_indexer_topk_workspace_bytes(64, 300)
    with pytest.raises(ops.DsaError, match="contiguous"):
        ops.indexer_topk(*args, workspace=torch.empty(1, dtype=torch.uint8, device="cuda").expand(need))
    assert torch.equal(ops.indexer_topk(*args), ops.indexer_topk(*args, workspace=torch.empty(need, dtype=torch.uint8, device="cuda")))
    ops.check_status("cuda")
