"""Selected positions that are out of range, in every attention kernel: skipped, and reported wherever in the list they stand."""
import pytest
import torch

from llmdivedeep_b200 import layer, ops
from tests.test_gpu_latent4 import attention_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,rows", [(16, (1, 12, 13, 20)), (32, (2, 13)), (64, (1, 20)), (128, (1, 8, 76))])
@pytest.mark.parametrize("width", [416, 656])
def test_decode(H, rows, width):
    """One behind the last slot that is used, in a list that is finished otherwise: its access is skipped and it is said, whatever
    kernel takes the call and however many parts the list has."""
    for T in rows:
        for at, worth in ((700, 256), (1999, 1 << 30), (65, 257)):
            q, rec, table, _ = attention_case(T, 1, H, 4, 1, seed=T)
            idx = torch.full((T, 2000), -1, dtype=torch.int32)
            idx[:, 0] = 5
            cache = rec.cuda() if width == 416 else layer.pack_latent_cache(torch.randn(rec.shape[0], 576, device="cuda").bfloat16())
            args = q.cuda(), cache, table.cuda()
            want = ops.sparse_mla_decode_paged(*args, idx.cuda(), 0.05)
            ops.check_status("cuda")
            for row in {0, T - 1}:                     # of a call of many: in a full round, in the last one
                bad = idx.clone()
                bad[row, at] = worth
                got = ops.sparse_mla_decode_paged(*args, bad.cuda(), 0.05)
                with pytest.raises(ops.DsaError, match="out of range"):
                    ops.check_status("cuda")
                assert torch.equal(got, want)


@pytest.mark.parametrize("H", [16, 128])
def test_prefill(H):
    T, S = 80, 300
    q, kv = torch.randn(T, H, 576, device="cuda").bfloat16(), torch.randn(S, 576, device="cuda").bfloat16()
    idx = torch.full((T, 2000), -1, dtype=torch.int32, device="cuda")
    idx[:, 0] = 5
    want = ops.sparse_mla_prefill(q, kv, idx, 0.05)
    ops.check_status("cuda")
    for row, at, worth in ((0, 700, S), (T - 1, 1999, 1 << 30), (7, 65, S + 1)):
        bad = idx.clone()
        bad[row, at] = worth
        got = ops.sparse_mla_prefill(q, kv, bad, 0.05)
        with pytest.raises(ops.DsaError, match="out of range"):
            ops.check_status("cuda")
        assert torch.equal(got, want)
