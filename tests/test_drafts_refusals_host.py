"""Calls of the cache's drafts that are refused before anything is launched."""
import pytest
import torch

from llmdivedeep_b200 import layer, ops


@pytest.mark.parametrize("per", [0, -1, -3, 4, 7])
def test_query_rows_that_are_no_whole_number_a_sequence(per):
    cache = layer.PagedCache(1, 4, 3, 128, "cpu")
    q = torch.zeros(6, 16, 576, dtype=torch.bfloat16)
    with pytest.raises(ops.DsaError, match="a sequence"):
        cache.window(0, q, 10, 0, 0.1, tokens_per_seq=per)
    with pytest.raises(ops.DsaError, match="a sequence"):
        cache.decode_drafts(0, torch.zeros(6, 64, 128).to(ops.FP8), torch.zeros(6, 64), q, 0.1, None, per)
